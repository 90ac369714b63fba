// norm_quant.hip — the residual's addition, RMS norm and outlier-aware int8
// rows in one pass (gfx950): what stands between two int8 linears.
//
//   s = x + y;  n = RN32(s / sqrt(mean(s^2) + eps) * w);  a8, sa, outliers of n
// The mean and the norm are formed in 64 bits and rounded to f32 once, so the
// int8 rows do not depend on an order of summation; the quantisation is
// quant_core.h's (frq_quant_i8_dev's bytes for the rows n).  A row is read
// once and stays in registers; only the selection of rows with many equal
// magnitudes puts it into LDS, over the candidates it has done with.
//
// Bound by the selection's passes over the registers, with the loads of other
// workgroups behind them: 4096 rows of 4096 channels, 219 MB, in 61 us (3.6
// TB/s; a large copy reaches 4.8), waves waiting for memory and at barriers
// 57% of their time; one row of 3584 in 7.7 us, by latency.  With the row n
// always in LDS the large case took 66 us.
#include "quant_core.h"

namespace frq {
namespace {

constexpr int MAX_K = 28672;  // a row in LDS, 112 KB, beside the selection's 15 KB

struct NormArgs {
    const float *x, *y, *w;
    double eps;
    int k, kp;
    float* sum;
    int8_t* a8;
    float* sa;
    uint32_t* oidx;
    float* oval;
    int* err;
};

struct __attribute__((packed, aligned(4))) F4u {
    float x, y, z, w;
};

__host__ __device__ constexpr int bitmap_quads(int kp) { return ((kp + 31) / 32 + 3) / 4; }

// Four values of a row at 4 i (rows of any alignment; zero past k).
__device__ __forceinline__ float4 row4(const float* p, int i, int k) {
    if (4 * i + 3 < k) {
        const F4u f = *reinterpret_cast<const F4u*>(p + 4 * i);
        return make_float4(f.x, f.y, f.z, f.w);
    }
    return make_float4(4 * i < k ? p[4 * i] : 0.0f, 4 * i + 1 < k ? p[4 * i + 1] : 0.0f,
                       4 * i + 2 < k ? p[4 * i + 2] : 0.0f, 0.0f);
}

template <int NV4, int NT>
__global__ __launch_bounds__(NT) void norm_quant_kernel(const NormArgs a) {
    __shared__ qc::RowLdsT<NT> L;
    __shared__ double wsum[NT / 64];
    extern __shared__ float4 lds4[];  // the bitmap, then the candidates or the row n
    const int tid = threadIdx.x, k = a.k, k4 = (k + 3) >> 2;
    const size_t row = blockIdx.x;
    uint32_t* bitmap = reinterpret_cast<uint32_t*>(lds4);
    float4* lrow = lds4 + bitmap_quads(a.kp);
    const float* x = a.x + row * k;
    float4 v[NV4], w[NV4];
#pragma unroll
    for (int i = 0; i < NV4; ++i) v[i] = row4(x, tid + NT * i, k);
    if (a.y) {
        const float* y = a.y + row * k;
        float4 u[NV4];
#pragma unroll
        for (int i = 0; i < NV4; ++i) u[i] = row4(y, tid + NT * i, k);
#pragma unroll
        for (int i = 0; i < NV4; ++i) {
            v[i].x += u[i].x;
            v[i].y += u[i].y;
            v[i].z += u[i].z;
            v[i].w += u[i].w;
        }
    }
#pragma unroll
    for (int i = 0; i < NV4; ++i) w[i] = row4(a.w, tid + NT * i, k);
    if (a.sum) {
        float* d = a.sum + row * k;
#pragma unroll
        for (int i = 0; i < NV4; ++i) {
            const int c = 4 * (tid + NT * i);
            if (c + 3 < k) {
                *reinterpret_cast<F4u*>(d + c) = F4u{v[i].x, v[i].y, v[i].z, v[i].w};
            } else {
                if (c < k) d[c] = v[i].x;
                if (c + 1 < k) d[c + 1] = v[i].y;
                if (c + 2 < k) d[c + 2] = v[i].z;
            }
        }
    }
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NV4; ++i) {
        ss = __builtin_fma((double)v[i].x, (double)v[i].x, ss);
        ss = __builtin_fma((double)v[i].y, (double)v[i].y, ss);
        ss = __builtin_fma((double)v[i].z, (double)v[i].z, ss);
        ss = __builtin_fma((double)v[i].w, (double)v[i].w, ss);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) ss += __shfl_xor(ss, d, 64);
    if ((tid & 63) == 0) wsum[tid >> 6] = ss;
    __syncthreads();
    ss = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) ss += wsum[i];
    const double inv = 1.0 / sqrt(ss / (double)k + a.eps);
#pragma unroll
    for (int i = 0; i < NV4; ++i) {
        v[i].x = (float)((double)v[i].x * inv * (double)w[i].x);
        v[i].y = (float)((double)v[i].y * inv * (double)w[i].y);
        v[i].z = (float)((double)v[i].z * inv * (double)w[i].z);
        v[i].w = (float)((double)v[i].w * inv * (double)w[i].w);
        const int left = k - 4 * (tid + NT * i);  // zero past k whatever inv is
        if (left < 4) v[i].w = 0.0f;
        if (left < 3) v[i].z = 0.0f;
        if (left < 2) v[i].y = 0.0f;
        if (left < 1) v[i].x = 0.0f;
    }
    int8_t* a8 = a.a8 + row * a.kp;
    uint32_t* a8w = reinterpret_cast<uint32_t*>(a8);
    uint32_t* oi = a.oidx + row * FRQ_T;
    float* ov = a.oval + row * FRQ_T;
    auto put = [&]() {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV4; ++i)
            if (tid + NT * i < k4) lrow[tid + NT * i] = v[i];
        __syncthreads();
    };
    const float* n = reinterpret_cast<const float*>(lrow);
    if (k <= FRQ_T) {  // every channel is an outlier
        put();
        for (int i = tid; i < a.kp / 4; i += NT) a8w[i] = 0u;
        if (tid < FRQ_T) {
            oi[tid] = tid < k ? (uint32_t)tid : 0u;
            ov[tid] = tid < k ? n[tid] : 0.0f;
        }
        if (tid == 0) a.sa[row] = 1.0f;
        return;
    }
    // zeros past k are the last to be taken, and k > 32 channels come first
    const qc::RowSel s = qc::row_select<NV4, NT>(n, 4 * k4, v, L, reinterpret_cast<unsigned long long*>(lrow), bitmap,
                                                   (a.kp + 31) / 32, put);
    if (s.nan) {  // frq_quant_i8_dev's placeholders, reported by frq_sync
        if (tid == 0) atomicOr(a.err, 1);
        for (int i = tid; i < k4; i += NT) a8w[i] = 0u;
    } else {
        qc::row_quantize<NV4, NT>(v, k4, bitmap, s.sa, s.fast, [&](int i4, uint32_t q) { a8w[i4] = q; });
    }
    for (int i = k4 + tid; i < a.kp / 4; i += NT) a8w[i] = 0u;
    if (tid < FRQ_T) {
        oi[tid] = L.sel_i[tid];
        ov[tid] = L.sel_v[tid];
    }
    if (tid == 0) a.sa[row] = s.sa;
}

template <int NV4, int NT>
hipError_t launch(const NormArgs& a, size_t m, hipStream_t s) {
    const size_t row = (size_t)((a.k + 3) / 4) * 16, cand = qc::FCAP * sizeof(unsigned long long);
    const size_t lds = (size_t)bitmap_quads(a.kp) * 16 + (row > cand ? row : cand);
    if (lds > 32 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(norm_quant_kernel<NV4, NT>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    norm_quant_kernel<NV4, NT><<<dim3((unsigned)m), dim3(NT), lds, s>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace frq

using namespace frq;

extern "C" int frq_norm_quant_i8_dev(frq_ctx* ctx, const float* d_x, const float* d_y, const float* d_w, double eps,
                                     size_t m, size_t k, float* d_sum, int8_t* d_a8, float* d_sa, uint32_t* d_oidx,
                                     float* d_oval) {
    if (!k || k > MAX_K) return set_error(FRQ_ERR_ARG, "frq_norm_quant_i8_dev: k must be in [1, 28672]");
    if (m > 0x7FFFFFFF) return set_error(FRQ_ERR_ARG, "too many rows");
    if (!(eps >= 0.0) || eps > 1e30) return set_error(FRQ_ERR_ARG, "eps must be 0 or positive");
    if (m && (!d_x || !d_w || !d_a8 || !d_sa || !d_oidx || !d_oval)) return set_error(FRQ_ERR_ARG, "null pointer");
    if ((uintptr_t)d_a8 & 3) return set_error(FRQ_ERR_ARG, "the int8 rows must be 4-byte aligned");
    if (!ctx) return set_error(FRQ_ERR_ARG, "null context");
    if (!m) return FRQ_OK;
    int prev = -1;
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != ctx_device(ctx)) (void)hipSetDevice(ctx_device(ctx));
    const NormArgs a{d_x, d_y, d_w, eps, (int)k, (int)round_up(k, FRQ_KALIGN), d_sum, d_a8, d_sa, d_oidx, d_oval,
                     ctx_err(ctx)};
    hipStream_t s = (hipStream_t)frq_get_stream(ctx);
    const size_t k4 = (k + 3) / 4;
    hipError_t e;
    // 256 threads a row; up to 256 rows, a row a CU, of 2049 .. 4096 channels 512
    // (512 against 256, calls one after the other: K = 2304 one row 7.0, 7.5 us, 256
    // rows 8.1, 8.3, 512 rows 11.2, 9.6; K = 4096 7.3, 8.0, then 8.8, 9.2, then 12.8,
    // 11.2; 4096 rows 58.1, 51.5)
    if (m <= 256 && k4 > 512 && k4 <= 1024) e = launch<2, 512>(a, m, s);
    else if (k4 <= 256) e = launch<1, 256>(a, m, s);
    else if (k4 <= 512) e = launch<2, 256>(a, m, s);
    else if (k4 <= 1024) e = launch<4, 256>(a, m, s);
    else if (k4 <= 2048) e = launch<8, 256>(a, m, s);
    else if (k4 <= 5120) e = launch<5, 1024>(a, m, s);
    else e = launch<7, 1024>(a, m, s);
    if (prev >= 0) (void)hipSetDevice(prev);
    return e == hipSuccess ? FRQ_OK : set_error(FRQ_ERR_HIP, std::string("launch norm_quant: ") + hipGetErrorString(e));
}
