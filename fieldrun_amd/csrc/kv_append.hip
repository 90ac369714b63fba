// kv_append.hip — fused q | k | v rows made ready for attention in one launch:
// biases, the norm of every query and key head, the rotation by position; q
// out in f32, keys and values into their pages (kv_rows.h, the cache's own
// rounding).
//
//   y = x + b;  y = y / sqrt(mean(y^2) + eps) * gain    (q and k, with gains)
//   (y_a, y_b) = (y_a cos t - y_b sin t, y_b cos t + y_a sin t),  t = pos freq_j
// (Rope::proj, head_norm and rope, src/rope.rs:72-117; src/gemma.rs:79-94) over
// the planes j: channels (j, j + rot / 2), or the neighbours (2 j, 2 j + 1).
// Everything is formed in 64 bits and rounded to f32 once, where the engines
// round every step: a far position's angle keeps its bits, and an int8 key does
// not depend on the order of a sum.
#include "kv_rows.h"

namespace frq {
namespace kv {
namespace {

struct Append {
    Move m;  // the rows' values: wv, and the slots
    const float *x, *bias, *qn, *kn;
    double eps;
    const double* freq;
    const int32_t* pos;
    float* q;
    int64_t q_pitch;
    int half, pairs;         // planes; neighbours
    int n_head;
    int rshift, units;       // rows a workgroup (a power of two), heads a workgroup
    int slices;              // workgroups over the heads
    unsigned value_groups;   // the first workgroups: the values
};

// cos and sin of an angle: the nearest multiple of pi / 2 taken off in two
// parts (the first one's rounding error is the second), the rest's Taylor series,
// whose next terms are below 5e-17.
__device__ __forceinline__ double2 turn_of(double t) {
    const double n = __builtin_rint(t * 0.63661977236758134308);
    double r = __builtin_fma(-n, 1.57079632679489655800, t);
    r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
    s = __builtin_fma(s, z, 1.0 / 6227020800.0);
    c = __builtin_fma(c, z, -1.0 / 87178291200.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    c = __builtin_fma(c, z, -0.5);
    s = __builtin_fma(s * z, r, r);
    c = __builtin_fma(c, z, 1.0);
    const int k = (int)(n - 4.0 * __builtin_floor(0.25 * n));  // the quarter, 0 .. 3
    const double a = k & 1 ? s : c, b = k & 1 ? c : s;
    return double2{k == 1 || k == 2 ? -a : a, k >= 2 ? -b : b};
}

__device__ __forceinline__ double lane_of(double v, int src) {  // the value of lane src
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * src, (int)(uint32_t)u);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * src, (int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int G>
__device__ __forceinline__ double row_sum(double v) {  // over G aligned lanes
    auto step = [&](unsigned long long o) { v += __builtin_bit_cast(double, (uint64_t)o); };
    auto bits = [&]() { return (unsigned long long)__builtin_bit_cast(uint64_t, v); };
    step(xshfl64<1>(bits()));
    step(xshfl64<2>(bits()));
    step(xshfl64<4>(bits()));
    if constexpr (G > 8) step(xshfl64<8>(bits()));
    if constexpr (G > 16) step(xshfl64<16>(bits()));
    if constexpr (G > 32) step(xshfl64<32>(bits()));
    return v;
}

// Values: WR rows of a kv head, as kv_write_kernel takes them.
template <int DT, int G, int WR>
__device__ __forceinline__ void append_values(const Append& a, unsigned block, Elem<DT>* lv) {
    using E = Elem<DT>;
    constexpr bool I8 = DT == FRQ_DT_ROWI8;
    constexpr int RP = 256 / G < WR ? 256 / G : WR, NP = WR / RP;
    constexpr int LP = lds_row<E>();
    __shared__ Places<WR> at;
    const Move& m = a.m;
    const int kvh = block % m.n_kv, hd = m.kv.hd, page = m.kv.page;
    const int64_t r0 = (int64_t)(block / m.n_kv) * WR;
    const int tid = threadIdx.x, c = 4 * (tid % G), pr = tid / G;
    const int64_t slot = tid < WR && r0 + tid < m.n ? m.slot[r0 + tid] : -1;
    const bool act = c < hd && pr < RP;
    const int64_t col = (int64_t)(a.n_head + m.n_kv + kvh) * hd + c;
    F4 y[NP], b{{0.0f, 0.0f, 0.0f, 0.0f}};
    if (act && a.bias) b = *reinterpret_cast<const F4*>(a.bias + col);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int64_t row = r0 + i * RP + pr;
        y[i] = act && row < m.n ? *reinterpret_cast<const F4*>(a.x + row * m.pitch + col) : F4{{0.0f, 0.0f, 0.0f, 0.0f}};
    }
    find_places(m, r0, slot, at);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = i * RP + pr;
        float vs = 0.0f;
        if (a.bias) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[i].v[j] += b.v[j];
        }
        if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) vs = fmaxf(vs, fabsf(y[i].v[j]));
            vs = fmaxf(row_max<G>(vs) / 127.0f, 1e-8f);
        }
        if (!act || at.pg[r] < 0) continue;
        const float vi = 1.0f / vs;  // int8
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (I8) lv[(c + j) * LP + r] = q8(y[i].v[j], vs, vi);
            else lv[(c + j) * LP + r] = (E)y[i].v[j];
        }
        if (I8 && c == 0)
            const_cast<float*>(m.kv.vs)[at.pg[r] * m.kv.sstride + kvh * page + at.off[r]] = vs;
    }
    __syncthreads();
    store_values<E, WR>(m, kvh, at, lv);
}

// Workgroups of values, then of queries and keys: some rows and heads, four heads
// a lane in flight, the rows' turns in LDS.  Bound by memory for long prompts: 8192
// rows of 36 heads of 128 channels, int8 pages, 277 MB in 66 us (4.2 TB/s); 8 rows
// a workgroup 76, 4 70, 1 68; two heads in flight 77 at 8 rows.  A step's few rows
// are bound by latency: one f16 row of 18 heads of 64 3.0 us, 61 f32 rows of 25 of 80 3.7.
constexpr int MAX_ROWS = 2;  // a workgroup's, of queries and keys
template <int DT, int G, int WR>
__global__ __launch_bounds__(256) void kv_append_kernel(const Append a) {
    using E = Elem<DT>;
    constexpr bool I8 = DT == FRQ_DT_ROWI8;
    constexpr int TURNS = MAX_ROWS * 2 * G * sizeof(double2), VALUES = 4 * G * lds_row<E>() * sizeof(E);
    __shared__ __align__(16) char lds[TURNS > VALUES ? TURNS : VALUES];
    if (blockIdx.x < a.value_groups) {
        append_values<DT, G, WR>(a, blockIdx.x, reinterpret_cast<E*>(lds));
        return;
    }
    const Move& m = a.m;
    double2* turn = reinterpret_cast<double2*>(lds);  // [rows][half]
    const unsigned block = blockIdx.x - a.value_groups;
    const int hd = m.kv.hd, page = m.kv.page, half = a.half, tid = threadIdx.x, lane = tid & 63;
    const int64_t r0 = (int64_t)(block / a.slices) << a.rshift;
    const int u0 = (block % a.slices) * a.units, u1 = min(u0 + a.units, a.n_head + m.n_kv);
    const int items = (u1 - u0) << a.rshift, rmask = (1 << a.rshift) - 1;
    const int c = 4 * (tid % G), first = tid / G;
    const bool act = c < hd;
    constexpr int NB = 4, NG = 256 / G;  // heads a lane has in flight, heads a pass
    F4 x[NB];
    auto load = [&](int p) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int it = p + i * NG + first;
            const int64_t row = r0 + (it & rmask);
            const bool in = act && it < items && row < m.n;
            x[i] = in ? *reinterpret_cast<const F4*>(a.x + row * m.pitch + (int64_t)(u0 + (it >> a.rshift)) * hd + c)
                      : F4{{0.0f, 0.0f, 0.0f, 0.0f}};
        }
    };
    load(0);
    for (int i = tid; i < half << a.rshift; i += 256) {
        const int r = i / half, j = i - r * half;
        turn[i] = r0 + r < m.n ? turn_of((double)a.pos[r0 + r] * a.freq[j]) : double2{1.0, 0.0};
    }
    __syncthreads();
    for (int p = 0; p < items; p += NB * NG) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (p + i * NG >= items) break;  // (of all lanes)
            const int it = p + i * NG + first, r = it & rmask, u = min(u0 + (it >> a.rshift), u1 - 1);
            const int64_t row = r0 + r;
            const bool in = act && it < items && row < m.n, key = u >= a.n_head;
            double y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = (double)x[i].v[j];
            if (a.bias && in) {
                const F4 b = *reinterpret_cast<const F4*>(a.bias + (int64_t)u * hd + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] += (double)b.v[j];
            }
            const float* gain = key ? a.kn : a.qn;
            if (a.qn || a.kn) {  // (the sum by all lanes: some may have other heads)
                double ss = 0.0;
#pragma unroll
                for (int j = 0; j < 4; ++j) ss = __builtin_fma(y[j], y[j], ss);
                ss = row_sum<G>(ss);
                if (gain && act) {
                    const F4 w = *reinterpret_cast<const F4*>(gain + c);
                    const double inv = 1.0 / sqrt(ss / (double)hd + a.eps);
#pragma unroll
                    for (int j = 0; j < 4; ++j) y[j] = y[j] * inv * (double)w.v[j];
                }
            }
            if (half) {
                const double2* cs = turn + r * half;
                if (a.pairs) {
                    if (c < 2 * half) {
#pragma unroll
                        for (int j = 0; j < 4; j += 2) {
                            const double2 t = cs[c / 2 + j / 2];
                            const double s = y[j], o = y[j + 1];
                            y[j] = s * t.x - o * t.y;
                            y[j + 1] = o * t.x + s * t.y;
                        }
                    }
                } else {
                    const bool low = c < half, high = !low && c < 2 * half;
                    const int src = low ? lane + half / 4 : high ? lane - half / 4 : lane;
                    double o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = lane_of(y[j], src);
                    if (low || high) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const double2 t = cs[(low ? c : c - half) + j];
                            y[j] = y[j] * t.x + (low ? -o[j] : o[j]) * t.y;
                        }
                    }
                }
            }
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = (float)y[j];
            float ks = 0.0f;
            if constexpr (I8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) ks = fmaxf(ks, fabsf(act ? f[j] : 0.0f));
                ks = fmaxf(row_max<G>(ks) / 127.0f, 1e-8f);
            }
            if (!in) continue;
            if (!key) {
                *reinterpret_cast<F4*>(a.q + row * a.q_pitch + (int64_t)u * hd + c) = F4{{f[0], f[1], f[2], f[3]}};
                continue;
            }
            int64_t pg;
            int off;
            if (!slot_of(m.slot[row], m.shift, m.kv.n_pages, &pg, &off)) continue;  // reported with the values
            const int kvh = u - a.n_head;
            const float ki = 1.0f / ks;  // int8
            Quad<E> k4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (I8) k4.v[j] = q8(f[j], ks, ki);
                else k4.v[j] = (E)f[j];
            }
            E* dk = reinterpret_cast<E*>(const_cast<char*>(m.kv.k) + pg * m.kv.stride) + ((int64_t)kvh * page + off) * hd;
            *reinterpret_cast<Quad<E>*>(dk + c) = k4;
            if (I8 && c == 0) const_cast<float*>(m.kv.ks)[pg * m.kv.sstride + kvh * page + off] = ks;
        }
        if (p + NB * NG < items) load(p + NB * NG);
    }
}

template <int DT, int G, int WR>
void launch_append(Append& a, hipStream_t s) {
    // Rows and heads a workgroup: 2 rows with all heads, less where that leaves
    // the chip unfilled, down to one pass over a workgroup's lanes.
    constexpr int NG = 256 / G;
    const int all = a.n_head + a.m.n_kv;
    auto groups = [&]() { return ((a.m.n + (1 << a.rshift) - 1) >> a.rshift) * ((all + a.units - 1) / a.units); };
    a.rshift = 1;
    a.units = all;
    while (a.rshift && (groups() < 1024 || (int64_t)1 << a.rshift >= 2 * a.m.n)) --a.rshift;
    while (groups() < 1024 && a.units << a.rshift > NG && a.units > 1) a.units = (a.units + 1) / 2;
    a.slices = (all + a.units - 1) / a.units;
    a.value_groups = (unsigned)((a.m.n + WR - 1) / WR * a.m.n_kv);
    kv_append_kernel<DT, G, WR><<<dim3((unsigned)(a.value_groups + groups())), dim3(256), 0, s>>>(a);
}
template <int DT, int WR>
void launch_append_g(Append& a, hipStream_t s) {
    if (a.m.kv.hd <= 32) launch_append<DT, 8, WR>(a, s);
    else if (a.m.kv.hd <= 64) launch_append<DT, 16, WR>(a, s);
    else if (a.m.kv.hd <= 128) launch_append<DT, 32, WR>(a, s);
    else launch_append<DT, 64, WR>(a, s);
}
// The values' rows a workgroup: 32, or 8 where workgroups of 32 are few, by
// kv_write's rule.
template <int DT>
void launch_append_r(Append& a, hipStream_t s) {
    constexpr int64_t few = DT == FRQ_DT_F32 ? 128 : 256;
    if ((a.m.n + 31) / 32 * a.m.n_kv < few) launch_append_g<DT, 8>(a, s);
    else launch_append_g<DT, 32>(a, s);
}

}  // namespace
}  // namespace kv
}  // namespace frq

using namespace frq;
using namespace frq::kv;

extern "C" int frq_kv_append_dev(frq_ctx* ctx, const frq_kv* kv, const frq_rotary* how, const float* d_qkv, size_t pitch,
                                 size_t n_head, const int32_t* d_pos, const int64_t* d_slot, size_t n, float* d_q,
                                 size_t q_pitch) {
    Append a{};
    if (int rc = check(kv, &a.m.kv, &a.m.shift)) return rc;
    if (!how) return bad("null rotary");
    if (how->rot % 8 || how->rot > kv->hd) return bad("rot must be a multiple of 8 up to hd");
    if (how->pairs != 0 && how->pairs != 1) return bad("pairs must be 0 or 1");
    if (!(how->eps >= 0.0) || how->eps > 1e30) return bad("eps must be 0 or positive");
    if (!n_head || n_head % kv->n_kv || n_head / kv->n_kv > 65535) return bad("n_head must be a multiple of n_kv");
    const size_t wide = (n_head + 2 * kv->n_kv) * kv->hd;
    if (pitch < wide || q_pitch < n_head * kv->hd || pitch > ((size_t)1 << 40) || q_pitch > ((size_t)1 << 40))
        return bad("pitch is below the heads' width");
    // (many rows: a workgroup for every two, and for 32 of every kv head; a launch has
    // fewer than 2^32 threads)
    if (n > ((size_t)1 << 31) || n * (n_head + 2 * kv->n_kv) > 0x7FFFFFFF ||
        ((n + 1) / 2 + (n + 31) / 32 * kv->n_kv) * 256 > 0xFFFFFFFFull)
        return bad("too many rows");
    if (n && (!d_qkv || !d_q || !d_slot || (how->rot && (!d_pos || !how->freq)))) return bad("null pointer");
    if (!ctx) return bad("null context");
    if (!n) return FRQ_OK;
    Guard g(ctx_device(ctx));
    a.m.slot = d_slot;
    a.m.n = (int64_t)n;
    a.m.pitch = (int64_t)pitch;
    a.m.n_kv = (int)kv->n_kv;
    a.m.err = ctx_err(ctx);
    a.x = d_qkv;
    a.bias = how->bias;
    a.qn = how->q_norm;
    a.kn = how->k_norm;
    a.eps = how->eps;
    a.freq = how->freq;
    a.pos = d_pos;
    a.q = d_q;
    a.q_pitch = (int64_t)q_pitch;
    a.half = (int)how->rot / 2;
    a.pairs = how->pairs;
    a.n_head = (int)n_head;
    hipStream_t s = (hipStream_t)frq_get_stream(ctx);
    if (kv->dtype == FRQ_DT_F32) launch_append_r<FRQ_DT_F32>(a, s);
    else if (kv->dtype == FRQ_DT_F16) launch_append_r<FRQ_DT_F16>(a, s);
    else launch_append_r<FRQ_DT_ROWI8>(a, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? FRQ_OK : hip_bad(e, "launch kv_append");
}
