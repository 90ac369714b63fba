// kv_rows.h — rows on their way into and out of the paged cache: the int8 rule,
// the places of a workgroup's rows, the checks of a cache's descriptor.
#pragma once

#include "kv_attn.h"

namespace frq {
namespace kv {
namespace {

constexpr int MAX_HD = 256;

struct Move {
    Cache kv;
    const int64_t* slot;
    int64_t n, pitch;
    int n_kv, shift;
    float *k, *v;              // read
    const float *wk, *wv;      // write
    int* err;
};

template <int DT>
using Elem = std::conditional_t<DT == FRQ_DT_F32, float, std::conditional_t<DT == FRQ_DT_F16, _Float16, int8_t>>;
template <typename E>
struct __attribute__((packed, aligned(1))) Quad {  // four elements anywhere (global memory takes any alignment)
    E v[4];
};

// round(x / step) of a row's values, |x| <= 127 step: the quotient as a
// product with RN(1 / step) and one residual correction (Markstein; the
// IEEE quotient, while 1 / step is a normal number), or the IEEE divide.
__device__ __forceinline__ int8_t q8(float x, float step, float inv) {
    float q = x * inv;
    q = step < 1e37f ? __builtin_fmaf(__builtin_fmaf(-q, step, x), inv, q) : x / step;
    const float t = __builtin_truncf(q);
    const float r = __builtin_fabsf(q - t) >= 0.5f ? t + __builtin_copysignf(1.0f, q) : t;
    return q != q ? (int8_t)0 : (int8_t)(int)__builtin_amdgcn_fmed3f(r, -127.0f, 127.0f);
}

// The places of the workgroup's rows: page (or -1: no place) and offset; then
// which fours of rows lie side by side in a page.
template <int WR>
struct Places {
    int64_t pg[WR];
    int off[WR];
    int four[WR / 4];
};
template <int WR>
__device__ __forceinline__ void find_places(const Move& m, int64_t r0, int64_t slot, Places<WR>& p) {
    const int r = threadIdx.x;
    if (r < WR) {
        int64_t pg = -1;
        int off = 0;
        if (r0 + r < m.n && !slot_of(slot, m.shift, m.kv.n_pages, &pg, &off)) {
            pg = -1;
            if (slot >= 0) atomicOr(m.err, ERR_INDEX);  // below zero: a row without a place
        }
        p.pg[r] = pg;
        p.off[r] = off;
    }
    __syncthreads();
    if (r < WR / 4) {
        bool side = p.pg[4 * r] >= 0;
        for (int j = 1; j < 4; ++j) side &= p.pg[4 * r + j] == p.pg[4 * r] && p.off[4 * r + j] == p.off[4 * r] + j;
        p.four[r] = side;
    }
    __syncthreads();
}

// The largest of G lanes' values (G a power of two, the lanes aligned).
template <int G>
__device__ __forceinline__ float row_max(float v) {
    auto step = [&](uint32_t o) { v = fmaxf(v, __uint_as_float(o)); };
    step(xshfl<1>(__float_as_uint(v)));
    step(xshfl<2>(__float_as_uint(v)));
    step(xshfl<4>(__float_as_uint(v)));
    if constexpr (G > 8) step(xshfl<8>(__float_as_uint(v)));
    if constexpr (G > 16) step(xshfl<16>(__float_as_uint(v)));
    if constexpr (G > 32) step(xshfl<32>(__float_as_uint(v)));
    return v;
}

// Elements of a channel's LDS row: fours word-aligned, and channels 4 apart (a
// wave's neighbouring lanes) 4 banks on (33 words, 17, 9).
template <typename E>
constexpr int lds_row() { return sizeof(E) == 4 ? 33 : sizeof(E) == 2 ? 34 : 36; }
template <typename E>
__device__ __forceinline__ Quad<E> from_lds(const E* p) {
    uint32_t w[sizeof(E)];
#pragma unroll
    for (unsigned i = 0; i < sizeof(E); ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    Quad<E> q;
    __builtin_memcpy(&q, w, sizeof(q));
    return q;
}
template <typename E>
__device__ __forceinline__ void to_lds(E* p, const Quad<E>& q) {
    uint32_t w[sizeof(E)];
    __builtin_memcpy(w, &q, sizeof(q));
#pragma unroll
    for (unsigned i = 0; i < sizeof(E); ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
}

// Values of WR rows from LDS (channel rows lv) into their pages: four tokens of
// a channel at a time where the rows lie side by side.
template <typename E, int WR>
__device__ __forceinline__ void store_values(const Move& m, int kvh, const Places<WR>& at, const E* lv) {
    constexpr int LP = lds_row<E>();
    const int hd = m.kv.hd, page = m.kv.page, tid = threadIdx.x;
    const int f = tid % (WR / 4);
    if (at.four[f]) {
        E* dv = reinterpret_cast<E*>(const_cast<char*>(m.kv.v) + at.pg[4 * f] * m.kv.stride) + (int64_t)kvh * hd * page +
                at.off[4 * f];
        for (int ch = tid / (WR / 4); ch < hd; ch += 256 / (WR / 4))
            *reinterpret_cast<Quad<E>*>(dv + (int64_t)ch * page) = from_lds(lv + ch * LP + 4 * f);
    } else {
        E* dv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            dv[j] = at.pg[4 * f + j] < 0 ? nullptr
                                         : reinterpret_cast<E*>(const_cast<char*>(m.kv.v) + at.pg[4 * f + j] * m.kv.stride) +
                                               (int64_t)kvh * hd * page + at.off[4 * f + j];
        for (int ch = tid / (WR / 4); ch < hd; ch += 256 / (WR / 4))
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (dv[j]) dv[j][(int64_t)ch * page] = lv[ch * LP + 4 * f + j];
    }
}

struct Guard {
    int prev = -1;
    explicit Guard(int d) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != d) (void)hipSetDevice(d);
    }
    ~Guard() {
        if (prev >= 0) (void)hipSetDevice(prev);
    }
};

int bad(const char* msg) { return set_error(FRQ_ERR_ARG, msg); }
int hip_bad(hipError_t e, const char* what) {
    return set_error(FRQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

size_t elem_size(int dtype) {
    return dtype == FRQ_DT_F32 ? 4 : dtype == FRQ_DT_F16 ? 2 : dtype == FRQ_DT_ROWI8 ? 1 : 0;
}

// The descriptor's own checks, before any device work.
int check(const frq_kv* h, Cache* kv, int* shift) {
    if (!h) return bad("null cache");
    const size_t sz = elem_size(h->dtype);
    if (!sz) return set_error(FRQ_ERR_DTYPE, "cache dtype must be f32, f16 or rowi8");
    if (!h->n_pages || h->n_pages > 0x7FFFFFFF) return bad("cache: n_pages must be in [1, 2^31)");
    if (h->page < 16 || h->page > 1024 || (h->page & (h->page - 1))) return bad("cache: page must be 16, 32, .. or 1024");
    if (!h->n_kv || h->n_kv > 65535) return bad("cache: n_kv must be in [1, 65535]");
    if (h->hd < 16 || h->hd > MAX_HD || h->hd % 16) return bad("cache: hd must be a multiple of 16 up to 256");
    if (!h->k || !h->v) return bad("cache: null pages");
    const bool i8 = h->dtype == FRQ_DT_ROWI8;
    if (i8 && (!h->k_scale || !h->v_scale)) return bad("cache: an int8 cache needs k_scale and v_scale");
    const size_t dense = h->n_kv * h->page * h->hd, sdense = h->n_kv * h->page;
    const size_t stride = h->page_stride ? h->page_stride : dense;
    const size_t sstride = h->scale_stride ? h->scale_stride : sdense;
    if (stride < dense || stride > ((size_t)1 << 40) || (i8 && (sstride < sdense || sstride > ((size_t)1 << 40))))
        return bad("cache: pages overlap (stride below a page's values)");
    if (((uintptr_t)h->k | (uintptr_t)h->v | (stride * sz)) & 15) return bad("cache: pages must be 16-byte aligned");
    if (i8 && ((((uintptr_t)h->k_scale | (uintptr_t)h->v_scale) & 15) || sstride % 4))
        return bad("cache: scales must be 16-byte aligned");
    kv->k = (const char*)h->k;
    kv->v = (const char*)h->v;
    kv->ks = h->k_scale;
    kv->vs = h->v_scale;
    kv->stride = (int64_t)(stride * sz);
    kv->sstride = (int64_t)sstride;
    kv->n_pages = (int64_t)h->n_pages;
    kv->page = (int)h->page;
    kv->hd = (int)h->hd;
    *shift = __builtin_ctzll(h->page);
    return FRQ_OK;
}

int check_rows(const frq_kv* h, const void* k, const void* v, size_t pitch, const int64_t* slot, size_t n, Move* m) {
    if (int rc = check(h, &m->kv, &m->shift)) return rc;
    if (n && (!k || !v || !slot)) return bad("null pointer");
    if (pitch < h->n_kv * h->hd || pitch > ((size_t)1 << 40)) return bad("pitch is below the kv heads' width");
    if (n > ((size_t)1 << 31) || (n + 31) / 32 * h->n_kv > 0x7FFFFFFF) return bad("too many rows");
    m->slot = slot;
    m->n = (int64_t)n;
    m->pitch = (int64_t)pitch;
    m->n_kv = (int)h->n_kv;
    return FRQ_OK;
}

}  // namespace
}  // namespace kv
}  // namespace frq
