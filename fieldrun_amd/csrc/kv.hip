// kv.hip — the paged key / value cache: rows quantised as they are written,
// read back, and the entry points of the attention over it (kv_attn.h).
//
// A page holds `page` tokens of every kv head: keys (kv, page, hd), values
// (kv, hd, page) — a value channel's tokens adjacent, which is the operand
// order of the attention's second product — and for int8 an f32 step per
// token and head.  The int8 rule is the engines' cache quantiser
// (forward_block_q, /root/reference/src/gemma.rs:314-324): step = max(max|x| /
// 127, 1e-8), q = round(x / step) half away from zero, clamped to +-127, a NaN
// quotient 0.
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

// Workgroup (WR rows, kv head); G lanes a row (a power of two >= hd / 4), four
// channels a lane, every load issued up front.  Keys go straight to their
// page; values through LDS, and from there four tokens of a channel at a time
// where the rows lie side by side (a prompt's do).  Bound by memory for long
// prompts: 8192 rows of 4 heads of 128 channels into int8, 42 MB, in 15.9 us
// (2.7 TB/s: the values' pieces are 32 bytes), back in 9.2 (4.6 TB/s), into f16
// 13.2 and back 11.8 (50 MB), f32 15.0 and 13.8 (67 MB); one token, 2.9 us, by
// latency.  (A token at a time both ways 29.5 us against 25.1, calls included.)
template <int DT, int G, int WR>
__global__ __launch_bounds__(256) void kv_write_kernel(const Move m) {
    using E = Elem<DT>;
    constexpr bool I8 = DT == FRQ_DT_ROWI8;
    constexpr int RP = 256 / G < WR ? 256 / G : WR, NP = WR / RP;  // rows a pass, passes
    constexpr int LP = lds_row<E>();
    __shared__ __align__(16) E lv[4 * G * LP];
    __shared__ Places<WR> at;
    const int kvh = blockIdx.x % m.n_kv, hd = m.kv.hd, page = m.kv.page;
    const int64_t r0 = (int64_t)(blockIdx.x / m.n_kv) * WR;
    const int tid = threadIdx.x, c = 4 * (tid % G), pr = tid / G;
    const int64_t slot = tid < WR && r0 + tid < m.n ? m.slot[r0 + tid] : -1;
    const bool act = c < hd && pr < RP;
    F4 x[NP], y[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int64_t row = r0 + i * RP + pr;
        if (act && row < m.n) {
            x[i] = *reinterpret_cast<const F4*>(m.wk + row * m.pitch + (int64_t)kvh * hd + c);
            y[i] = *reinterpret_cast<const F4*>(m.wv + row * m.pitch + (int64_t)kvh * hd + c);
        } else {
            x[i] = y[i] = F4{{0.0f, 0.0f, 0.0f, 0.0f}};
        }
    }
    find_places(m, r0, slot, at);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = i * RP + pr;
        float ks = 0.0f, vs = 0.0f;
        if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ks = fmaxf(ks, fabsf(x[i].v[j]));
                vs = fmaxf(vs, fabsf(y[i].v[j]));
            }
            ks = row_max<G>(ks);
            vs = row_max<G>(vs);
            ks = fmaxf(ks / 127.0f, 1e-8f);
            vs = fmaxf(vs / 127.0f, 1e-8f);
        }
        if (!act || at.pg[r] < 0) continue;
        const float ki = 1.0f / ks, vi = 1.0f / vs;  // int8
        Quad<E> k4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (I8) {
                k4.v[j] = q8(x[i].v[j], ks, ki);
                lv[(c + j) * LP + r] = q8(y[i].v[j], vs, vi);
            } else {
                k4.v[j] = (E)x[i].v[j];
                lv[(c + j) * LP + r] = (E)y[i].v[j];
            }
        }
        const int64_t pg = at.pg[r];
        E* dk = reinterpret_cast<E*>(const_cast<char*>(m.kv.k) + pg * m.kv.stride) + ((int64_t)kvh * page + at.off[r]) * hd;
        *reinterpret_cast<Quad<E>*>(dk + c) = k4;
        if (I8 && c == 0) {
            const int64_t s = pg * m.kv.sstride + kvh * page + at.off[r];
            const_cast<float*>(m.kv.ks)[s] = ks;
            const_cast<float*>(m.kv.vs)[s] = vs;
        }
    }
    __syncthreads();
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

// The way back: keys by rows, values by fours of tokens into LDS and from
// there by rows.
template <int DT, int G, int WR>
__global__ __launch_bounds__(256) void kv_read_kernel(const Move m) {
    using E = Elem<DT>;
    constexpr bool I8 = DT == FRQ_DT_ROWI8;
    constexpr int RP = 256 / G < WR ? 256 / G : WR, NP = WR / RP;
    constexpr int LP = lds_row<E>();
    __shared__ __align__(16) E lv[4 * G * LP];
    __shared__ Places<WR> at;
    const int kvh = blockIdx.x % m.n_kv, hd = m.kv.hd, page = m.kv.page;
    const int64_t r0 = (int64_t)(blockIdx.x / m.n_kv) * WR;
    const int tid = threadIdx.x, c = 4 * (tid % G), pr = tid / G;
    find_places(m, r0, tid < WR && r0 + tid < m.n ? m.slot[r0 + tid] : -1, at);
    const bool act = c < hd && pr < RP;
    Quad<E> k4[NP];
    float ks[NP], vs[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = i * RP + pr;
        ks[i] = vs[i] = 1.0f;
        if (!act || at.pg[r] < 0) continue;
        const int64_t pg = at.pg[r];
        k4[i] = *reinterpret_cast<const Quad<E>*>(reinterpret_cast<const E*>(m.kv.k + pg * m.kv.stride) +
                                                  ((int64_t)kvh * page + at.off[r]) * hd + c);
        if constexpr (I8) {
            const int64_t s = pg * m.kv.sstride + kvh * page + at.off[r];
            ks[i] = m.kv.ks[s];
            vs[i] = m.kv.vs[s];
        }
    }
    const int f = tid % (WR / 4);
    if (at.four[f]) {
        const E* sv = reinterpret_cast<const E*>(m.kv.v + at.pg[4 * f] * m.kv.stride) + (int64_t)kvh * hd * page + at.off[4 * f];
#pragma unroll 4
        for (int ch = tid / (WR / 4); ch < hd; ch += 256 / (WR / 4))
            to_lds(lv + ch * LP + 4 * f, *reinterpret_cast<const Quad<E>*>(sv + (int64_t)ch * page));
    } else {
        // (rows without a place read the first page and are not kept)
        const E* sv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            sv[j] = reinterpret_cast<const E*>(m.kv.v + max(at.pg[4 * f + j], (int64_t)0) * m.kv.stride) +
                    (int64_t)kvh * hd * page + at.off[4 * f + j];
#pragma unroll 2
        for (int ch = tid / (WR / 4); ch < hd; ch += 256 / (WR / 4)) {
            E t[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = sv[j][(int64_t)ch * page];
#pragma unroll
            for (int j = 0; j < 4; ++j) lv[ch * LP + 4 * f + j] = t[j];
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int r = i * RP + pr;
        if (!act || at.pg[r] < 0) continue;
        F4 x, y;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x.v[j] = (float)k4[i].v[j] * ks[i];
            y.v[j] = (float)lv[(c + j) * LP + r] * vs[i];
        }
        const int64_t d = (r0 + r) * m.pitch + (int64_t)kvh * hd + c;
        *reinterpret_cast<F4*>(m.k + d) = x;
        *reinterpret_cast<F4*>(m.v + d) = y;
    }
}

// The decode launch's tiles, then the prompt launch's (grid_b 0: none).
__global__ __launch_bounds__(256) void kv_join_kernel(const Args a, const Args b, unsigned grid_a) {
    __shared__ f4 so[256];
    __shared__ float sm[256], sl[256];
    if (blockIdx.x < grid_a) join_item<16>(a, blockIdx.x, so, sm, sl);
    else join_item<128>(b, blockIdx.x - grid_a, so, sm, sl);
}

// The plans of many sequences (workgroup 0: the decode launch's, 1: the
// prompt's): the call's keys, then the items and slots before each 64
// sequences.  16 waves, 64 sequences each at a time, bound by the latency of
// two passes over the lengths.
__global__ __launch_bounds__(1024) void kv_plan_kernel(const Call ca, const Call cb, int32_t* plan_a, int32_t* plan_b,
                                                       int* err) {
    __shared__ int64_t keys[16];
    const bool dec = blockIdx.x == 0;
    const Call c = dec ? ca : cb;
    int32_t* plan = dec ? plan_a : plan_b;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, blocks = (c.n_seq + 63) / 64;
    int64_t total = 0;
    for (int64_t s = threadIdx.x; s < c.n_seq; s += 1024) {
        const Seq q = seq_at(c, (int)s);
        total += keys_of(q);
        if (q.bad && dec) atomicOr(err, ERR_INDEX);
    }
    total = wave_total(total);
    if (lane == 0) keys[w] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) total += keys[i];
    const int klen = chunk_of(c, total);
    for (int b = w; b < blocks; b += 16) {
        Seq q{};
        if (b * 64 + lane < c.n_seq) q = seq_at(c, b * 64 + lane);
        const int n = q.tiles ? chunks_of(q, klen) : 1, mine = q.tiles * n;
        const int items = lane_sums(mine), slots = lane_sums(n > 1 ? mine : 0);
        if (lane == 63) {
            plan[2 + 2 * (int64_t)b] = items;
            plan[3 + 2 * (int64_t)b] = slots;
        }
    }
    __syncthreads();
    if (w) return;
    if (lane == 0) {
        plan[0] = klen;
        plan[1] = 0;
    }
    int items = 0, slots = 0;
    for (int b0 = 0; b0 < blocks; b0 += 64) {
        const bool in = b0 + lane < blocks;
        int32_t* at = plan + 2 + 2 * (int64_t)(b0 + lane);
        const int x = in ? at[0] : 0, y = in ? at[1] : 0;
        const int xs = lane_sums(x), ys = lane_sums(y);
        if (in) {
            at[0] = items + xs - x;
            at[1] = slots + ys - y;
        }
        items += lane_bcast(xs, 63);
        slots += lane_bcast(ys, 63);
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

// Rows a workgroup: 32, or 8 where workgroups of 32 leave the chip unfilled and
// the latency of one bounds the call (61 f32 rows of 5 heads of 80 written in
// 3.9 us against 5.0 and read in 3.8 against 5.1; there and back with the calls:
// 1500 int8 rows of 4 heads of 128, 188 workgroups of 32, 10.1 us against 14.1).
// More calls for 32: 1500 f32 rows of 5 heads of 256, 235 workgroups, 20.5 us
// against 23.0; 8192 int8 rows read in 9.6 against 13.8 (at 64, whole lines of
// int8 values, 11.2, and written in 19.4 against 16.6).
template <bool WRITE, int DT, int WR>
void launch_move_g(const Move& m, int64_t groups, hipStream_t s) {
    const dim3 g((unsigned)groups), b(256);
    auto go = [&](auto lanes) {
        constexpr int G = decltype(lanes)::value;
        if constexpr (WRITE) kv_write_kernel<DT, G, WR><<<g, b, 0, s>>>(m);
        else kv_read_kernel<DT, G, WR><<<g, b, 0, s>>>(m);
    };
    if (m.kv.hd <= 32) go(std::integral_constant<int, 8>{});
    else if (m.kv.hd <= 64) go(std::integral_constant<int, 16>{});
    else if (m.kv.hd <= 128) go(std::integral_constant<int, 32>{});
    else go(std::integral_constant<int, 64>{});
}
template <bool WRITE, int DT>
void launch_move_r(const Move& m, hipStream_t s) {
    const int64_t groups = (m.n + 31) / 32 * m.n_kv;
    constexpr int64_t few = DT == FRQ_DT_F32 ? 128 : 256;
    if (groups < few) launch_move_g<WRITE, DT, 8>(m, (m.n + 7) / 8 * m.n_kv, s);
    else launch_move_g<WRITE, DT, 32>(m, groups, s);
}
template <bool WRITE>
hipError_t launch_move(const Move& m, int dtype, hipStream_t s) {
    if (dtype == FRQ_DT_F32) launch_move_r<WRITE, FRQ_DT_F32>(m, s);
    else if (dtype == FRQ_DT_F16) launch_move_r<WRITE, FRQ_DT_F16>(m, s);
    else launch_move_r<WRITE, FRQ_DT_ROWI8>(m, s);
    return hipGetLastError();
}

// Decode items wanted: the chip's workgroups at two a CU (256, 512, 768, 1024:
// 48 int8 sequences of up to 6001 tokens 65, 47, 55, 56 us; one of 131071 f16
// 103, 109, 115, 109; 16 f32 windows of 4096 164, 124, 123, 133).
constexpr int64_t DEC_TARGET = 512;
// Prompt items wanted: a round and not quite two a CU; more cost the joining
// more than the balance gives (400, 640, 1024, 1536: kernel and join of 7 ragged
// int8 prompts 123 + 8, 127 + 18, 110 + 24, 108 + 24 us; of 2048 rows over 8192
// keys 503 + 5 at 400, 486 + 25 at 1024).  Where one workgroup fills a CU (over
// 128 channels) less than a round: 189 rows of 32 heads of 256 over 2611 int8
// keys 135 us at 400, 92 at 240.
constexpr int64_t PROMPT_TARGET = 400, PROMPT_TARGET_WIDE = 240;
// A sequence of up to so many (row, head) pairs is the decode kernel's (decode
// against prompt kernel: 126 pairs over 1000 tokens 14.4, 31.3 us, over 8192
// 27.9, 35.7, 8 times over 2000 45.5, 39.2; 252 pairs over 1000 15.2, 31.7, but
// 8 times over 2000 71, 49.5).
constexpr int DEC_PAIRS = 128;

// The work of an attention call, and its workspace: the items' records, the
// decode tiles' parts, where a sequence may ask with several rows the prompt
// tiles', and for many sequences both launches' plans.
struct Plan {
    Call dec, prompt;
    size_t rec_dec, rec_prompt, part_dec, part_prompt, plan_dec, plan_prompt, bytes;  // offsets, the whole
};
Plan plan_of(const frq_kv* kv, size_t n_row, size_t n_head, size_t n_seq) {
    Plan p{};
    Call& c = p.dec;
    c.n_seq = (int)n_seq;
    c.n_row = (int)n_row;
    c.rep = (int)(n_head / kv->n_kv);
    c.n_kv = (int)kv->n_kv;
    // Two tiles a wave at least; prompts two or four a workgroup (256 instead: one
    // f32 sequence of 959 tokens, 15 heads of 256, 27 us against 21; 108 f32 rows
    // of 16 heads of 64 over 400 tokens 33 against 25.  f16 at 128: 113 sequences of
    // up to 579 tokens 31 us against 26; prompts at 64: 4 sequences of 166 rows
    // with a window of 8 42 us against 23).
    c.min_chunk = kv->dtype == FRQ_DT_F32 ? 128 : 256;
    c.min_pairs = 1;
    c.max_pairs = 0x7FFFFFFF;
    c.tp = 16;
    c.target = DEC_TARGET;
    p.prompt = c;
    p.prompt.min_pairs = DEC_PAIRS + 1;
    p.prompt.tp = 128;
    // (n_row <= n_seq: no room for parts, every tile's keys in one run)
    p.prompt.target = n_row <= n_seq ? 1 : kv->hd > 128 ? PROMPT_TARGET_WIDE : PROMPT_TARGET;
    p.prompt.min_chunk = 128;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += round_up(bytes, 256);
        return r;
    };
    p.rec_dec = take((size_t)max_items(p.dec) * sizeof(Record));
    p.rec_prompt = take((size_t)max_items(p.prompt) * sizeof(Record));
    p.part_dec = take((size_t)max_slots(DEC_TARGET, c.n_kv) * c.n_kv * 16 * (kv->hd + 2) * 4);
    p.part_prompt = take(n_row > n_seq ? (size_t)max_slots(p.prompt.target, c.n_kv) * c.n_kv * 128 * (kv->hd + 2) * 4 : 0);
    p.plan_dec = take((size_t)plan_words(c.n_seq) * 4);
    p.plan_prompt = take((size_t)plan_words(c.n_seq) * 4);
    p.bytes = at;
    return p;
}

}  // namespace
}  // namespace kv
}  // namespace frq

using namespace frq;
using namespace frq::kv;

extern "C" {

int frq_kv_write_dev(frq_ctx* ctx, const frq_kv* kv, const float* d_k, const float* d_v, size_t pitch,
                     const int64_t* d_slot, size_t n) {
    Move m{};
    if (int rc = check_rows(kv, d_k, d_v, pitch, d_slot, n, &m)) return rc;
    if (!ctx) return bad("null context");
    if (!n) return FRQ_OK;
    Guard g(ctx_device(ctx));
    m.wk = d_k;
    m.wv = d_v;
    m.err = ctx_err(ctx);
    const hipError_t e = launch_move<true>(m, kv->dtype, (hipStream_t)frq_get_stream(ctx));
    return e == hipSuccess ? FRQ_OK : hip_bad(e, "launch kv_write");
}

int frq_kv_read_dev(frq_ctx* ctx, const frq_kv* kv, const int64_t* d_slot, size_t n, float* d_k, float* d_v,
                    size_t pitch) {
    Move m{};
    if (int rc = check_rows(kv, d_k, d_v, pitch, d_slot, n, &m)) return rc;
    if (!ctx) return bad("null context");
    if (!n) return FRQ_OK;
    Guard g(ctx_device(ctx));
    m.k = d_k;
    m.v = d_v;
    m.err = ctx_err(ctx);
    const hipError_t e = launch_move<false>(m, kv->dtype, (hipStream_t)frq_get_stream(ctx));
    return e == hipSuccess ? FRQ_OK : hip_bad(e, "launch kv_read");
}

size_t frq_kv_attn_ws(const frq_kv* kv, size_t n_row, size_t n_head, size_t n_seq, size_t pages_pitch) {
    (void)pages_pitch;
    if (!kv || !kv->n_kv || kv->n_kv > 65535 || kv->hd > MAX_HD || !n_head || n_head % kv->n_kv ||
        n_head / kv->n_kv > 65535 || n_row > 0x7FFFFFFF || n_seq > 0x7FFFFFFF)
        return 0;
    return plan_of(kv, n_row, n_head, n_seq).bytes;
}

int frq_kv_attn_dev(frq_ctx* ctx, const frq_kv* kv, const float* d_q, size_t q_pitch, size_t n_row, size_t n_head,
                    const int32_t* d_pages, size_t pages_pitch, const int32_t* d_len, const int32_t* d_first,
                    size_t n_seq, double scale, double cap, size_t window, float* d_out, size_t out_pitch, void* d_ws,
                    size_t ws_bytes) {
    Args a{};
    int shift = 0;
    if (int rc = check(kv, &a.kv, &shift)) return rc;
    if (!n_head || n_head % kv->n_kv || n_head / kv->n_kv > 65535) return bad("n_head must be a multiple of n_kv");
    // (sequences are counted in 64s: room for 63 more)
    if (n_row > 0x7FFFFFFF || n_seq > 0x7FFFFFFF - 63 || n_row * (n_head / kv->n_kv) > 0x7FFFFFFF)
        return bad("too many rows or sequences");
    if (!d_first && n_row != n_seq) return bad("without row offsets every sequence has one row");
    const size_t width = n_head * kv->hd;
    if (q_pitch < width || out_pitch < width || q_pitch > ((size_t)1 << 40) || out_pitch > ((size_t)1 << 40))
        return bad("pitch is below the heads' width");
    // (keys past a sequence's last are counted to the end of a tile: room below 2^31)
    if (pages_pitch > 0x7FFFFFFF || (pages_pitch << shift) > 0x7FFFFFFF - 1024)
        return bad("a table holds up to 2^31 - 1024 tokens");
    if (window > 0x7FFFFFFF) window = 0;  // wider than any sequence
    if (!(scale >= -1e30 && scale <= 1e30) || !(cap >= 0.0 && cap <= 1e30))
        return bad("scale must be within 1e30, cap 0 or positive");
    if (n_row && n_seq && (!d_q || !d_out || !d_len || (!d_pages && pages_pitch))) return bad("null pointer");
    if (d_ws && ((uintptr_t)d_ws & 15)) return bad("the workspace must be 16-byte aligned");
    if (!ctx) return bad("null context");
    if (!n_row || !n_seq) return FRQ_OK;
    const Plan plan = plan_of(kv, n_row, n_head, n_seq);
    const size_t need = plan.bytes;
    if (d_ws && ws_bytes < need) return bad("the workspace is below frq_kv_attn_ws");
    Guard g(ctx_device(ctx));
    hipStream_t s = (hipStream_t)frq_get_stream(ctx);
    if (!d_ws) {
        // the context's workspace may move with a later call: a graph would
        // keep its old address
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        const hipError_t e = hipStreamIsCapturing(s, &st);
        if (e != hipSuccess) return hip_bad(e, "hipStreamIsCapturing");
        if (st != hipStreamCaptureStatusNone) return bad("under graph capture the caller gives the workspace");
        if (int rc = ctx_ws(ctx, need, &d_ws)) return rc;
    }
    a.c = plan.dec;
    a.c.len = d_len;
    a.c.first = d_first;
    a.c.width = (int)pages_pitch;
    a.c.shift = shift;
    a.c.window = (int)window;
    a.q = d_q;
    a.q_pitch = (int64_t)q_pitch;
    a.out_pitch = (int64_t)out_pitch;
    a.pages_pitch = (int64_t)pages_pitch;
    a.pages = d_pages;
    a.out = d_out;
    a.err = ctx_err(ctx);
    a.scale = scale == 0.0 ? 1.0f : (float)(scale < 0.0 ? -scale : scale);
    a.sign = scale == 0.0 ? 0.0f : scale < 0.0 ? -1.0f : 1.0f;
    // (below 2^-27 every cap gives weights within a rounding of equal ones; there
    // score_scale's 2^100 over the cap would leave f32, or the cap be zero in it)
    a.cap = cap > 0.0 && cap < 7.450580596923828e-9 ? 7.450580596923828e-9f : (float)cap;
    a.dtype = kv->dtype;
    // Each sequence is served by the kernel of its number of pairs; one that
    // no sequence can be for is not launched.
    // (f32 keys of over 128 channels stay with the decode kernel: three parts of
    // q leave the prompt kernel one wave a SIMD.  2048 rows of 8 heads over 4, the
    // decode kernel against the prompt kernel: 256 channels 288, 340 us over
    // themselves, 72, 78 at 600 rows, 1612, 1508 over 8192 tokens; 192 channels 225,
    // 202 and 1280, 676.  Widths of an odd number of 32s do not fit the LDS.)
    const bool prompts = d_first && n_row * (size_t)a.c.rep > (size_t)DEC_PAIRS &&
                         !(kv->dtype == FRQ_DT_F32 && kv->hd > 128);
    a.c.max_pairs = prompts ? DEC_PAIRS : 0x7FFFFFFF;
    char* ws = (char*)d_ws;
    a.rec = (Record*)(ws + plan.rec_dec);
    a.part = (float*)(ws + plan.part_dec);
    a.slots = max_slots(DEC_TARGET, a.c.n_kv);
    Args b = a;
    b.c.min_pairs = plan.prompt.min_pairs;
    b.c.max_pairs = plan.prompt.max_pairs;
    b.c.tp = plan.prompt.tp;
    b.c.target = plan.prompt.target;
    b.c.min_chunk = plan.prompt.min_chunk;
    b.rec = (Record*)(ws + plan.rec_prompt);
    b.part = (float*)(ws + plan.part_prompt);
    b.slots = n_row > n_seq ? max_slots(b.c.target, a.c.n_kv) : 0;
    const int64_t ga = max_items(a.c) * a.c.n_kv, gb = prompts ? max_items(b.c) * b.c.n_kv : 0;
    if (ga + gb > 0x7FFFFFFF) return bad("too many rows or sequences");
    const Launch la{(unsigned)ga, s}, lb{(unsigned)gb, s};
    hipError_t e = hipSuccess;
    if (n_seq > (size_t)PLAN_SEQS) {
        int32_t *pa = (int32_t*)(ws + plan.plan_dec), *pb = (int32_t*)(ws + plan.plan_prompt);
        kv_plan_kernel<<<dim3(prompts ? 2 : 1), dim3(1024), 0, s>>>(a.c, b.c, pa, pb, a.err);
        e = hipGetLastError();
        if (e != hipSuccess) return hip_bad(e, "launch kv_plan");
        a.c.plan = pa;
        b.c.plan = pb;
    }
    e = kv->dtype == FRQ_DT_F32   ? launch_decode_f32(a, la)
                   : kv->dtype == FRQ_DT_F16 ? launch_decode_f16(a, la)
                                             : launch_decode_i8(a, la);
    if (e != hipSuccess) return hip_bad(e, "launch kv_decode");
    if (prompts) {
        e = kv->dtype == FRQ_DT_F32   ? launch_prompt_f32(b, lb)
            : kv->dtype == FRQ_DT_F16 ? launch_prompt_f16(b, lb)
                                      : launch_prompt_i8(b, lb);
        if (e != hipSuccess) return hip_bad(e, "launch kv_prompt");
    }
    kv_join_kernel<<<dim3((unsigned)(ga + gb)), dim3(256), 0, s>>>(a, b, (unsigned)ga);
    e = hipGetLastError();
    return e == hipSuccess ? FRQ_OK : hip_bad(e, "launch kv_join");
}

}  // extern "C"
