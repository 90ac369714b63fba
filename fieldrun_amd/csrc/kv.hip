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

constexpr int WR = 32;   // rows a workgroup of the write and read kernels
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

__device__ __forceinline__ int8_t q8(float x, float step) {
    const float r = roundf(x / step);
    return r != r ? (int8_t)0 : (int8_t)fminf(fmaxf(r, -127.0f), 127.0f);
}

// The places of the workgroup's rows: page (or -1: no place) and offset.
__device__ __forceinline__ void places(const Move& m, int64_t r0, int64_t* pg, int* off) {
    if (threadIdx.x < WR) {
        int64_t p = -1;
        int o = 0;
        if (r0 + threadIdx.x < m.n) {
            const int64_t s = m.slot[r0 + threadIdx.x];
            if (!slot_of(s, m.shift, m.kv.n_pages, &p, &o)) {
                p = -1;
                if (s >= 0) atomicOr(m.err, ERR_INDEX);  // below zero: a row without a place
            }
        }
        pg[threadIdx.x] = p;
        off[threadIdx.x] = o;
    }
    __syncthreads();
}

// Workgroup (WR rows, kv head).  A wave takes a row at a time: its keys go
// straight to the page, its values to LDS and from there token by token
// along each channel, so that neighbouring slots make whole segments.
template <int DT>
__global__ __launch_bounds__(256) void kv_write_kernel(const Move m) {
    using E = Elem<DT>;
    extern __shared__ char lds_raw[];
    E* lv = reinterpret_cast<E*>(lds_raw);  // [hd][WR + pad]
    constexpr int LP = WR + 4 / sizeof(E);
    __shared__ int64_t pg[WR];
    __shared__ int off[WR];
    const int kvh = blockIdx.x % m.n_kv, hd = m.kv.hd, page = m.kv.page;
    const int64_t r0 = (int64_t)(blockIdx.x / m.n_kv) * WR;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    places(m, r0, pg, off);
    for (int r = wave; r < WR; r += 4) {
        if (pg[r] < 0) continue;
        const float* sk = m.wk + (r0 + r) * m.pitch + (int64_t)kvh * hd;
        const float* sv = m.wv + (r0 + r) * m.pitch + (int64_t)kvh * hd;
        E* dk = reinterpret_cast<E*>(const_cast<char*>(m.kv.k) + pg[r] * m.kv.stride) + ((int64_t)kvh * page + off[r]) * hd;
        float x[MAX_HD / 64], y[MAX_HD / 64];
#pragma unroll
        for (int i = 0; i < MAX_HD / 64; ++i) {
            const int c = lane + 64 * i;
            x[i] = c < hd ? sk[c] : 0.0f;
            y[i] = c < hd ? sv[c] : 0.0f;
        }
        float ks = 0.0f, vs = 0.0f;
        if constexpr (DT == FRQ_DT_ROWI8) {
            float mk = 0.0f, mv = 0.0f;
#pragma unroll
            for (int i = 0; i < MAX_HD / 64; ++i) {
                mk = fmaxf(mk, fabsf(x[i]));
                mv = fmaxf(mv, fabsf(y[i]));
            }
#pragma unroll
            for (int d = 32; d; d >>= 1) {
                mk = fmaxf(mk, __shfl_xor(mk, d, 64));
                mv = fmaxf(mv, __shfl_xor(mv, d, 64));
            }
            ks = fmaxf(mk / 127.0f, 1e-8f);
            vs = fmaxf(mv / 127.0f, 1e-8f);
            if (lane == 0) {
                const int64_t at = pg[r] * m.kv.sstride + kvh * page + off[r];
                const_cast<float*>(m.kv.ks)[at] = ks;
                const_cast<float*>(m.kv.vs)[at] = vs;
            }
        }
#pragma unroll
        for (int i = 0; i < MAX_HD / 64; ++i) {
            const int c = lane + 64 * i;
            if (c >= hd) continue;
            if constexpr (DT == FRQ_DT_ROWI8) {
                dk[c] = q8(x[i], ks);
                lv[c * LP + r] = q8(y[i], vs);
            } else {
                dk[c] = (E)x[i];
                lv[c * LP + r] = (E)y[i];
            }
        }
    }
    __syncthreads();
    const int r = threadIdx.x % WR;
    if (pg[r] < 0) return;
    E* dv = reinterpret_cast<E*>(const_cast<char*>(m.kv.v) + pg[r] * m.kv.stride) + (int64_t)kvh * hd * page + off[r];
    for (int c = threadIdx.x / WR; c < hd; c += 256 / WR) dv[(int64_t)c * page] = lv[c * LP + r];
}

// The way back: keys by rows, values through LDS.
template <int DT>
__global__ __launch_bounds__(256) void kv_read_kernel(const Move m) {
    using E = Elem<DT>;
    extern __shared__ char lds_raw[];
    E* lv = reinterpret_cast<E*>(lds_raw);
    constexpr int LP = WR + 4 / sizeof(E);
    __shared__ int64_t pg[WR];
    __shared__ int off[WR];
    const int kvh = blockIdx.x % m.n_kv, hd = m.kv.hd, page = m.kv.page;
    const int64_t r0 = (int64_t)(blockIdx.x / m.n_kv) * WR;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    places(m, r0, pg, off);
    {
        const int r = threadIdx.x % WR;
        if (pg[r] >= 0) {
            const E* sv = reinterpret_cast<const E*>(m.kv.v + pg[r] * m.kv.stride) + (int64_t)kvh * hd * page + off[r];
            for (int c = threadIdx.x / WR; c < hd; c += 256 / WR) lv[c * LP + r] = sv[(int64_t)c * page];
        }
    }
    __syncthreads();
    for (int r = wave; r < WR; r += 4) {
        if (pg[r] < 0) continue;
        float* dk = m.k + (r0 + r) * m.pitch + (int64_t)kvh * hd;
        float* dv = m.v + (r0 + r) * m.pitch + (int64_t)kvh * hd;
        const E* sk = reinterpret_cast<const E*>(m.kv.k + pg[r] * m.kv.stride) + ((int64_t)kvh * page + off[r]) * hd;
        float ks = 1.0f, vs = 1.0f;
        if constexpr (DT == FRQ_DT_ROWI8) {
            const int64_t at = pg[r] * m.kv.sstride + kvh * page + off[r];
            ks = m.kv.ks[at];
            vs = m.kv.vs[at];
        }
        for (int c = lane; c < hd; c += 64) {
            float x = (float)sk[c], y = (float)lv[c * LP + r];
            if constexpr (DT == FRQ_DT_ROWI8) {
                x *= ks;
                y *= vs;
            }
            dk[c] = x;
            dv[c] = y;
        }
    }
}

// The decode launch's tiles, then the prompt launch's (grid_b 0: none).
__global__ __launch_bounds__(256) void kv_join_kernel(const Args a, const Args b, unsigned grid_a) {
    __shared__ f4 so[256];
    __shared__ float sm[256], sl[256];
    if (blockIdx.x < grid_a) join_item<16>(a, blockIdx.x, so, sm, sl);
    else join_item<128>(b, blockIdx.x - grid_a, so, sm, sl);
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
    if (n > ((size_t)1 << 31) || (n + WR - 1) / WR * h->n_kv > 0x7FFFFFFF) return bad("too many rows");
    m->slot = slot;
    m->n = (int64_t)n;
    m->pitch = (int64_t)pitch;
    m->n_kv = (int)h->n_kv;
    return FRQ_OK;
}

template <bool WRITE>
hipError_t launch_move(const Move& m, int dtype, hipStream_t s) {
    const dim3 g((unsigned)((m.n + WR - 1) / WR * m.n_kv)), b(256);
    const size_t sz = elem_size(dtype), lds = (size_t)m.kv.hd * (WR * sz + 4);
#define KV_MOVE(DT)                                              \
    if (WRITE) kv_write_kernel<DT><<<g, b, lds, s>>>(m);         \
    else kv_read_kernel<DT><<<g, b, lds, s>>>(m)
    if (dtype == FRQ_DT_F32) { KV_MOVE(FRQ_DT_F32); }
    else if (dtype == FRQ_DT_F16) { KV_MOVE(FRQ_DT_F16); }
    else { KV_MOVE(FRQ_DT_ROWI8); }
#undef KV_MOVE
    return hipGetLastError();
}

constexpr int64_t DEC_TARGET = 1024;    // decode items wanted: two rounds of the chip's workgroups
constexpr int64_t PROMPT_TARGET = 400;  // prompt items wanted: a round and not quite two a CU
constexpr int DEC_PAIRS = 64;           // a sequence of up to so many (row, head) pairs is the decode kernel's

// The work of an attention call, and its workspace: the items' records, the
// decode tiles' parts and, where a sequence may ask with several rows, the
// prompt tiles'.
struct Plan {
    Call dec, prompt;
    size_t rec_dec, rec_prompt, part_dec, part_prompt, bytes;  // offsets, the whole
};
Plan plan_of(const frq_kv* kv, size_t n_row, size_t n_head, size_t n_seq) {
    Plan p{};
    Call& c = p.dec;
    c.n_seq = (int)n_seq;
    c.n_row = (int)n_row;
    c.rep = (int)(n_head / kv->n_kv);
    c.n_kv = (int)kv->n_kv;
    c.min_chunk = 256;
    c.min_pairs = 1;
    c.max_pairs = 0x7FFFFFFF;
    c.tp = 16;
    c.target = DEC_TARGET;
    p.prompt = c;
    p.prompt.min_pairs = DEC_PAIRS + 1;
    p.prompt.tp = 128;
    p.prompt.target = n_row > n_seq ? PROMPT_TARGET : 1;  // no room for parts: every tile's keys in one run
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += round_up(bytes, 256);
        return r;
    };
    p.rec_dec = take((size_t)max_items(p.dec) * sizeof(Record));
    p.rec_prompt = take((size_t)max_items(p.prompt) * sizeof(Record));
    p.part_dec = take((size_t)max_slots(DEC_TARGET, c.n_kv) * c.n_kv * 16 * (kv->hd + 2) * 4);
    p.part_prompt = take(n_row > n_seq ? (size_t)max_slots(PROMPT_TARGET, c.n_kv) * c.n_kv * 128 * (kv->hd + 2) * 4 : 0);
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
    if (n_row > 0x7FFFFFFF || n_seq > 0x7FFFFFFF || n_row * (n_head / kv->n_kv) > 0x7FFFFFFF)
        return bad("too many rows or sequences");
    if (!d_first && n_row != n_seq) return bad("without row offsets every sequence has one row");
    const size_t width = n_head * kv->hd;
    if (q_pitch < width || out_pitch < width || q_pitch > ((size_t)1 << 40) || out_pitch > ((size_t)1 << 40))
        return bad("pitch is below the heads' width");
    if (pages_pitch > 0x7FFFFFFF || (pages_pitch << shift) > 0x7FFFFFFF) return bad("a table holds up to 2^31 - 1 tokens");
    if (window > 0x7FFFFFFF) window = 0;  // wider than any sequence
    if (!(scale - scale == 0.0) || !(cap >= 0.0) || cap > 1e30) return bad("scale must be finite, cap 0 or positive");
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
    a.cap = (float)cap;
    // Each sequence is served by the kernel of its number of pairs; one that
    // no sequence can be for is not launched.
    const bool prompts = d_first && kv->dtype != FRQ_DT_F32 && n_row * (size_t)a.c.rep > (size_t)DEC_PAIRS;
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
    b.rec = (Record*)(ws + plan.rec_prompt);
    b.part = (float*)(ws + plan.part_prompt);
    b.slots = n_row > n_seq ? max_slots(PROMPT_TARGET, a.c.n_kv) : 0;
    const int64_t ga = max_items(a.c) * a.c.n_kv, gb = prompts ? max_items(b.c) * b.c.n_kv : 0;
    if (ga + gb > 0x7FFFFFFF) return bad("too many rows or sequences");
    const Launch la{(unsigned)ga, s}, lb{(unsigned)gb, s};
    hipError_t e = kv->dtype == FRQ_DT_F32   ? launch_decode_f32(a, la)
                   : kv->dtype == FRQ_DT_F16 ? launch_decode_f16(a, la)
                                             : launch_decode_i8(a, la);
    if (e != hipSuccess) return hip_bad(e, "launch kv_decode");
    if (prompts) {
        e = kv->dtype == FRQ_DT_F16 ? launch_prompt_f16(b, lb) : launch_prompt_i8(b, lb);
        if (e != hipSuccess) return hip_bad(e, "launch kv_prompt");
    }
    kv_join_kernel<<<dim3((unsigned)(ga + gb)), dim3(256), 0, s>>>(a, b, (unsigned)ga);
    e = hipGetLastError();
    return e == hipSuccess ? FRQ_OK : hip_bad(e, "launch kv_join");
}

}  // extern "C"
