// kv_attn.h — attention over a paged key / value cache (gfx950): the decode
// kernel, the joining of its parts, and what the prompt kernel shares with it.
//
//   z_j = scale q . k_j          (cap > 0: cap tanh(z_j / cap))
//   out = sum_j exp(z_j - m) v_j / sum_j exp(z_j - m)
// over the keys j that the row sees, in one pass with a running maximum m and
// sum; keys are cut into chunks over workgroups and the parts (m, sum, out)
// joined by a second launch.
//
// Both products run transposed on the matrix cores, so that a lane owns one
// (row, head) pair throughout: S^T = K Q^T (A: 16 key rows, B: 16 pairs) puts
// a pair's scores in lane % 16, where P^T is at once the B operand of
// O^T = V^T P^T and the running maximum, the sum and the rescaling of O are
// per lane.  A score tile's key rows are taken in the order that makes its
// results the next product's operand (lane group g of P^T holds keys
// 8 g .. 8 g + 7 of a 32-key tile: key row r of half u is key
// 8 (r / 4) + 4 u + r % 4), and the cache keeps the values of a page
// transposed (hd, page), so both operands are 16-byte loads straight from the
// pages and nothing goes through LDS.
//
// On the 16-bit matrix cores: the cache's f16 and int8 entries are exact f16;
// an f32 q row, scaled by a power of two to below 2, is the sum of two f16, 22
// bits of its larger entries and down to 2^-25 of the largest for all (f32 would
// hold more of a small entry that meets a large key's), likewise the
// probabilities (scaled by 2^11, so that what f16 cannot hold of them is below
// 2^-36 of the largest); the products of both halves add up in the f32
// accumulators.  An f32 cache uses the f32 matrix cores for decoding, where
// memory bounds the call, and three bf16 parts of both operands for prompts.
#pragma once

#include "frq_internal.h"
#include "kv_index.h"

namespace frq {
namespace kv {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
// f32 rows of the caller are 4-byte aligned
struct __attribute__((packed, aligned(4))) F4 {
    float v[4];
};

constexpr int ERR_INDEX = 2;  // error word: a page, slot, length or offset out of range

struct Cache {  // frq_kv as the kernels take it
    const char *k, *v;
    const float *ks, *vs;
    int64_t stride, sstride;  // bytes between pages, scales between pages
    int64_t n_pages;
    int page, hd;
};

// An item as the joining launch reads it (chunks 1: nothing to join; seq: its
// complement where a row sees a key under a page id out of range).
struct Record {
    int row0, rows, tile, chunk, chunks, slot, len, seq;
};
struct Args {
    Call c;
    Cache kv;
    const float* q;
    int64_t q_pitch, out_pitch, pages_pitch;
    const int32_t* pages;
    float* out;
    Record* rec;  // an item each
    float* part;  // slots of tp (hd + 2) floats a kv head: (m, sum) pairs, then out
    int64_t slots;
    int* err;
    float scale, sign, cap;  // |scale| and the sign that q takes (0: scale 1)
    int dtype;
};

// An item's place: its sequence, tile and chunk; every lane has the same.
struct Item {
    Seq q;
    int seq, tile, chunk, chunks, klen;
    int slot;  // the chunk 0 slot of this tile (chunks > 1)
    bool found;
};

__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
template <typename T>
__device__ __forceinline__ T lane_bcast(T v, int src) {
    if constexpr (sizeof(T) == 8) {
        const int lo = __builtin_amdgcn_readlane((int)(uint64_t)v, src);
        const int hi = __builtin_amdgcn_readlane((int)((uint64_t)v >> 32), src);
        return (T)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
    } else {
        return (T)__builtin_amdgcn_readlane((int)v, src);
    }
}

// Inclusive sums over the lanes (DPP: within rows of 16, then the rows' ends).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) {
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int lane_sums(int x) {
    x = dpp_add<0x111, 0xF>(x);
    x = dpp_add<0x112, 0xF>(x);
    x = dpp_add<0x114, 0xF>(x);
    x = dpp_add<0x118, 0xF>(x);
    x = dpp_add<0x142, 0xA>(x);
    return dpp_add<0x143, 0xC>(x);
}

__device__ __forceinline__ int64_t wave_total(int64_t v) {
    v += (int64_t)xshfl64<1>(v);
    v += (int64_t)xshfl64<2>(v);
    v += (int64_t)xshfl64<4>(v);
    v += (int64_t)xshfl64<8>(v);
    v += (int64_t)xshfl64<16>(v);
    return lane_bcast(v + (int64_t)xshfl64<32>(v), 0);
}

__device__ __forceinline__ float wave_sum(float v) {
    auto step = [&](uint32_t o) { v += __uint_as_float(o); };
    step(xshfl<1>(__float_as_uint(v)));
    step(xshfl<2>(__float_as_uint(v)));
    step(xshfl<4>(__float_as_uint(v)));
    step(xshfl<8>(__float_as_uint(v)));
    step(xshfl<16>(__float_as_uint(v)));
    step(xshfl<32>(__float_as_uint(v)));
    return v;
}

__device__ __forceinline__ int wave_most(int v) {
    v = max(v, (int)xshfl<1>(v));
    v = max(v, (int)xshfl<2>(v));
    v = max(v, (int)xshfl<4>(v));
    v = max(v, (int)xshfl<8>(v));
    v = max(v, (int)xshfl<16>(v));
    return uni(max(v, (int)xshfl<32>(v)));
}

// Finds item `id`, each wave by itself: up to 64 sequences from their lengths
// and offsets alone, first the call's keys (the chunk length), then the items
// before; more from the call's plan, which holds the chunk length and the
// items before each 64.  (A call with every workgroup summing them all, against
// the plan's launch: 41 / 43 us at 80 sequences of 1200 tokens, 35.3 / 34.2 at
// 128 of 800, 47.6 / 41.5 at 256 of 400, 1669 / 305 at 4096 of 100.)  Of each 64 those with chunks longer
// than half the longest come first, so that the last workgroups to start have
// the least to do; a sequence's last tiles come first, which see the most.
__device__ __forceinline__ Item find_item(const Call& c, int id, int* err) {
    const int lane = threadIdx.x & 63;
    Item it{};
    int s0 = 0, items = 0, slots = 0, klen;
    if (c.plan) {
        const int blocks = (c.n_seq + 63) / 64;
        klen = c.plan[0];
        for (int b0 = 0; b0 < blocks; b0 += 64) {
            const bool in = b0 + lane < blocks;
            const int64_t at = 2 + 2 * (int64_t)(in ? b0 + lane : 0);
            const int before = c.plan[at], slot = c.plan[at + 1];
            const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && before <= id));
            if (n) {
                s0 = 64 * (b0 + n - 1);
                items = lane_bcast(before, n - 1);
                slots = lane_bcast(slot, n - 1);
            }
            if (n < 64) break;
        }
    }
    Seq q{};
    if (s0 + lane < c.n_seq) q = seq_at(c, s0 + lane);
    if (!c.plan) {
        if (q.bad && id == 0 && threadIdx.x < 64) atomicOr(err, ERR_INDEX);
        const int64_t total = c.n_seq > 1 ? wave_total(keys_of(q)) : lane_bcast(keys_of(q), 0);
        klen = chunk_of(c, total);
    }
    const int n = q.tiles ? chunks_of(q, klen) : 1, own = even_chunk(q, n), mine = q.tiles * n;
    const int most = wave_most(own);
    const bool first = own > most / 2;
    const int parts = n > 1 ? mine : 0;
    const int a = lane_sums(first ? mine : 0), b = lane_sums(first ? 0 : mine);
    const int head = lane_bcast(a, 63);
    const int at = id - items - (first ? a : head + b) + mine;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(at >= 0 && at < mine);
    const int sums = lane_sums(parts);
    if (hit) {
        const int l = __builtin_ctzll(hit);
        it.seq = s0 + l;
        it.q.row0 = lane_bcast(q.row0, l);
        it.q.rows = lane_bcast(q.rows, l);
        it.q.len = lane_bcast(q.len, l);
        it.chunks = lane_bcast(n, l);
        it.klen = lane_bcast(own, l);
        const int i = lane_bcast(at, l), t = uni(i / it.chunks);
        it.tile = lane_bcast(q.tiles, l) - 1 - t;
        it.chunk = i - t * it.chunks;
        it.slot = slots + lane_bcast(sums, l) - lane_bcast(parts, l) + it.tile * it.chunks;
        it.found = true;
    }
    return it;
}

__device__ __forceinline__ void note_item(Record* r, int id, const Item& it) {
    if (threadIdx.x == 0)
        r[id] = Record{it.q.row0, it.q.rows, it.tile, it.chunk, it.found ? it.chunks : 1, it.slot, it.q.len, it.seq};
}

__device__ __forceinline__ void note_hole(const Args& a, int id, int seq) {
    if (threadIdx.x == 0) {
        atomicOr(a.err, ERR_INDEX);
        if (blockIdx.x % a.c.n_kv == 0) a.rec[id].seq = ~seq;  // as note_item; every kv head finds the same
    }
}

__device__ __forceinline__ float fmax16(float v) {  // over the four lane groups of a pair
    v = fmaxf(v, __uint_as_float(xshfl<16>(__float_as_uint(v))));
    return fmaxf(v, __uint_as_float(xshfl<32>(__float_as_uint(v))));
}
__device__ __forceinline__ float fsum16(float v) {
    v += __uint_as_float(xshfl<16>(__float_as_uint(v)));
    return v + __uint_as_float(xshfl<32>(__float_as_uint(v)));
}

// What out is multiplied by: a row that sees no key (its position below 0) is
// zeros, one whose scores are all -inf is NaN, as the formula has it.
__device__ __forceinline__ float over(float l, int pos) {
    return l > 0.0f || l != l ? 1.0f / l : pos < 0 ? 0.0f : __builtin_nanf("");
}

// The loops read page 0 for a page id out of range.  Such an id is an error
// where a row would see a key under it (pages are of 16 tokens and more, a tile
// begins at a multiple of 32: a page wholly before the window may be gone).
// Then the tile's results are formed anew behind the joining, without those
// keys: a chunk says so by this in the place of its sums.
constexpr float HOLE = -1.0f;
__device__ __forceinline__ bool page_bad(const Args& a, int seq, int lo, int hi) {
    const int32_t* table = a.pages + (int64_t)seq * a.pages_pitch;
    for (int pg = lo >> a.c.shift; lo <= hi && pg <= hi >> a.c.shift; ++pg)
        if (page_ok(table[pg], a.kv.n_pages) < 0) return true;
    return false;
}

// tanh to about 2e-7 of its value: a polynomial near zero, where
// (1 - t) / (1 + t) would cancel.
__device__ __forceinline__ float tanh_f(float x) {
    const float a = __builtin_fabsf(x), y = x * x;
    const float t = __builtin_amdgcn_exp2f(-2.8853900817779268f * a);
    const float big = (1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t);
    float p = __builtin_fmaf(y, 0.021869488536155203f, -0.05396825396825397f);
    p = __builtin_fmaf(y, p, 0.13333333333333333f);
    p = __builtin_fmaf(y, p, -0.3333333333333333f);
    const float small = __builtin_fmaf(a * y, p, a);
    return __builtin_copysignf(a < 0.3f ? small : big, x);
}

// int8 words -> eight exact f16: byte ^ 0x80 under the exponent of 1024 is
// 1024 + 128 + value.
__device__ __forceinline__ h8 i8_to_h8(u2 w) {
    h2 r[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t x = w[i] ^ 0x80808080u;
        r[2 * i] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u));
        r[2 * i + 1] = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u));
    }
    const h2 b = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = r[i] - b;
    return h8{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}

// x = hi + lo, each rounded to nearest: 22 bits and the sign.  In pairs: a
// packed conversion, x - hi as one mixed FMA (exact), a packed conversion.
typedef float f2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void split8(const float (&x)[8], h8& hi, h8& lo) {
    u4 a, b;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        a[j / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x[j], x[j + 1]}), h2));
        f2 d;
        float d0, d1;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d0) : "v"(a[j / 2]), "v"(x[j]));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d1) : "v"(a[j / 2]), "v"(x[j + 1]));
        d = f2{d0, d1};
        b[j / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(d, h2));
    }
    hi = __builtin_bit_cast(h8, a);
    lo = __builtin_bit_cast(h8, b);
}

constexpr float LOG2E = 1.4426950408889634f;
// Probabilities are held times 2^P_BIAS against a maximum that moves only when
// one would pass 2^(P_BIAS + P_SLACK) = 2^15 (f16 holds up to 2^16): after a
// sequence's first keys out is hardly ever rescaled, and what f16 cannot hold
// of a probability stays below 2^(-25 - P_BIAS) of the largest.
constexpr float P_BIAS = 11.0f, P_SLACK = 4.0f;
// f32 and int8 values may be as large as f32 goes: there the weights (int8: the
// finished sums) are held times 2^-down, with the slack and the keys' number in
// it, so that no sum is larger than the largest value.  (Values below about
// 2^(down - 126) lose bits in turn, 1e-33 at 4096 keys.)
__device__ __forceinline__ int down_of(int keys) { return 5 + 32 - __builtin_clz(keys | 1); }

// A pair's running maximum m, one of the scores as the products leave them,
// their factor mul not in it, and what the weights of scores s are formed with,
// exp2(s mul + mb): one FMA each, right while m mul rounds by less than 2^-4, to
// all weights alike.  Beyond FAR (to the end of f32, where a rounding is more than
// the slack) the scores of the tile have m taken off first, which mb then has not.
constexpr float FAR = 1048576.0f;  // 2^20
struct Top {
    float m, mb;
    bool far;  // of any pair of the wave
    __device__ __forceinline__ explicit Top(float bias) : m(-__builtin_inff()), mb(bias), far(false) {}
    __device__ __forceinline__ float base() const { return m == -__builtin_inff() ? 0.0f : m; }
    // Whether a tile's largest score has to become some pair's maximum.
    __device__ __forceinline__ bool moves(float mx, float mul) const {
        return __builtin_amdgcn_ballot_w64((mx - m) * mul > P_SLACK) != 0;
    }
    // Then: what the pair's sums so far count.
    __device__ __forceinline__ float move(float mx, float mul, float bias) {
        const float was = m;
        m = (mx - m) * mul > P_SLACK ? mx : m;
        const float z = base() * mul;
        far = __builtin_amdgcn_ballot_w64(__builtin_fabsf(z) > FAR) != 0;
        mb = far ? bias : bias - z;
        return __builtin_amdgcn_exp2f((was - base()) * mul);
    }
};
// The scale of scores of q times 2^-e: not zero, and no larger than what f32
// can multiply such scores by (over f16 and int8 keys they are 0 or more than
// 2^-52, and differ by 2^-76 or not at all, so that 2^100 parts them as any
// larger factor would).
__device__ __forceinline__ float score_scale(float scale, int e) {
    return fminf(fmaxf(__builtin_ldexpf(scale, e), 1.17549435e-38f), 1.2676506002282294e30f);
}

// int8: a key's value step goes into its probability, w = p step, and the
// pair's weights are held over a power of two of their own, so that neither
// steps of any size nor other rows' keys cost a pair its bits: ev is the
// exponent field of the pair's largest weight so far, falling with the
// maximum's rescaling (alpha), and weights and out are held times
// 2^(W_EXP - ev), the largest weight thus below 2^15.
constexpr int W_EXP = 127 + 14;
__device__ __forceinline__ int weight_exp(int ev, float alpha, float wm) {
    const int ea = (int)(__float_as_uint(alpha) >> 23) - 126;  // alpha < 2^ea; alpha == 1: one too many
    const int was = alpha == 1.0f ? ev : max(0, ev + ea);
    return max(was, (int)(__float_as_uint(wm) >> 23));
}

// What differs by the stored type: DT FRQ_DT_F32, F16 or ROWI8.
template <int DT>
struct Type {
    static constexpr bool F32 = DT == FRQ_DT_F32, I8 = DT == FRQ_DT_ROWI8;
    static constexpr int SZ = F32 ? 4 : I8 ? 1 : 2;
    static constexpr int KT = F32 ? 16 : 32;   // keys a tile of one wave
    static constexpr int PL = F32 ? 4 : 8;     // consecutive values a lane holds of an operand
    static constexpr int KS = F32 ? 16 : 32;   // hd a step
    using Raw = std::conditional_t<I8, u2, u4>;  // a lane's load
};

template <int DT>
__device__ __forceinline__ float value_at(const char* p) {
    if constexpr (DT == FRQ_DT_F32) return *reinterpret_cast<const float*>(p);
    else return (float)*reinterpret_cast<const _Float16*>(p);
}

template <int DT>
__device__ __forceinline__ typename Type<DT>::Raw load_raw(const char* p) {
    return *reinterpret_cast<const typename Type<DT>::Raw*>(p);
}

// Which of two f16 in a word are not finite, as a mask of their bits.
__device__ __forceinline__ uint32_t odd_h2(uint32_t w) {
    return ((w & 0x7C00u) == 0x7C00u ? 0x0000FFFFu : 0u) | ((w & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u);
}

// The 16 pairs of a lane's column: q times a power of two, as B operands.
template <int DT, int NS>
struct QOp {
    static constexpr bool F32 = Type<DT>::F32;
    h8 hi[F32 ? 1 : NS], lo[F32 ? 1 : NS];
    f4 x[F32 ? NS : 1];
    int e;  // q = 2^e times what is held
};

// q points at the pair's hd values; lane group g takes PL of each step's KS.
template <int DT, int HD, int NS>
__device__ __forceinline__ void load_q(const float* q, float sign, int g, QOp<DT, NS>& o) {
    using T = Type<DT>;
    float x[NS][T::PL];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int c = s * T::KS + g * T::PL;
        const bool in = HD % T::KS == 0 || c < HD;
#pragma unroll
        for (int j = 0; j < T::PL; j += 4) {
            const F4 f = *reinterpret_cast<const F4*>(q + (in ? c + j : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[s][j + i] = in ? f.v[i] * sign : 0.0f;
        }
    }
    if constexpr (T::F32) {
        o.e = 0;
#pragma unroll
        for (int s = 0; s < NS; ++s) o.x[s] = f4{x[s][0], x[s][1], x[s][2], x[s][3]};
    } else {
        float mx = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, __builtin_fabsf(x[s][j]));
        const int eb = (int)(__float_as_uint(fmax16(mx)) >> 23);
        o.e = eb == 0 || eb == 255 ? 0 : eb - 127;  // zero, subnormal and non-finite rows as they are
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = __builtin_ldexpf(x[s][j], -o.e);
            split8(x[s], o.hi[s], o.lo[s]);
        }
    }
}

// ---- decode: a wave takes whole key tiles for 16 pairs ----------------------
// HD channels: NS steps of the scores (the last half empty where HD is 16 mod
// 32), NT tiles of the values.  NW waves share a chunk's tiles and join in LDS.
//
// Bound by the reading of keys and values, each once for 16 heads and rows: a
// wave's loads of the next tile's keys are in flight under the softmax, of its
// values under the next scores, straight into registers (LDS would add a pass
// and a barrier a tile), page ids a tile ahead.  With two workgroups of four
// waves a CU (the kernel alone; a large copy reaches 4.8 TB/s): f16, one
// sequence of 131071 tokens, 8 kv heads of 128 channels, 95 us, 5.6 TB/s; f32, a
// window of 4096, 16 sequences, 4 kv heads of 256, 108 us, 4.8 TB/s; int8, 48
// sequences of up to 6001, 4 kv heads of 128 with 7 heads each, 41 us, 3.7 TB/s:
// there the unpacking, the steps and the softmax of half the bytes keep the
// vector units busy 40% of the time, and waves wait the other half.  Slower
// (batch, long, window): loads past the caches 47, 110, 122 us; eight waves a
// workgroup 55 and 168 (batch, window); a wave's tiles side by side 107 and 131
// (long, window).
template <int DT, int HD, int NW>
__global__ __launch_bounds__(64 * NW, HD <= 192 ? 2 : 1) void kv_decode_kernel(const Args a) {
    using T = Type<DT>;
    constexpr int NS = (HD + T::KS - 1) / T::KS, NT = HD / 16;
    constexpr bool WHOLE = HD % T::KS == 0;
    constexpr int KT = T::KT, NU = KT / 16;
    constexpr int ORow = HD + 4;
    __shared__ float red[NW / 2][16][ORow];
    __shared__ float stat[NW][16][2];
    __shared__ int holes[NW];
    const int n_kv = a.c.n_kv;
    const int kvh = blockIdx.x % n_kv;
    const Item it = find_item(a.c, blockIdx.x / n_kv, a.err);
    if (kvh == 0) note_item(a.rec, blockIdx.x / n_kv, it);
    if (!it.found) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    constexpr int hd = HD;
    const int page = a.kv.page, shift = a.c.shift;
    // the pair of this lane's column; columns past the last pair repeat it
    const int pairs = it.q.rows * a.c.rep;
    const int p0 = it.tile * 16, np = min(16, pairs - p0);
    const int pr = p0 + min(col, np - 1);
    const int row = pr / a.c.rep, head = kvh * a.c.rep + pr % a.c.rep;
    const int pos = it.q.len - it.q.rows + row;
    // the tile's first and last row
    const int pos_a = uni(it.q.len - it.q.rows + p0 / a.c.rep);
    const int pos_b = uni(it.q.len - it.q.rows + (p0 + np - 1) / a.c.rep);
    const int see_lo = key_lo(a.c, pos), lo_a = key_lo(a.c, pos_a), lo_b = key_lo(a.c, pos_b);
    const int64_t beg64 = tile_lo(a.c, pos_a) + (int64_t)it.chunk * it.klen;
    const int end = uni((int)min(beg64 + it.klen, (int64_t)pos_b + 1));
    const int beg = uni((int)min(beg64, (int64_t)max(end, 0)));
    const int tiles = end > beg ? (end - beg + KT - 1) / KT : 0;
    QOp<DT, NS> q;
    load_q<DT, HD, NS>(a.q + (int64_t)(it.q.row0 + row) * a.q_pitch + (int64_t)head * hd, a.sign, g, q);
    // scores times mul are in the domain of exp2; with a cap they are made so
    const bool capped = a.cap > 0.0f;
    const float scl = score_scale(a.scale, q.e);
    const float mul = capped ? 1.0f : scl * LOG2E, rcap = capped ? scl / a.cap : 0.0f;
    const int32_t* table = a.pages + (int64_t)it.seq * a.pages_pitch;
    const int last_page = max(0, it.q.len - 1) >> shift;
    const char* kb = a.kv.k + (int64_t)kvh * page * hd * T::SZ;
    const char* vb = a.kv.v + (int64_t)kvh * page * hd * T::SZ;

    typename T::Raw kr[NU][NS], vr[NT];
    float ksc[T::I8 ? 8 : 1], vsc[T::I8 ? 8 : 1];  // int8: the steps of the keys base + 8 g ..
    f4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = f4{0, 0, 0, 0};
    constexpr float BIAS = T::I8 || T::F32 ? 0.0f : P_BIAS;
    const int down = down_of(it.q.len);
    Top top(BIAS);
    float l = 0.0f;
    int ev = 0;  // int8: out is held times 2^(W_EXP - ev)
    uint32_t odd = 0;
    const bool alike = lo_a == lo_b && pos_a == pos_b;  // every pair sees the same

    // the page ids of a tile's two halves, loaded a tile ahead of the loads
    // that use them; a bad one reads page 0 and is looked into at the end
    int pid[2], nid[2];
    bool bad = false;
    auto ids = [&](int base) {
#pragma unroll
        for (int h = 0; h < 2; ++h) nid[h] = table[min((base + 16 * h) >> shift, last_page)];
    };
    auto pages = [&]() {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int id = page_ok(nid[h], a.kv.n_pages);
            bad |= id < 0;
            pid[h] = __builtin_amdgcn_readfirstlane(max(id, 0));
        }
    };
    auto load_k = [&](int base) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int d = T::F32 ? col : 8 * (col >> 2) + 4 * u + (col & 3);
            const int64_t pg = d >= 16 ? pid[1] : pid[0];
            const char* p = kb + pg * a.kv.stride + (int64_t)((base + d) & (page - 1)) * hd * T::SZ;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const int c = s * T::KS + g * T::PL;
                kr[u][s] = load_raw<DT>(p + (WHOLE || c < hd ? c : 0) * T::SZ);
            }
        }
        if constexpr (T::I8) {
            const int64_t pg = g >= 2 ? pid[1] : pid[0];
            const float* p = a.kv.ks + pg * a.kv.sstride + kvh * page + ((base + 8 * g) & (page - 1));
#pragma unroll
            for (int j = 0; j < 8; j += 4) *reinterpret_cast<f4*>(ksc + j) = *reinterpret_cast<const f4*>(p + j);
        }
    };
    auto load_v = [&](int base) {
        const int64_t pg = T::PL * g >= 16 ? pid[1] : pid[0];
        const int at = (base + T::PL * g) & (page - 1);
        const char* p = vb + pg * a.kv.stride + ((int64_t)col * page + at) * T::SZ;
#pragma unroll
        for (int t = 0; t < NT; ++t)
            vr[t] = load_raw<DT>(p + (int64_t)t * 16 * page * T::SZ);
        if constexpr (T::I8) {
            const float* s = a.kv.vs + pg * a.kv.sstride + kvh * page + at;
#pragma unroll
            for (int j = 0; j < 8; j += 4) *reinterpret_cast<f4*>(vsc + j) = *reinterpret_cast<const f4*>(s + j);
        }
    };
    if (wave < tiles) {
        ids(beg + wave * KT);
        pages();
        ids(beg + (wave + NW) * KT);
        load_k(beg + wave * KT);
        load_v(beg + wave * KT);
    }
    for (int ti = wave; ti < tiles; ti += NW) {
        const int base = beg + ti * KT;
        const bool more = ti + NW < tiles;
        const int next = base + NW * KT;
        // ---- scores: s[4 u + i] is key base + PL g + 4 u + i of this lane's pair
        f4 sc[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            sc[u] = f4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if constexpr (T::F32) {
                    f4 x = __builtin_bit_cast(f4, kr[u][s]);
                    if (!WHOLE && s * T::KS + g * T::PL >= hd) x = f4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], q.x[s][j], sc[u], 0, 0, 0);
                } else {
                    h8 x;
                    if constexpr (T::I8) x = i8_to_h8(kr[u][s]);
                    else x = __builtin_bit_cast(h8, kr[u][s]);
                    if (!WHOLE && s * T::KS + g * T::PL >= hd) x = h8{0, 0, 0, 0, 0, 0, 0, 0};
                    sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.hi[s], sc[u], 0, 0, 0);
                    sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.lo[s], sc[u], 0, 0, 0);
                }
            }
        }
        float s[4 * NU];
#pragma unroll
        for (int j = 0; j < 4 * NU; ++j) {
            s[j] = sc[j / 4][j % 4];
            if constexpr (T::I8) s[j] *= ksc[j];
        }
        float vcur[T::I8 ? 8 : 1];
        if constexpr (T::I8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) vcur[j] = vsc[j];
        }
        if (more) {
            pages();
            ids(next + NW * KT);
            load_k(next);
        }
        if (capped) {
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) s[j] = (a.cap * LOG2E) * tanh_f(s[j] * rcap);
        }
        // keys that not every pair of the tile sees
        const bool edge = base < lo_b || base + KT - 1 > pos_a;
        if (edge) {
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) {
                const int key = base + T::PL * g + j;
                if (key < see_lo || key > pos) {
                    s[j] = -__builtin_inff();
                    if constexpr (T::I8) vcur[j] = 0.0f;  // its step may be anything
                }
            }
        }
        // ---- running maximum and sum
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < 4 * NU; ++j) mx = fmaxf(mx, s[j]);
        float alpha = top.move(fmax16(mx), mul, BIAS);
        bool moved = alpha != 1.0f;
        if (__builtin_expect(top.far, 0)) {
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) s[j] -= top.base();
        }
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4 * NU; ++j) {
            s[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j], mul, top.mb));
            if constexpr (T::F32) s[j] = __builtin_ldexpf(s[j], -down);
            sum += s[j];
        }
        l = l * alpha + sum;
        if constexpr (T::I8) {
            float wm = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s[j] *= vcur[j];
                wm = fmaxf(wm, __builtin_fabsf(s[j]));
            }
            const int en = weight_exp(ev, alpha, fmax16(wm));
            moved |= en != ev;
            alpha = __builtin_ldexpf(alpha, ev - en);
            ev = en;
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] = __builtin_ldexpf(s[j], W_EXP - ev);
        }
        if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] *= alpha;
        }
        // ---- values.  Keys that no pair sees may hold anything, and a zero
        // probability would carry what is not finite to pairs that do not see
        // it: both are zeroed in a tile that not every pair sees whole, the
        // second noted and given to its pairs after the loop
        if constexpr (!T::I8) {
            if (edge) {
                constexpr int PW = T::F32 ? 1 : 2;  // values a word
                u4 keep;
#pragma unroll
                for (int j = 0; j < T::PL; ++j) {
                    const int key = base + T::PL * g + j;
                    const uint32_t w = key < lo_a || key > pos_b ? 0u : PW == 1 ? ~0u : j & 1 ? 0xFFFF0000u : 0x0000FFFFu;
                    keep[j / PW] = j % PW ? keep[j / PW] | w : w;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    vr[t] &= keep;
                    if (!alike) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t x = vr[t][j];
                            const uint32_t n = PW == 2 ? odd_h2(x) : (x & 0x7F800000u) == 0x7F800000u ? ~0u : 0u;
                            odd |= n;
                            vr[t][j] = x & ~n;
                        }
                    }
                }
            }
        }
        if constexpr (T::F32) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const f4 x = __builtin_bit_cast(f4, vr[t]);
#pragma unroll
                for (int j = 0; j < 4; ++j) o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], s[j], o[t], 0, 0, 0);
            }
        } else {
            h8 hi, lo;
            split8(s, hi, lo);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                h8 x;
                if constexpr (T::I8) x = i8_to_h8(vr[t]);
                else x = __builtin_bit_cast(h8, vr[t]);
                o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, hi, o[t], 0, 0, 0);
                o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, lo, o[t], 0, 0, 0);
            }
        }
        if (more) load_v(next);
    }
    if constexpr (!T::I8) {
        // rare: the keys of those tiles again, one by one
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) != 0, 0)) {
            for (int key = beg; key < end; ++key) {
                const int t0 = (key - beg) / KT, base = beg + t0 * KT;
                if (t0 % NW != wave || (base >= lo_b && base + KT - 1 <= pos_a)) continue;
                const int64_t pg = max(page_ok(table[key >> shift], a.kv.n_pages), 0);
                const char* p = vb + pg * a.kv.stride + (int64_t)(key & (page - 1)) * T::SZ;
                const bool sees = key >= see_lo && key <= pos;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = value_at<DT>(p + (int64_t)(16 * t + 4 * g + i) * page * T::SZ);
                        if (sees && !(x - x == 0.0f)) o[t][i] += x;
                    }
            }
        }
    }
    // ---- the waves' parts: the largest maximum, then sums in a fixed order
    l = fsum16(T::I8 ? __builtin_ldexpf(l, -down) : l);
    const float m = top.m * mul;
    if (g == 0) {
        stat[wave][col][0] = m;
        stat[wave][col][1] = l;
    }
    if (lane == 0) holes[wave] = bad;
    __syncthreads();
    float mm = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, stat[w][col][0]);
    const float mr = mm == -__builtin_inff() ? 0.0f : mm;
    int hole = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) hole |= holes[w];
    float lsum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) lsum += stat[w][col][1] * __builtin_amdgcn_exp2f(stat[w][col][0] - mr);
    float f = __builtin_amdgcn_exp2f(m - mr);
    if constexpr (T::I8) f = __builtin_ldexpf(f, ev - W_EXP - down);
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] *= f;
#pragma unroll
    for (int h = NW / 2; h; h >>= 1) {
        if (wave >= h && wave < 2 * h) {
#pragma unroll
            for (int t = 0; t < NT; ++t) *reinterpret_cast<f4*>(&red[wave - h][col][16 * t + 4 * g]) = o[t];
        }
        __syncthreads();
        if (wave < h) {
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] += *reinterpret_cast<const f4*>(&red[wave][col][16 * t + 4 * g]);
        }
        __syncthreads();
    }
    if (wave != 0) return;
    if (__builtin_expect(hole, 0) && page_bad(a, it.seq, max(lo_a, beg), min(pos_b, end - 1))) {
        note_hole(a, blockIdx.x / n_kv, it.seq);
        lsum = HOLE;
    }
    if (col >= np) return;
    if (it.chunks == 1) {
        const float r = over(lsum, pos);
        float* d = a.out + (int64_t)(it.q.row0 + row) * a.out_pitch + (int64_t)head * hd + 4 * g;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            F4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y.v[i] = o[t][i] * r;
            *reinterpret_cast<F4*>(d + 16 * t) = y;
        }
    } else {
        const int64_t slot = it.slot + it.chunk;
        if (slot < 0 || slot >= a.slots) return;  // the host's bound holds them all
        float* d = a.part + (slot * n_kv + kvh) * (int64_t)(16 * (hd + 2));
        if (g == 0) {
            d[2 * col] = mm;
            d[2 * col + 1] = lsum;
        }
        d += 32 + (int64_t)col * hd + 4 * g;
#pragma unroll
        for (int t = 0; t < NT; ++t)
            *reinterpret_cast<f4*>(d + 16 * t) = o[t];
    }
}

__device__ __forceinline__ int pick4(int j, int a, int b, int c, int d) {
    const int lo = j & 1 ? b : a, hi = j & 1 ? d : c;
    return j & 2 ? hi : lo;
}

// ---- prompt: 128 pairs a workgroup, keys and values through LDS -------------
// Four waves of 32 pairs each on the 32 x 32 x 16 products; the workgroup's
// key tiles (KT keys) are staged in LDS as f16, double-buffered, the next
// tile's loads in flight under the current one's products.  A lane again owns
// a pair (lane % 32): key row r of a score tile is the key whose bits 2 and 3
// are r's swapped, so that the probabilities come out as the B operand of
// O^T = V^T P^T.
//
// LDS rows are cut into 16-byte pieces, piece c of row r at c ^ (r mod a power
// of two), so that the 32 rows a read takes the same piece of lie in
// different banks.
//
// Bound by the matrix cores, and by the clock under them (1.7 GHz, the cores
// busy half the time): f16, 28 heads of 128 channels over 4, 2048 rows after
// 6144 cached tokens, is 210 GFLOP of the formula, which the two halves of q
// and p make 420, in 464 us; int8, 7 sequences of up to 1501 tokens, 24 GFLOP,
// in 101.  One f16 for p would cost its bits below 2^-11.  128 pairs a workgroup
// let two fit a CU (64 KB of LDS, 256 registers); equal priorities of both 503 us
// against 481.
//
// An f32 cache is staged as three bf16 (exact: 8 bits each), q and the
// probabilities likewise, and a product is the six of theirs that reach 2^-24
// of it: six matrix instructions, where the f32 ones would take the time of
// sixteen (the f16 case over an f32 cache 1637 us against 2768).  Its tiles are
// loaded into registers and have one buffer.
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void split8(const float (&x)[8], b8 (&y)[3]) {
    u4 w[3];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float r[2] = {x[j], x[j + 1]};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            w[k][j / 2] = __builtin_amdgcn_perm(__float_as_uint(r[1]), __float_as_uint(r[0]), 0x07060302u);
#pragma unroll
            for (int i = 0; i < 2; ++i) r[i] -= __uint_as_float(__float_as_uint(r[i]) & 0xFFFF0000u);
        }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) y[k] = __builtin_bit_cast(b8, w[k]);
}
__device__ __forceinline__ void split8(const float (&x)[8], h8 (&y)[2]) { split8(x, y[0], y[1]); }
typedef float f16v __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f16v product(const h8 (&x)[1], const h8 (&y)[2], f16v c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[0], y[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x[0], y[1], c, 0, 0, 0);
}
__device__ __forceinline__ f16v product(const b8 (&x)[3], const b8 (&y)[3], f16v c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[2], y[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], y[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], y[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[0], c, 0, 0, 0);
}

template <int DT, int HD>
struct Prompt {
    static constexpr bool F32 = DT == FRQ_DT_F32;
    static constexpr int N32 = (HD + 31) / 32;
    using Op = std::conditional_t<F32, b8, h8>;
    static constexpr int NA = F32 ? 3 : 1, NB = F32 ? 3 : 2;  // parts of a cache operand, of q and p
    static constexpr int NBUF = F32 ? 1 : 2;                  // buffers
    static constexpr int WAVES = !F32 && N32 <= 4 ? 2 : 1;    // a SIMD
    static constexpr int KT = N32 % 2 || (!F32 && N32 <= 4) ? 64 : 32;  // keys a tile
    static constexpr int HP = 32 * N32;             // HD, padded
    static constexpr int KC = HP / 8, VC = KT / 8;  // pieces of a key row, of a value row
    static constexpr int KX = KC % 16 == 0 ? 15 : KC % 8 == 0 ? 7 : 3, VX = VC - 1;
    static constexpr int IPW = KT * KC / 256;       // pieces a thread stages of each
    static constexpr int BUF = KT * HP;             // elements of one matrix's tile (of one part)
    static constexpr int LDS = 2 * NBUF * NA * BUF * 2 + (DT == FRQ_DT_ROWI8 ? 2 * 2 * KT * 4 : 0);
};

template <int DT, int HD>
__global__ __launch_bounds__(256, (Prompt<DT, HD>::WAVES)) void kv_prompt_kernel(const Args a) {
    using P = Prompt<DT, HD>;
    using Op = typename P::Op;
    constexpr bool I8 = DT == FRQ_DT_ROWI8, F32 = P::F32, F16 = !I8 && !F32;
    constexpr int SZ = I8 ? 1 : F32 ? 4 : 2, NA = P::NA, NB = P::NB, NBUF = P::NBUF;
    constexpr int NS = HD / 16, NH = P::N32, NK = P::KT / 32, KT = P::KT, IPW = P::IPW;
    extern __shared__ __align__(1024) char lds[];
    __shared__ int flag, hole;  // a value was taken out; a page id was bad
    uint16_t* lk = reinterpret_cast<uint16_t*>(lds);                   // [NBUF][NA][KT][HP]
    uint16_t* lv = lk + NBUF * NA * P::BUF;                            // [NBUF][NA][HP][KT]
    float* lks = reinterpret_cast<float*>(lv + NBUF * NA * P::BUF);    // [2][KT] int8 steps
    float* lvs = lks + 2 * KT;
    const int n_kv = a.c.n_kv;
    const int kvh = blockIdx.x % n_kv;
    const Item it = find_item(a.c, blockIdx.x / n_kv, a.err);
    if (kvh == 0) note_item(a.rec, blockIdx.x / n_kv, it);
    if (!it.found) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 31, h = lane >> 5;
    constexpr int hd = HD;
    const int page = a.kv.page, shift = a.c.shift, rep = a.c.rep;
    const int pairs = it.q.rows * rep, off = it.q.len - it.q.rows;
    // the workgroup's pairs and keys
    const int t0 = it.tile * 128, tn = min(128, pairs - t0);
    const int wpos_a = uni(off + t0 / rep), wpos_b = uni(off + (t0 + tn - 1) / rep);  // its first and last row
    const int64_t beg64 = tile_lo(a.c, wpos_a) + (int64_t)it.chunk * it.klen;
    const int end = uni((int)min(beg64 + it.klen, (int64_t)wpos_b + 1));
    const int beg = uni((int)min(beg64, (int64_t)max(end, 0)));
    const int tiles = end > beg ? (end - beg + KT - 1) / KT : 0;
    // the wave's, the lane's; columns past the last pair repeat it
    const int p0 = t0 + min(32 * wave, tn - 1), np = max(1, min(32, tn - 32 * wave));
    const bool idle = 32 * wave >= tn;
    const int pr = p0 + min(col, np - 1);
    const int row = pr / rep, head = kvh * rep + pr % rep, pos = off + row;
    const int pos_a = uni(off + p0 / rep), pos_b = uni(off + (p0 + np - 1) / rep);
    const int see_lo = key_lo(a.c, pos), lo_a = key_lo(a.c, pos_a), lo_b = key_lo(a.c, pos_b);

    // ---- q, times a power of two (f16), as the B operands of the scores
    Op qv[NS][NB];
    int qe;
    {
        const float* q = a.q + (int64_t)(it.q.row0 + row) * a.q_pitch + (int64_t)head * hd;
        float x[NS][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int c = 16 * s + 8 * h;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                const F4 f = *reinterpret_cast<const F4*>(q + c + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[s][j + i] = f.v[i] * a.sign;
                    mx = fmaxf(mx, __builtin_fabsf(x[s][j + i]));
                }
            }
        }
        mx = fmaxf(mx, __uint_as_float(xshfl<32>(__float_as_uint(mx))));
        const int eb = (int)(__float_as_uint(mx) >> 23);
        qe = F32 || eb == 0 || eb == 255 ? 0 : eb - 127;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = __builtin_ldexpf(x[s][j], -qe);
            split8(x[s], qv[s]);
        }
    }
    // scores times mul are in the domain of exp2; with a cap they are made so
    const bool capped = a.cap > 0.0f;
    const float scl = score_scale(a.scale, qe);
    const float mul = capped ? 1.0f : scl * LOG2E, rcap = capped ? scl / a.cap : 0.0f;

    // ---- staging: this thread's pieces (the same place in every tile)
    const int32_t* table = a.pages + (int64_t)it.seq * a.pages_pitch;
    const int last_page = max(0, it.q.len - 1) >> shift;
    const char* kb = a.kv.k + (int64_t)kvh * page * hd * SZ;
    const char* vb = a.kv.v + (int64_t)kvh * page * hd * SZ;
    // A thread stages pieces (wave IPW + i) 64 + lane of both tiles.  A wave's
    // pieces of the keys are KT / 4 whole rows, one page's; its pieces of the
    // values hold the same 8 tokens of different channels.  Page ids are
    // scalar, loaded a tile ahead of the loads that use them and looked at
    // only there; a bad one reads page 0 and is looked into at the end.
    static_assert(64 / P::VC % P::VC == 0 && IPW * 64 * 4 == KT * P::KC && KT / 4 <= 16, "");
    constexpr int VR = 64 / P::VC;                        // channels a wave's piece takes
    const int vr0 = (wave * IPW * 64 + lane) / P::VC;     // channel of piece 0
    const int vd = 8 * ((lane % P::VC) ^ (vr0 & P::VX));  // its first token
    bool bad = false;
    int g0 = 0, g1 = 0, g2 = 0, g3 = 0;  // the ids of the tile's 16-token groups
    auto ids = [&](int base) {
        g0 = table[min(base >> shift, last_page)];
        g1 = table[min((base + 16) >> shift, last_page)];
        if (KT == 64) {
            g2 = table[min((base + 32) >> shift, last_page)];
            g3 = table[min((base + 48) >> shift, last_page)];
        }
    };
    auto page_of = [&](int id) -> int64_t {
        const int ok = page_ok(id, a.kv.n_pages);
        bad |= ok < 0;
        return max(ok, 0);
    };
    using Raw = std::conditional_t<I8, u2, u4>;
    constexpr int NR = F32 ? 2 : 1;  // loads a piece
    Raw rk[F16 ? 1 : IPW][NR], rv[F16 ? 1 : IPW][NR];
    float rs = 0.0f;
    auto fetch = [&](int base, int buf) {
        int ln = lane;
        asm volatile("" : "+v"(ln));  // addresses are formed anew for every tile, not held over the products
        const int r0 = wave * (IPW * VR) + ln / P::VC, tok = 8 * ((ln % P::VC) ^ (r0 & P::VX));
        const char* rows = kb + page_of(pick4(wave * (KT / 4) / 16, g0, g1, g2, g3)) * a.kv.stride +
                           (int64_t)((base + wave * (KT / 4)) & (page - 1)) * (hd * SZ);
        const char* toks = vb + page_of(pick4(tok / 16, g0, g1, g2, g3)) * a.kv.stride + ((base + tok) & (page - 1)) * SZ;
#pragma unroll
        for (int i = 0; i < IPW; ++i) {
            const int d = (i * 64 + ln) / P::KC, r = r0 + i * VR;
            const int c = 8 * (((i * 64 + ln) % P::KC) ^ ((wave * (KT / 4) + d) & P::KX));
            // past hd q is zero, any piece will do; channels past hd are not kept
            const char* pk = rows + (d * hd + (P::HP == hd || c < hd ? c : 0)) * SZ;
            const char* pv = toks + (P::HP == hd || r < hd ? r : 0) * page * SZ;
            if constexpr (!F16) {
#pragma unroll
                for (int x = 0; x < NR; ++x) {
                    rk[i][x] = reinterpret_cast<const Raw*>(pk)[x];
                    rv[i][x] = reinterpret_cast<const Raw*>(pv)[x];
                }
            } else {
                dma16_lds(pk, lk + buf * P::BUF + (wave * IPW + i) * 512);
                dma16_lds(pv, lv + buf * P::BUF + (wave * IPW + i) * 512);
            }
        }
        if constexpr (I8) {
            if (tid < 2 * KT) {  // the steps, a thread a key of each
                const int d = tid % KT;
                const int64_t at = page_of(pick4(d / 16, g0, g1, g2, g3)) * a.kv.sstride + kvh * page + ((base + d) & (page - 1));
                rs = tid < KT ? a.kv.ks[at] : a.kv.vs[at];
            }
        }
    };
    // In a tile that not every pair of the workgroup sees whole, values of keys
    // that none sees (they may be anything) and values that are not finite (a
    // zero probability would carry them to pairs that do not see them) are
    // zeroed; the second are noted and given to their pairs after the loop.
    // (int8 values are finite, and a key that is not seen has weight zero.)
    const int wlo_a = key_lo(a.c, wpos_a), wlo_b = key_lo(a.c, wpos_b);
    auto land = [&](int base, int buf) {
        const bool edge = base < wlo_b || base + KT - 1 > wpos_a;
        if constexpr (I8) {
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
                const int p = (wave * IPW + i) * 64 + lane;
                *reinterpret_cast<h8*>(lk + buf * P::BUF + p * 8) = i8_to_h8(rk[i][0]);
                *reinterpret_cast<h8*>(lv + buf * P::BUF + p * 8) = i8_to_h8(rv[i][0]);
            }
            if (tid < KT) lks[buf * KT + tid] = rs;
            else if (tid < 2 * KT) lvs[buf * KT + tid - KT] = rs;
        } else if constexpr (F32) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
                const int p = (wave * IPW + i) * 64 + lane;
                float x[8], y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[j] = __uint_as_float(rk[i][j / 4][j % 4]);
                    y[j] = __uint_as_float(rv[i][j / 4][j % 4]);
                    if (edge) {
                        const int key = base + vd + j;
                        const bool seen = key >= wlo_a && key <= wpos_b, fin = y[j] - y[j] == 0.0f;
                        odd |= seen && !fin;
                        y[j] = seen && fin ? y[j] : 0.0f;
                    }
                }
                b8 xs[3], ys[3];
                split8(x, xs);
                split8(y, ys);
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    *reinterpret_cast<b8*>(lk + (buf * NA + k) * P::BUF + p * 8) = xs[k];
                    *reinterpret_cast<b8*>(lv + (buf * NA + k) * P::BUF + p * 8) = ys[k];
                }
            }
            if (odd) flag = 1;
        } else {
            wait_vmcnt<0>();
            if (!edge) return;
            uint32_t odd = 0;
#pragma unroll 1
            for (int i = 0; i < IPW; ++i) {
                u4* at = reinterpret_cast<u4*>(lv + buf * P::BUF + ((wave * IPW + i) * 64 + lane) * 8);
                u4 v = *at;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = base + vd + j;
                    if (key < wlo_a || key > wpos_b) v[j / 2] &= j & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t n = odd_h2(v[j]);
                    odd |= n;
                    v[j] &= ~n;
                }
                *at = v;
            }
            if (odd) flag = 1;
        }
    };

    f16v o[NH];
#pragma unroll
    for (int t = 0; t < NH; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    constexpr float BIAS = I8 || F32 ? 0.0f : P_BIAS;
    const int down = down_of(it.q.len);
    Top top(BIAS);
    float l = 0.0f;
    int ev = 0;
    const int krow = (col & 19) | (col & 4) << 1 | (col & 8) >> 1;  // the key of this lane's score row
    if (tid == 0) flag = hole = 0;
    // two workgroups share a CU, the second 256 behind the first: one ahead of
    // the other keeps the one's products over the other's softmax
    if ((blockIdx.x >> 8) & 1) __builtin_amdgcn_s_setprio(2);
    __syncthreads();
    if (tiles) {
        ids(beg);
        fetch(beg, 0);
        land(beg, 0);
        if (tiles > 1) ids(beg + KT);
    }
    __syncthreads();
    for (int ti = 0; ti < tiles; ++ti) {
        const int base = beg + ti * KT, buf = NBUF == 1 ? 0 : ti & 1, other = NBUF - 1 - buf;
        if (ti + 1 < tiles) {
            fetch(base + KT, other);
            if (ti + 2 < tiles) ids(base + 2 * KT);
        }
        if (!idle) {
#pragma unroll 1
            for (int u = 0; u < NK; ++u) {
                const int kb0 = base + 32 * u;
                if (kb0 > pos_b || kb0 + 31 < lo_a) continue;
                // operands are read a group ahead of their products, the
                // first of the values ahead of the softmax
                // piece (2 st + h) ^ (row mod) of the key row, 4 u + 2 k + h
                // ^ (row mod) of the value row: the parts of the lane as they
                // are, the step's by one xor-add
                const char* tk = lds + buf * NA * (2 * P::BUF);
                const char* tv = lds + (NBUF + buf) * NA * (2 * P::BUF);
                const uint32_t ka = (32 * u + krow) * (P::KC * 16), kx = (h ^ (krow & P::KX)) * 16;
                const uint32_t va = col * (P::VC * 16), vx = ((h ^ (col & P::VX)) ^ (4 * u)) * 16;
                auto key_op = [&](int st, Op(&x)[NA]) {
#pragma unroll
                    for (int k = 0; k < NA; ++k)
                        x[k] = *reinterpret_cast<const Op*>(tk + ((kx ^ (32 * st)) + ka) + k * (2 * P::BUF));
                };
                auto val_op = [&](int i, Op(&x)[NA]) {  // channel rows 32 (i / 2) .., keys 16 (i % 2) + 8 h ..
#pragma unroll
                    for (int k = 0; k < NA; ++k)
                        x[k] = *reinterpret_cast<const Op*>(tv + ((vx ^ (32 * (i % 2))) + va) + (i / 2) * (32 * P::VC * 16) +
                                                            k * (2 * P::BUF));
                };
                constexpr int G = F32 ? 2 : 4;  // operands a group
                Op xa[G][NA], xb[G][NA];
                f16v s;  // s[8 t + j] is key kb0 + 16 t + 8 h + j
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
                for (int i = 0; i < G; ++i)
                    if (i < NS) key_op(i, xa[i]);
#pragma unroll
                for (int g = 0; g < NS; g += 2 * G) {
#pragma unroll
                    for (int i = 0; i < G; ++i)
                        if (g + G + i < NS) key_op(g + G + i, xb[i]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        if (g + i >= NS) continue;
                        s = product(xa[i], qv[(g + i) % NS], s);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < G; ++i)
                        if (g + 2 * G + i < NS) key_op(g + 2 * G + i, xa[i]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        if (g + G + i >= NS) continue;
                        s = product(xb[i], qv[(g + G + i) % NS], s);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int i = 0; i < G; ++i)
                    if (i < 2 * NH) val_op(i, xa[i]);
                const bool edge = kb0 < lo_b || kb0 + 31 > pos_a;
                if constexpr (I8) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] *= lks[buf * KT + 32 * u + 16 * (i / 8) + 8 * h + i % 8];
                }
                if (capped) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = (a.cap * LOG2E) * tanh_f(s[i] * rcap);
                }
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = kb0 + 16 * (i / 8) + 8 * h + i % 8;
                        if (key < see_lo || key > pos) s[i] = -__builtin_inff();
                    }
                }
                float mx = s[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
                mx = fmaxf(mx, __uint_as_float(xshfl<32>(__float_as_uint(mx))));
                // (moved for every tile the f16 case takes 486 us against 475)
                float alpha = 1.0f;
                if (top.moves(mx, mul)) {
                    alpha = top.move(mx, mul, BIAS);
                    l *= alpha;
                    if constexpr (!I8) {
#pragma unroll
                        for (int t = 0; t < NH; ++t) o[t] *= alpha;
                    }
                }
                if (__builtin_expect(top.far, 0)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] -= top.base();
                }
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], mul, top.mb));
                    if constexpr (F32) s[i] = __builtin_ldexpf(s[i], -down);
                    sum += s[i];
                }
                l += sum;
                if constexpr (I8) {
                    float wm = 0.0f, step[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) step[i] = lvs[buf * KT + 32 * u + 16 * (i / 8) + 8 * h + i % 8];
                    if (edge) {  // the step of a key that is not seen may be anything
#pragma unroll
                        for (int i = 0; i < 16; ++i) step[i] = s[i] == 0.0f ? 0.0f : step[i];
                        __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[i] *= step[i];
                        wm = fmaxf(wm, __builtin_fabsf(s[i]));
                    }
                    wm = fmaxf(wm, __uint_as_float(xshfl<32>(__float_as_uint(wm))));
                    const int en = weight_exp(ev, alpha, wm);
                    const bool moved = alpha != 1.0f || en != ev;
                    alpha = __builtin_ldexpf(alpha, ev - en);
                    ev = en;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = __builtin_ldexpf(s[i], W_EXP - ev);
                    if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
                        for (int t = 0; t < NH; ++t) o[t] *= alpha;
                    }
                }
                Op pv[2][NB];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = s[8 * t + j];
                    split8(x, pv[t]);
                }
#pragma unroll
                for (int g = 0; g < 2 * NH; g += 2 * G) {
#pragma unroll
                    for (int i = 0; i < G; ++i)
                        if (g + G + i < 2 * NH) val_op(g + G + i, xb[i]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        const int t = (g + i) / 2;
                        if (g + i >= 2 * NH) continue;
                        o[t % NH] = product(xa[i], pv[i % 2], o[t % NH]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < G; ++i)
                        if (g + 2 * G + i < 2 * NH) val_op(g + 2 * G + i, xa[i]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        const int t = (g + G + i) / 2;
                        if (g + G + i >= 2 * NH) continue;
                        o[t % NH] = product(xb[i], pv[i % 2], o[t % NH]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        if (NBUF == 1) __syncthreads();
        if (ti + 1 < tiles) land(base + KT, other);
        __syncthreads();
    }
    if (bad) hole = 1;  // (each wave has looked at the ids of its own pieces)
    __syncthreads();
    if constexpr (!I8) {
        if (flag) {  // rare: the keys of those tiles again, one by one (the last barrier was after the last note)
            for (int key = beg; key < end; ++key) {
                const int base = beg + (key - beg) / KT * KT;
                if (base >= wlo_b && base + KT - 1 <= wpos_a) continue;
                const int64_t pg = max(page_ok(table[key >> shift], a.kv.n_pages), 0);
                const char* p = vb + pg * a.kv.stride + (int64_t)(key & (page - 1)) * SZ;
                const bool sees = key >= see_lo && key <= pos;
#pragma unroll
                for (int t = 0; t < NH; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int c = 32 * t + 8 * (i / 4) + 4 * h + i % 4;
                        if (c >= hd) continue;
                        const float x = value_at<DT>(p + (int64_t)c * page * SZ);
                        if (sees && !(x - x == 0.0f)) o[t][i] += x;
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
    }
    if constexpr (I8) l = __builtin_ldexpf(l, -down);
    l += __uint_as_float(xshfl<32>(__float_as_uint(l)));
    if (__builtin_expect(hole, 0) && page_bad(a, it.seq, max(wlo_a, beg), min(wpos_b, end - 1))) {
        note_hole(a, blockIdx.x / n_kv, it.seq);
        l = HOLE;
    }
    if (idle || col >= np) return;
    const float m = top.m * mul;
    if (it.chunks == 1) {
        const float r = over(l, pos);
        float* d = a.out + (int64_t)(it.q.row0 + row) * a.out_pitch + (int64_t)head * hd + 4 * h;
#pragma unroll
        for (int t = 0; t < NH; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int c = 32 * t + 2 * i;
                if (c >= hd) continue;
                F4 y;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    y.v[j] = (I8 ? __builtin_ldexpf(o[t][i + j], ev - W_EXP - down) : o[t][i + j]) * r;
                *reinterpret_cast<F4*>(d + c) = y;
            }
    } else {
        const int64_t slot = it.slot + it.chunk;
        if (slot < 0 || slot >= a.slots) return;  // the host's bound holds them all
        float* d = a.part + (slot * n_kv + kvh) * (int64_t)(128 * (hd + 2));
        const int pair = 32 * wave + col;
        if (h == 0) {
            d[2 * pair] = m;
            d[2 * pair + 1] = l;
        }
        d += 256 + (int64_t)pair * hd + 4 * h;
#pragma unroll
        for (int t = 0; t < NH; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int c = 32 * t + 2 * i;
                if (c >= hd) continue;
                f4 y;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = I8 ? __builtin_ldexpf(o[t][i + j], ev - W_EXP - down) : o[t][i + j];
                *reinterpret_cast<f4*>(d + c) = y;
            }
    }
}

template <int DT>
__device__ __forceinline__ float entry(const char* p) {  // a stored key's or value's
    if constexpr (DT == FRQ_DT_ROWI8) return (float)*reinterpret_cast<const int8_t*>(p);
    else return value_at<DT>(p);
}
// The outputs beg .. end - 1 of the tile (float4 of pairs) without the keys under
// page ids out of range: a wave a pair, eight keys at a time, a lane every 64th
// channel.  For calls in error, and no faster than that: one f16 sequence of
// 131071 tokens 0.11 s, 2048 rows over 8192 tokens 47 ms.
template <int DT, int TP>
__device__ __forceinline__ void redo_share(const Args& a, const Record& it, int kvh, int beg, int end) {
    constexpr bool I8 = DT == FRQ_DT_ROWI8;
    constexpr int SZ = DT == FRQ_DT_F32 ? 4 : I8 ? 1 : 2;
    const int lane = threadIdx.x & 63, hd = a.kv.hd, page = a.kv.page, rep = a.c.rep;
    const int32_t* table = a.pages + (int64_t)(it.seq < 0 ? ~it.seq : it.seq) * a.pages_pitch;
    const int p0 = it.tile * TP, h4 = hd / 4;
    for (int pair = beg / h4 + uni(threadIdx.x >> 6); pair * h4 < end; pair += 4) {
        const int row = (p0 + pair) / rep, head = kvh * rep + (p0 + pair) % rep, pos = it.len - it.rows + row;
        const float* q = a.q + (int64_t)(it.row0 + row) * a.q_pitch + (int64_t)head * hd;
        float x[4], o[4], m = -__builtin_inff(), l = 0.0f;
        int e = 0;  // q is held times 2^-e, as by the loops
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = 64 * i + lane < hd ? q[64 * i + lane] * a.sign : 0.0f;
            o[i] = 0.0f;
            e = max(e, (int)(__float_as_uint(__builtin_fabsf(x[i])) >> 23));
        }
        e = wave_most(e);
        e = DT == FRQ_DT_F32 || e == 0 || e == 255 ? 0 : e - 127;
        const float scl = score_scale(a.scale, e);
        const int down = down_of(it.len);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_ldexpf(x[i], -e);
        int seen = -1;  // (over's place of a row: below 0 if it sees nothing)
        constexpr int U = 8;  // keys at once, one page's
        const int lo = key_lo(a.c, pos);
#pragma unroll 1
        for (int k0 = lo & -U; k0 <= pos; k0 += U) {
            const int64_t pg = page_ok(table[k0 >> a.c.shift], a.kv.n_pages);
            if (pg < 0) continue;
            const int at = k0 & (page - 1);
            const char* k = a.kv.k + pg * a.kv.stride + ((int64_t)kvh * page + at) * hd * SZ;
            const char* v = a.kv.v + pg * a.kv.stride + ((int64_t)kvh * hd * page + at) * SZ;
            const int64_t step = pg * a.kv.sstride + kvh * page + at;
            float z[U], mn = m;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                z[u] = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (64 * i + lane < hd)
                        z[u] = __builtin_fmaf(x[i], entry<DT>(k + (u * hd + 64 * i + lane) * SZ), z[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                z[u] = wave_sum(z[u]);
                if constexpr (I8) z[u] *= a.kv.ks[step + u];
                z[u] = a.cap > 0.0f ? (a.cap * LOG2E) * tanh_f(z[u] * (scl / a.cap)) : z[u] * (scl * LOG2E);
                if (k0 + u < lo || k0 + u > pos) z[u] = -__builtin_inff();
                mn = fmaxf(mn, z[u]);
            }
            const float mr = mn == -__builtin_inff() ? 0.0f : mn, alpha = __builtin_amdgcn_exp2f(m - mr);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] *= alpha;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k0 + u < lo || k0 + u > pos) continue;
                float w = __builtin_ldexpf(__builtin_amdgcn_exp2f(z[u] - mr), -down);
                l += w;
                if constexpr (I8) w *= a.kv.vs[step + u];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (64 * i + lane < hd) o[i] += w * entry<DT>(v + ((int64_t)(64 * i + lane) * page + u) * SZ);
            }
            seen = 0;
        }
        const float r = over(l, seen);
        float* d = a.out + (int64_t)(it.row0 + row) * a.out_pitch + (int64_t)head * hd;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 64 * i + lane, e = pair * h4 + c / 4;
            if (c < hd && e >= beg && e < end) d[c] = o[i] * r;
        }
    }
}
template <int TP>
__device__ __forceinline__ void redo_share(const Args& a, const Record& it, int kvh, int beg, int end) {
    if (a.dtype == FRQ_DT_F32) redo_share<FRQ_DT_F32, TP>(a, it, kvh, beg, end);
    else if (a.dtype == FRQ_DT_F16) redo_share<FRQ_DT_F16, TP>(a, it, kvh, beg, end);
    else redo_share<FRQ_DT_ROWI8, TP>(a, it, kvh, beg, end);
}

// ---- joining the chunks' parts ----------------------------------------------
// The workgroup of a tile's chunk i joins the i-th share of the tile's
// outputs, so that a long sequence's parts are read by many workgroups.
// Threads are (float4 of the share, run of chunks); each folds its chunks,
// then the runs are merged pairwise, always in the same order.  Bound by
// latency: 4.5 to 5.5 us at 60 to 280 chunks of 16 pairs of 128 channels, 10 us for
// 7 prompts' 128 pairs (a float4 a thread at a time: 585 rows of 8 heads of 256
// 64 us in all against 57).
template <int TP>
__device__ __forceinline__ void join_item(const Args& a, unsigned block, f4* so, float* sm, float* sl) {
    const int n_kv = a.c.n_kv, kvh = block % n_kv;
    const Record it = a.rec[block / n_kv];
    if (it.chunks <= 1) {
        if (__builtin_expect(it.seq < 0, 0))
            redo_share<TP>(a, it, kvh, 0, min(TP, it.rows * a.c.rep - it.tile * TP) * (a.kv.hd / 4));
        return;
    }
    if (it.slot < 0 || it.slot + it.chunks > a.slots) return;
    const int hd = a.kv.hd, tid = threadIdx.x;
    const int p0 = it.tile * TP, np = min(TP, it.rows * a.c.rep - p0);
    const int n4 = np * (hd / 4), per = (n4 + it.chunks - 1) / it.chunks;
    const int beg = it.chunk * per, end = min(n4, beg + per);
    int pe = 1;
    while (pe < per && pe < 256) pe *= 2;
    const int runs = 256 / pe, run = tid / pe;
    const int64_t pitch = (int64_t)TP * (hd + 2) * n_kv;
    const float* part = a.part + (it.slot * n_kv + kvh) * (int64_t)(TP * (hd + 2));
    auto store = [&](int pair, int c4, f4 o, float l) {
        const int pr = p0 + pair, row = pr / a.c.rep, head = kvh * a.c.rep + pr % a.c.rep;
        const float r = over(l, it.len - it.rows + row);
        F4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y.v[i] = o[i] * r;
        *reinterpret_cast<F4*>(a.out + (int64_t)(it.row0 + row) * a.out_pitch + (int64_t)head * hd + 4 * c4) = y;
    };
    bool hole = false;
    if (runs == 1) {  // large shares: U float4 a thread at once
        constexpr int U = 4;
        for (int b = beg + tid; b < end; b += 256 * U) {
            int pair[U], c4[U];
            float m[U], l[U];
            f4 o[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int e = min(b + 256 * u, end - 1);
                pair[u] = e / (hd / 4);
                c4[u] = e % (hd / 4);
                m[u] = -__builtin_inff();
                l[u] = 0.0f;
                o[u] = f4{0, 0, 0, 0};
            }
            for (int c = 0; c < it.chunks; ++c) {
                const float* d = part + c * pitch;
                float mc[U], lc[U];
                f4 oc[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    mc[u] = d[2 * pair[u]];
                    lc[u] = d[2 * pair[u] + 1];
                    hole |= lc[u] == HOLE;
                    oc[u] = *reinterpret_cast<const f4*>(d + 2 * TP + (int64_t)pair[u] * hd + 4 * c4[u]);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float mn = fmaxf(m[u], mc[u]), mr = mn == -__builtin_inff() ? 0.0f : mn;
                    const float x = __builtin_amdgcn_exp2f(m[u] - mr), y = __builtin_amdgcn_exp2f(mc[u] - mr);
                    m[u] = mn;
                    l[u] = l[u] * x + lc[u] * y;
                    o[u] = o[u] * x + oc[u] * y;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (b + 256 * u < end) store(pair[u], c4[u], o[u], l[u]);
        }
    }
    for (int b = beg; runs > 1 && b < end; b += pe) {
        const int e = b + tid % pe;
        const bool in = e < end;
        const int pair = in ? e / (hd / 4) : 0, c4 = in ? e % (hd / 4) : 0;
        float m = -__builtin_inff(), l = 0.0f;
        f4 o{0, 0, 0, 0};
        for (int c = run; c < it.chunks; c += runs) {
            const float* d = part + c * pitch;
            const float mc = d[2 * pair], lc = d[2 * pair + 1];
            hole |= lc == HOLE;
            const f4 oc = *reinterpret_cast<const f4*>(d + 2 * TP + (int64_t)pair * hd + 4 * c4);
            const float mn = fmaxf(m, mc), mr = mn == -__builtin_inff() ? 0.0f : mn;
            const float x = __builtin_amdgcn_exp2f(m - mr), y = __builtin_amdgcn_exp2f(mc - mr);
            m = mn;
            l = l * x + lc * y;
            o = o * x + oc * y;
        }
        for (int h = runs / 2; h; h >>= 1) {
            if (run >= h && run < 2 * h) {
                so[tid] = o;
                sm[tid] = m;
                sl[tid] = l;
            }
            __syncthreads();
            if (run < h) {
                const int t = tid + h * pe;
                const float mn = fmaxf(m, sm[t]), mr = mn == -__builtin_inff() ? 0.0f : mn;
                const float x = __builtin_amdgcn_exp2f(m - mr), y = __builtin_amdgcn_exp2f(sm[t] - mr);
                m = mn;
                l = l * x + sl[t] * y;
                o = o * x + so[t] * y;
            }
            __syncthreads();
        }
        if (run == 0 && in) store(pair, c4, o, l);
    }
    if (__builtin_expect(__syncthreads_or(hole), 0)) redo_share<TP>(a, it, kvh, beg, end);
}

// The launchers of one stored type (each in a file of its own).
struct Launch {
    unsigned grid;  // items x kv heads
    hipStream_t s;
};
hipError_t launch_decode_f32(const Args& a, const Launch& l);
hipError_t launch_decode_f16(const Args& a, const Launch& l);
hipError_t launch_decode_i8(const Args& a, const Launch& l);
hipError_t launch_prompt_f32(const Args& a, const Launch& l);
hipError_t launch_prompt_f16(const Args& a, const Launch& l);
hipError_t launch_prompt_i8(const Args& a, const Launch& l);

// Every width has a kernel of its own: with the steps of a width known only at
// run time (the next of 64, 128 and 256, masked) 192 channels took 21 us where
// 256 took 10, 16 channels the time of 64.
template <int HD>
using Width = std::integral_constant<int, HD>;
template <int MOST, typename F>
hipError_t by_width(int hd, F&& f) {
    switch (hd) {
        case 16: return f(Width<16>{});
        case 32: return f(Width<32>{});
        case 48: return f(Width<48>{});
        case 64: return f(Width<64>{});
        case 80: return f(Width<80>{});
        case 96: return f(Width<96>{});
        case 112: return f(Width<112>{});
        case 128: return f(Width<128>{});
    }
    if constexpr (MOST > 128) {
        switch (hd) {
            case 144: return f(Width<144>{});
            case 160: return f(Width<160>{});
            case 176: return f(Width<176>{});
            case 192: return f(Width<192>{});
            case 208: return f(Width<208>{});
            case 224: return f(Width<224>{});
            case 240: return f(Width<240>{});
            case 256: return f(Width<256>{});
        }
    }
    return hipErrorNotSupported;  // not a width that the checks let through
}

template <int DT>
hipError_t launch_decode(const Args& a, const Launch& l) {
    return by_width<256>(a.kv.hd, [&](auto w) {
        kv_decode_kernel<DT, decltype(w)::value, 4><<<dim3(l.grid), dim3(256), 0, l.s>>>(a);
        return hipGetLastError();
    });
}

template <int DT, int HD>
hipError_t run_prompt(const Args& a, const Launch& l) {
    constexpr int lds = Prompt<DT, HD>::LDS;
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kv_prompt_kernel<DT, HD>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    kv_prompt_kernel<DT, HD><<<dim3(l.grid), dim3(256), lds, l.s>>>(a);
    return hipGetLastError();
}
template <int DT>
hipError_t launch_prompt(const Args& a, const Launch& l) {
    return by_width<DT == FRQ_DT_F32 ? 128 : 256>(a.kv.hd,
                                                  [&](auto w) { return run_prompt<DT, decltype(w)::value>(a, l); });
}

}  // namespace kv
}  // namespace frq
