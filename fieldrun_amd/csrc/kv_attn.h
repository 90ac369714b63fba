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
// 32-bit exactness on the f16 matrix cores: the cache's f16 and int8 entries
// are exact f16; an f32 q row, scaled by a power of two to below 2, is the sum
// of two f16 (22 bits and more), likewise the probabilities (scaled by 2^14,
// so that what f16 cannot hold of them is below 2^-38 of the largest); the
// products of both halves add up in the f32 accumulators.  An f32 cache uses
// the f32 matrix cores.
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

struct Args {
    Call c;
    Cache kv;
    const float* q;
    int64_t q_pitch, out_pitch, pages_pitch;
    const int32_t* pages;
    float* out;
    float* part;  // slots of tp (hd + 2) floats a kv head: (m, sum) pairs, then out
    int64_t slots;
    int* err;
    float scale, cap;
};

// An item's place: its sequence, tile and chunk; every lane has the same.
struct Item {
    Seq q;
    int seq, tile, chunk, chunks, klen;
    int64_t slot;  // the chunk 0 slot of this tile (chunks > 1)
    bool found;
};

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

// Finds item `id`: each wave by itself, 64 sequences at a time, first the
// call's keys (the chunk length), then the items before.  No memory but the
// lengths and offsets, no barrier.
__device__ __forceinline__ Item find_item(const Call& c, int64_t id, int* err) {
    const int lane = threadIdx.x & 63;
    Item it{};
    if (c.n_seq == 1) {
        it.q = seq_at(c, 0);
        if (it.q.bad && threadIdx.x == 0 && id == 0) atomicOr(err, ERR_INDEX);
        it.klen = chunk_of(c, keys_of(it.q));
        it.chunks = chunks_of(it.q, it.klen);
        it.found = id < (int64_t)it.q.tiles * it.chunks;
        it.tile = (int)(id / it.chunks);
        it.chunk = (int)(id % it.chunks);
        it.slot = (int64_t)it.tile * it.chunks;
        return it;
    }
    int64_t total = 0;
    for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
        if (s0 + lane < c.n_seq) {
            const Seq q = seq_at(c, s0 + lane);
            total += keys_of(q);
            if (q.bad && id == 0 && threadIdx.x < 64) atomicOr(err, ERR_INDEX);
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) total += __shfl_xor((long long)total, d, 64);
    it.klen = chunk_of(c, total);
    int64_t items = 0, slots = 0;  // of the sequences before
    for (int s0 = 0; s0 < c.n_seq; s0 += 64) {
        Seq q{};
        if (s0 + lane < c.n_seq) q = seq_at(c, s0 + lane);
        const int n = q.tiles ? chunks_of(q, it.klen) : 1;
        const int64_t mine = (int64_t)q.tiles * n;
        int64_t a = mine, b = n > 1 ? mine : 0;  // inclusive sums
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t x = __shfl_up((long long)a, d, 64), y = __shfl_up((long long)b, d, 64);
            if (lane >= d) {
                a += x;
                b += y;
            }
        }
        const uint64_t hit = __builtin_amdgcn_ballot_w64(items + a > id);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            it.seq = s0 + l;
            it.q = seq_at(c, it.seq);
            it.chunks = lane_bcast(n, l);
            const int64_t at = id - items - (lane_bcast(a, l) - lane_bcast(mine, l));
            it.tile = (int)(at / it.chunks);
            it.chunk = (int)(at % it.chunks);
            it.slot = slots + lane_bcast(b, l) - (it.chunks > 1 ? lane_bcast(mine, l) : 0) +
                      (int64_t)it.tile * it.chunks;
            it.found = true;
            return it;
        }
        items += lane_bcast(a, 63);
        slots += lane_bcast(b, 63);
    }
    return it;
}

__device__ __forceinline__ float fmax16(float v) {  // over the four lane groups of a pair
    v = fmaxf(v, __uint_as_float(xshfl<16>(__float_as_uint(v))));
    return fmaxf(v, __uint_as_float(xshfl<32>(__float_as_uint(v))));
}
__device__ __forceinline__ float fsum16(float v) {
    v += __uint_as_float(xshfl<16>(__float_as_uint(v)));
    return v + __uint_as_float(xshfl<32>(__float_as_uint(v)));
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

// x = hi + lo, each rounded to nearest: 22 bits and the sign.
__device__ __forceinline__ void split8(const float (&x)[8], h8& hi, h8& lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        hi[j] = (_Float16)x[j];
        lo[j] = (_Float16)(x[j] - (float)hi[j]);
    }
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float P_BIAS = 14.0f;  // probabilities are held times 2^14

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
__device__ __forceinline__ typename Type<DT>::Raw load_raw(const char* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const typename Type<DT>::Raw*>(p));
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
template <int DT, int NS, bool FULL>
__device__ __forceinline__ void load_q(const float* q, int hd, int g, QOp<DT, NS>& o) {
    using T = Type<DT>;
    float x[NS][T::PL];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int c = s * T::KS + g * T::PL;
        const bool in = FULL || c < hd;
#pragma unroll
        for (int j = 0; j < T::PL; j += 4) {
            const F4 f = *reinterpret_cast<const F4*>(q + (in ? c + j : 0));
#pragma unroll
            for (int i = 0; i < 4; ++i) x[s][j + i] = in ? f.v[i] : 0.0f;
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
// NS steps of hd (hd <= 32 NS; FULL: equal).  NW waves share a chunk's tiles
// and join in LDS.
template <int DT, int N32, bool FULL, int NW>
__global__ __launch_bounds__(64 * NW) void kv_decode_kernel(const Args a) {
    using T = Type<DT>;
    constexpr int NS = 32 * N32 / T::KS, NT = 2 * N32;  // steps of hd in the scores, 16-wide tiles of hd in the values
    constexpr int KT = T::KT, NU = KT / 16;
    constexpr int ORow = 32 * N32 + 4;
    __shared__ float red[NW / 2][16][ORow];
    __shared__ float stat[NW][16][2];
    __shared__ int stat_e[NW];
    const int n_kv = a.c.n_kv;
    const int kvh = blockIdx.x % n_kv;
    const Item it = find_item(a.c, blockIdx.x / n_kv, a.err);
    if (!it.found) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int col = lane & 15, g = lane >> 4;
    const int hd = a.kv.hd, page = a.kv.page, shift = a.c.shift;
    // the pair of this lane's column; columns past the last pair repeat it
    const int pairs = it.q.rows * a.c.rep;
    const int p0 = it.tile * 16, np = min(16, pairs - p0);
    const int pr = p0 + min(col, np - 1);
    const int row = pr / a.c.rep, head = kvh * a.c.rep + pr % a.c.rep;
    const int pos = it.q.len - it.q.rows + row;
    const int pos_a = it.q.len - it.q.rows + p0 / a.c.rep;                 // the tile's first row
    const int pos_b = it.q.len - it.q.rows + (p0 + np - 1) / a.c.rep;      // and last
    const int see_lo = key_lo(a.c, pos), lo_a = key_lo(a.c, pos_a), lo_b = key_lo(a.c, pos_b);
    const int beg = max(it.q.lo + it.chunk * it.klen, lo_a / ALIGN * ALIGN);
    const int end = (int)min((int64_t)it.q.lo + (int64_t)(it.chunk + 1) * it.klen, (int64_t)pos_b + 1);
    const int tiles = end > beg ? (end - beg + KT - 1) / KT : 0;
    QOp<DT, NS> q;
    load_q<DT, NS, FULL>(a.q + (int64_t)(it.q.row0 + row) * a.q_pitch + (int64_t)head * hd, hd, g, q);
    const float scl = __builtin_ldexpf(a.scale, q.e) * (a.cap > 0.0f ? 1.0f : LOG2E);
    const float rcap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    const int32_t* table = a.pages + (int64_t)it.seq * a.pages_pitch;
    const int last_page = max(0, it.q.len - 1) >> shift;
    const char* kb = a.kv.k + (int64_t)kvh * page * hd * T::SZ;
    const char* vb = a.kv.v + (int64_t)kvh * page * hd * T::SZ;

    typename T::Raw kr[NU][NS], vr[NT];
    float ksc[T::I8 ? 8 : 1], vsc[T::I8 ? 8 : 1];  // int8: the steps of the keys base + 8 g ..
    f4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = f4{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.0f;
    int ev = 0;  // int8: out is held times 2^(127 - ev)

    // the page of key `base + d` (d < KT) as the lanes need it; a bad id is
    // reported and reads page 0
    int pid[2];
    auto pages_of = [&](int base) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = min((base + 16 * h) >> shift, last_page);
            const int id = page_ok(table[at], a.kv.n_pages);
            if (id < 0 && lane == 0) atomicOr(a.err, ERR_INDEX);
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
                if (!FULL && s * T::KS >= hd) continue;
                const int c = s * T::KS + g * T::PL;
                kr[u][s] = load_raw<DT>(p + (FULL || c < hd ? c : 0) * T::SZ);
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
            if (FULL || t * 16 < hd) vr[t] = load_raw<DT>(p + (int64_t)t * 16 * page * T::SZ);
        if constexpr (T::I8) {
            const float* s = a.kv.vs + pg * a.kv.sstride + kvh * page + at;
#pragma unroll
            for (int j = 0; j < 8; j += 4) *reinterpret_cast<f4*>(vsc + j) = *reinterpret_cast<const f4*>(s + j);
        }
    };
    if (wave < tiles) {
        pages_of(beg + wave * KT);
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
                if (!FULL && s * T::KS >= hd) continue;
                if constexpr (T::F32) {
                    f4 x = __builtin_bit_cast(f4, kr[u][s]);
                    if (!FULL && s * T::KS + g * T::PL >= hd) x = f4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sc[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], q.x[s][j], sc[u], 0, 0, 0);
                } else {
                    h8 x;
                    if constexpr (T::I8) x = i8_to_h8(kr[u][s]);
                    else x = __builtin_bit_cast(h8, kr[u][s]);
                    if (!FULL && s * T::KS + g * T::PL >= hd) x = h8{0, 0, 0, 0, 0, 0, 0, 0};
                    sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.hi[s], sc[u], 0, 0, 0);
                    sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q.lo[s], sc[u], 0, 0, 0);
                }
            }
        }
        float s[4 * NU];
#pragma unroll
        for (int j = 0; j < 4 * NU; ++j) {
            s[j] = sc[j / 4][j % 4] * scl;
            if constexpr (T::I8) s[j] *= ksc[j];
        }
        float vcur[T::I8 ? 8 : 1];
        if constexpr (T::I8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) vcur[j] = vsc[j];
        }
        if (more) {
            pages_of(next);
            load_k(next);
        }
        if (a.cap > 0.0f) {
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) s[j] = (a.cap * LOG2E) * tanh_f(s[j] * rcap);
        }
        // keys that not every pair of the tile sees
        const bool edge = base < lo_b || base + KT - 1 > pos_a;
        if (edge) {
#pragma unroll
            for (int j = 0; j < 4 * NU; ++j) {
                const int key = base + T::PL * g + j;
                if (key < see_lo || key > pos) s[j] = -__builtin_inff();
                if constexpr (T::I8)
                    if (key < lo_a || key > pos_b) vcur[j] = 0.0f;
            }
        }
        // ---- running maximum and sum
        float mx = s[0];
#pragma unroll
        for (int j = 1; j < 4 * NU; ++j) mx = fmaxf(mx, s[j]);
        const float mn = fmaxf(m, fmax16(mx));
        const float mr = mn == -__builtin_inff() ? 0.0f : mn;
        float alpha = __builtin_amdgcn_exp2f(m - mr);
        bool moved = mn != m;
        m = mn;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4 * NU; ++j) {
            s[j] = __builtin_amdgcn_exp2f(s[j] - mr + P_BIAS);
            sum += s[j];
        }
        l = l * alpha + sum;
        if constexpr (T::I8) {
            // the values' steps go into the probabilities, over the largest
            // step's power of two so far
            float vm = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) vm = fmaxf(vm, __builtin_fabsf(vcur[j]));
            const int en = max(ev, (int)(__float_as_uint(fmax16(vm)) >> 23));
            if (en != ev) {
                alpha = __builtin_ldexpf(alpha, ev - en);
                ev = en;
                moved = true;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] = s[j] == 0.0f ? 0.0f : s[j] * __builtin_ldexpf(vcur[j], 127 - ev);
        }
        if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] *= alpha;
        }
        // ---- values
        if constexpr (T::F32) {
            if (edge) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int key = base + 4 * g + j;
                        if (key < lo_a || key > pos_b) vr[t][j] = 0u;
                    }
            }
            auto product = [&]() {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (!FULL && t * 16 >= hd) continue;
                    const f4 x = __builtin_bit_cast(f4, vr[t]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], s[j], o[t], 0, 0, 0);
                }
            };
            uint32_t odd = 0;
            if (edge && lo_a + pos_a != lo_b + pos_b) {  // rows differ in what they see
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (FULL || t * 16 < hd) odd |= (vr[t][j] & 0x7F800000u) == 0x7F800000u;
            }
            if (!__builtin_amdgcn_ballot_w64(odd)) {
                product();
            } else {
                // a value that is not finite, and a zero probability would
                // carry it to rows that do not see it: key by key, each
                // product kept by the pairs that see the key
                for (int d = 0; d < KT; ++d) {
                    const bool sees = base + d >= see_lo && base + d <= pos;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if (!FULL && t * 16 >= hd) continue;
                        f4 y{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const bool mine = 4 * g + j == d;
                            y = __builtin_amdgcn_mfma_f32_16x16x4f32(mine ? __uint_as_float(vr[t][j]) : 0.0f,
                                                                     mine ? s[j] : 0.0f, y, 0, 0, 0);
                        }
                        if (sees) o[t] += y;
                    }
                }
            }
        } else {
            h8 hi, lo;
            split8(s, hi, lo);
            uint32_t odd = 0;
            if constexpr (!T::I8) {
                if (edge) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int key = base + 8 * g + j;
                            if (key < lo_a || key > pos_b) vr[t][j / 2] &= j & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                        }
                    if (lo_a + pos_a != lo_b + pos_b) {
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (FULL || t * 16 < hd)
                                    odd |= (vr[t][j] & 0x7C00u) == 0x7C00u || (vr[t][j] & 0x7C000000u) == 0x7C000000u;
                    }
                }
            }
            if (!__builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (!FULL && t * 16 >= hd) continue;
                    h8 x;
                    if constexpr (T::I8) x = i8_to_h8(vr[t]);
                    else x = __builtin_bit_cast(h8, vr[t]);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, hi, o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, lo, o[t], 0, 0, 0);
                }
            } else if constexpr (!T::I8) {
                for (int d = 0; d < KT; ++d) {  // as for f32 above
                    const bool sees = base + d >= see_lo && base + d <= pos;
                    h8 ph, pl;
                    u4 keep;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const bool mine = 8 * g + j == d;
                        ph[j] = mine ? hi[j] : (_Float16)0.0f;
                        pl[j] = mine ? lo[j] : (_Float16)0.0f;
                        if (j & 1) keep[j / 2] |= mine ? 0xFFFF0000u : 0u;
                        else keep[j / 2] = mine ? 0x0000FFFFu : 0u;
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if (!FULL && t * 16 >= hd) continue;
                        const h8 x = __builtin_bit_cast(h8, (u4)(vr[t] & keep));
                        f4 y{0, 0, 0, 0};
                        y = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ph, y, 0, 0, 0);
                        y = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, pl, y, 0, 0, 0);
                        if (sees) o[t] += y;
                    }
                }
            }
        }
        if (more) load_v(next);
    }
    // ---- the waves' parts: the largest maximum, then sums in a fixed order
    l = fsum16(l);
    if (g == 0) {
        stat[wave][col][0] = m;
        stat[wave][col][1] = l;
    }
    if (lane == 0) stat_e[wave] = ev;
    __syncthreads();
    float mm = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, stat[w][col][0]);
    const float mr = mm == -__builtin_inff() ? 0.0f : mm;
    float lsum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) lsum += stat[w][col][1] * __builtin_amdgcn_exp2f(stat[w][col][0] - mr);
    float f = __builtin_amdgcn_exp2f(m - mr);
    if constexpr (T::I8) f = __builtin_ldexpf(f, ev - 127);
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
    if (wave != 0 || col >= np) return;
    if (it.chunks == 1) {
        const float r = lsum > 0.0f || lsum != lsum ? 1.0f / lsum : 0.0f;  // no key seen: zeros
        float* d = a.out + (int64_t)(it.q.row0 + row) * a.out_pitch + (int64_t)head * hd + 4 * g;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (!FULL && t * 16 >= hd) continue;
            F4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y.v[i] = o[t][i] * r;
            *reinterpret_cast<F4*>(d + 16 * t) = y;
        }
    } else {
        const int64_t slot = it.slot + it.chunk;
        if (slot >= a.slots) return;  // the host's bound holds them all
        float* d = a.part + (slot * n_kv + kvh) * (int64_t)(16 * (hd + 2));
        if (g == 0) {
            d[2 * col] = mm;
            d[2 * col + 1] = lsum;
        }
        d += 32 + (int64_t)col * hd + 4 * g;
#pragma unroll
        for (int t = 0; t < NT; ++t)
            if (FULL || t * 16 < hd) *reinterpret_cast<f4*>(d + 16 * t) = o[t];
    }
}

// ---- joining the chunks' parts ----------------------------------------------
// The workgroup of a tile's chunk i joins the i-th share of the tile's
// outputs, so that a long sequence's parts are read by many workgroups.
// Threads are (float4 of the share, run of chunks); each folds its chunks,
// then the runs are merged pairwise, always in the same order.
template <int TP>
__global__ __launch_bounds__(256) void kv_join_kernel(const Args a) {
    __shared__ f4 so[256];
    __shared__ float sm[256], sl[256];
    const int n_kv = a.c.n_kv, kvh = blockIdx.x % n_kv;
    const Item it = find_item(a.c, blockIdx.x / n_kv, a.err);
    if (!it.found || it.chunks == 1 || it.slot + it.chunks > a.slots) return;
    const int hd = a.kv.hd, tid = threadIdx.x;
    const int p0 = it.tile * TP, np = min(TP, it.q.rows * a.c.rep - p0);
    const int n4 = np * (hd / 4), per = (n4 + it.chunks - 1) / it.chunks;
    const int beg = it.chunk * per, end = min(n4, beg + per);
    int pe = 1;
    while (pe < per && pe < 256) pe *= 2;
    const int runs = 256 / pe, run = tid / pe;
    const int64_t pitch = (int64_t)TP * (hd + 2) * n_kv;
    const float* part = a.part + (it.slot * n_kv + kvh) * (int64_t)(TP * (hd + 2));
    for (int b = beg; b < end; b += pe) {
        const int e = b + tid % pe;
        const bool in = e < end;
        const int pair = in ? e / (hd / 4) : 0, c4 = in ? e % (hd / 4) : 0;
        float m = -__builtin_inff(), l = 0.0f;
        f4 o{0, 0, 0, 0};
        for (int c = run; c < it.chunks; c += runs) {
            const float* d = part + c * pitch;
            const float mc = d[2 * pair], lc = d[2 * pair + 1];
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
        if (run == 0 && in) {
            const int pr = p0 + pair, row = pr / a.c.rep, head = kvh * a.c.rep + pr % a.c.rep;
            const float r = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            F4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y.v[i] = o[i] * r;
            *reinterpret_cast<F4*>(a.out + (int64_t)(it.q.row0 + row) * a.out_pitch + (int64_t)head * hd + 4 * c4) = y;
        }
    }
}

// The launchers of one stored type (each in a file of its own).
struct Launch {
    unsigned grid;  // items x kv heads
    hipStream_t s;
};
hipError_t launch_decode_f32(const Args& a, const Launch& l);
hipError_t launch_decode_f16(const Args& a, const Launch& l);
hipError_t launch_decode_i8(const Args& a, const Launch& l);

// The kernel of a head width: whole steps of 32 at the widths models have,
// else the next of three with its last steps masked.
template <int DT>
hipError_t launch_decode(const Args& a, const Launch& l) {
    constexpr int NW = 4;
    const int hd = a.kv.hd;
    const dim3 g(l.grid), b(64 * NW);
    if (hd == 64) kv_decode_kernel<DT, 2, true, NW><<<g, b, 0, l.s>>>(a);
    else if (hd == 96) kv_decode_kernel<DT, 3, true, NW><<<g, b, 0, l.s>>>(a);
    else if (hd == 128) kv_decode_kernel<DT, 4, true, NW><<<g, b, 0, l.s>>>(a);
    else if (hd == 256) kv_decode_kernel<DT, 8, true, NW><<<g, b, 0, l.s>>>(a);
    else if (hd <= 64) kv_decode_kernel<DT, 2, false, NW><<<g, b, 0, l.s>>>(a);
    else if (hd <= 128) kv_decode_kernel<DT, 4, false, NW><<<g, b, 0, l.s>>>(a);
    else kv_decode_kernel<DT, 8, false, NW><<<g, b, 0, l.s>>>(a);
    return hipGetLastError();
}

}  // namespace kv
}  // namespace frq
