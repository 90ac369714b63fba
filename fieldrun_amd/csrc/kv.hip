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
#include "kv_rows.h"

namespace frq {
namespace kv {
namespace {

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
    store_values<E, WR>(m, kvh, at, lv);
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
template <bool EX>
__global__ __launch_bounds__(256) void kv_join_kernel(const Args a, const Args b, unsigned grid_a) {
    __shared__ f4 so[256];
    __shared__ float sm[256], sl[256], fac[EX ? JOIN_FACTORS : 1];
    if (blockIdx.x < grid_a) join_item<16, EX>(a, blockIdx.x, so, sm, sl, fac);
    else join_item<128, EX>(b, blockIdx.x - grid_a, so, sm, sl, fac);
}

// The plans of many sequences (workgroup 0: the decode launch's, 1: the
// prompt's): which launch serves those of c.uncut pairs, the call's keys, then the
// items and slots before each 64 sequences.  16 waves, 64 sequences each at a
// time, bound by the latency of two passes over the lengths.
template <bool EX>
__global__ __launch_bounds__(1024) void kv_plan_kernel(const Call ca, const Call cb, int32_t* plan_a, int32_t* plan_b,
                                                       int* err) {
    __shared__ int64_t keys[16], tiles[16], uncut_keys[16], walked[16];
    __shared__ int longest[16];
    const bool dec = blockIdx.x == 0;
    const Call c = dec ? ca : cb;
    const int pairs = EX ? c.uncut : 0;
    int32_t* plan = dec ? plan_a : plan_b;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, blocks = (c.n_seq + 63) / 64;
    int64_t total = 0, all = 0;  // keys, tiles; (pairs: wanted() asks for none) sequences of `pairs` and more
    for (int64_t s = threadIdx.x; s < c.n_seq; s += 1024) {
        const Seq q = seq_at(c, (int)s);
        total += keys_of(q);
        all += pairs ? (int64_t)q.rows * c.rep >= pairs : q.tiles;
        if (q.bad && dec) atomicOr(err, ERR_INDEX);
    }
    total = wave_total(total);
    all = wave_total(all);
    if (lane == 0) {
        keys[w] = total;
        tiles[w] = all;
    }
    __syncthreads();
    total = all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        total += keys[i];
        all += tiles[i];
    }
    bool filled = false;
    if (__builtin_expect(pairs && all, 0)) {
        int64_t uncut = 0, walk = 0;
        int most = 0;
        for (int64_t s = threadIdx.x; s < c.n_seq; s += 1024) {
            const Seq q = seq_at(c, (int)s);
            if ((int64_t)q.rows * c.rep < pairs) continue;
            const int own = lone_keys(c, q);
            uncut += keys_of(q);
            walk += lone_tiles(c, q) * own;
            most = max(most, own);
        }
        uncut = wave_total(uncut);
        walk = wave_total(walk);
        most = wave_most(most);
        if (lane == 0) {
            uncut_keys[w] = uncut;
            walked[w] = walk;
            longest[w] = most;
        }
        __syncthreads();
        uncut = walk = 0;
        for (int i = 0; i < 16; ++i) {
            uncut += uncut_keys[i];
            walk += walked[i];
            most = max(most, longest[i]);
        }
        filled = fills(walk, most, c.n_kv);
        if (filled != c.prompt) total -= uncut;
    }
    const int klen = chunk_of(c, total, wanted(c, all));
    for (int b = w; b < blocks; b += 16) {
        Seq q{};
        if (b * 64 + lane < c.n_seq) q = seq_at(c, b * 64 + lane);
        if (pairs && all) drop_uncut(c, filled, q);
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
        plan[1] = filled;
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
// With sinks or trees one round of half of that (chunk_of_even) where the tiles have
// nearly the same keys (windows mostly, and one sequence always) and memory or one
// workgroup a CU bounds them: windows over f32 keys, over 192 channels, one sequence.
// 512 against it: 16 f32 windows of 4096 by 256 channels 121, 107 us, 35 of 325 52, 35, 20
// f16 ones of 1000 34, 29, f32 of 128 channels 28, 25, one int8 window of 50000 34, 31, 16
// rows of one f16 tree over 8000 27.7, 25.8.  But 20 f32 sequences of 100 to 6001 by 256
// channels 101, 129 (of 256 items: these keep the target), 8 f16 trees of 35 pairs over
// 2000 27, 33, f32 49, 54.
constexpr int EVEN_TARGET = 256;
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

// Trees: a sequence's rows all see (nearly) the same keys, so the prompt kernel's
// tiles of 128 pairs save their reading anew, from little more than a tile of the
// decode kernel on: 16 f16 sequences of up to 4000 tokens with 112 pairs 126 us
// on the decode kernel, 60 on the prompt kernel, 4 of 128 pairs 68, 46, one of 256
// pairs over 32768 tokens 238, 95.  Where the whole call is small its latency
// counts: one sequence of 112 pairs over 8000 tokens 27, 32 us, of 56 over 211
// 9.7, 19.6, of 336 over 2000 27, 27.  (The tokens are those that the table has room
// for, as lengths are device data: 56 pairs over 211 tokens with 4 heads of 128 take 13 us
// with a table of 256 tokens, 23 with one of 32768.)
constexpr int TREE_PAIRS = 32;
constexpr double EX_WORK = 6e6;  // rows x heads x keys
// With sinks or trees the prompt kernel serves every sequence where they have more
// than EX_PAIRS pairs in the mean (without trees, in a small call or over f32 keys, more
// than the decode kernel's; calls with neither keep each row's kernel, and so its
// bits), and their tiles fit the chip at once or are mostly large sequences': the
// launch of the other takes longer than what it saves.  Both launches against one:
// 2048 f16 rows of 28 heads in windows of 1024 89, 86 us, 500 rows beside 31 of one
// row 71, 56, 20 sequences of 84 pairs 54, 37, int8 in windows of 4000 117, 77; trees:
// 4 of 128 pairs 45, 41, 16 int8 of up to 182 72, 67.  But f32, 72 pairs 76, 99; 2000 rows
// beside 31 of one 109, 127; trees of 24 pairs, f16 of 64 channels 39, 55.
constexpr size_t EX_PAIRS = 64;
// With sinks or trees the items fill the chip's workgroups once, less the chunks
// that every tile is rounded up by (wanted(), from the lengths): one tree of 256 pairs
// over 32768 f16 tokens 104 us at 400 items, 91 at the rule's 496; 16 int8 ones of up to
// 182 pairs 84 at 512, 63 at the rule's 424 (65 at 388, the host's bound of the tiles;
// 20 f16 ones 77 by that, 72); 2048 rows in windows of 1024 111, 85 at the rule's 256; 4
// f32 trees of 182 pairs, one workgroup a CU, 119 at 400, 79 at the rule's.
int64_t ex_slots(const frq_kv* kv) { return kv->dtype == FRQ_DT_F32 || kv->hd > 128 ? 256 : 512; }
// A batch with idle sequences, no more rows than sequences, has no room for prompt
// tiles' parts (n_row <= n_seq below): with sinks or trees the prompt kernel takes
// sequences there only where they fill it (fills(), kv_index.h, from the lengths), and
// none of a batch that needs no plan, which has 64 rows at most.  Prompt kernel, decode
// kernel: 64 slots and one tree of 112 pairs over 32768 tokens, 2 kv heads of 64, f16
// 902, 29 us, int8 1253, 27, f32 2124, 55; over 211 f16 21, 11; 2048 slots, 4 kv heads of
// 128, one prompt of 2800 pairs with a window of 1000 f16 76, 65, int8 90, 62, f32 151,
// 109; of 5600 83, 113, 96, 103, 158, 202; 40 trees of 70 pairs over 2000 tokens 104, 130,
// 135, 114, 234, 252.  The choice costs the plan 3 to 5 us.  (Without sinks or trees these
// batches keep their kernels, and so their bits.)
// The work of an attention call, and its workspace: the items' records, the
// decode tiles' parts, where a sequence may ask with several rows the prompt
// tiles', and for many sequences both launches' plans.
struct Plan {
    Call dec, prompt;
    size_t rec_dec, rec_prompt, part_dec, part_prompt, plan_dec, plan_prompt, bytes;  // offsets, the whole
};
// ex: with trees or sinks; keys: those that a row sees at most, by the table's room.
Plan plan_of(const frq_kv* kv, size_t n_row, size_t n_head, size_t n_seq, bool ex, bool trees, size_t keys) {
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
    if (ex && ((kv->dtype == FRQ_DT_F32 && !trees) || kv->hd > 192 || n_seq == 1)) c.even = EVEN_TARGET;
    const bool big = (double)n_row * (double)n_head * (double)keys > EX_WORK;
    p.prompt.min_pairs = 1 + (!trees ? DEC_PAIRS : big ? TREE_PAIRS : 0x7FFFFFFE);
    if (ex && n_row <= n_seq) {
        if (n_seq > (size_t)PLAN_SEQS) p.prompt.uncut = p.prompt.min_pairs;
        else p.prompt.min_pairs = 0x7FFFFFFF;
    }
    p.prompt.tp = 128;
    // (n_row <= n_seq: no room for parts, every tile's keys in one run)
    p.prompt.target = n_row <= n_seq ? 1 : ex ? ex_slots(kv) : kv->hd > 128 ? PROMPT_TARGET_WIDE : PROMPT_TARGET;
    if (ex && n_row > n_seq) p.prompt.slots = (int)p.prompt.target;
    // (f32 keys of over 128 channels have no prompt kernel)
    const bool f32 = kv->dtype == FRQ_DT_F32;
    const size_t pairs = n_row * c.rep, mean = big && (trees || !f32) ? EX_PAIRS : DEC_PAIRS;
    if (ex && n_row > n_seq && !(f32 && kv->hd > 128) && (big || !trees) && pairs > mean * n_seq &&
        (pairs >= 4 * DEC_PAIRS * n_seq || max_tiles(p.prompt) * c.n_kv <= ex_slots(kv)))
        p.prompt.min_pairs = 1;
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

struct More {  // than every attention call has
    size_t sinks;
    const uint64_t* tree;
    size_t tree_pitch;
    bool trees;
};
int attend(frq_ctx* ctx, const frq_kv* kv, const float* d_q, size_t q_pitch, size_t n_row, size_t n_head,
           const int32_t* d_pages, size_t pages_pitch, const int32_t* d_len, const int32_t* d_first, size_t n_seq,
           double scale, double cap, size_t window, const More& more, float* d_out, size_t out_pitch, void* d_ws,
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
    // (sinks beyond every table: all is seen)
    size_t sinks = window ? more.sinks : 0;
    if (sinks > (pages_pitch << shift)) window = sinks = 0;
    if (more.trees && (!more.tree_pitch || more.tree_pitch > ((size_t)1 << 40))) return bad("a tree has masks of a word or more");
    if (!(scale >= -1e30 && scale <= 1e30) || !(cap >= 0.0 && cap <= 1e30))
        return bad("scale must be within 1e30, cap 0 or positive");
    if (n_row && n_seq && (!d_q || !d_out || !d_len || (!d_pages && pages_pitch))) return bad("null pointer");
    if (more.trees && n_row && n_seq && !more.tree) return bad("null pointer");
    if (d_ws && ((uintptr_t)d_ws & 15)) return bad("the workspace must be 16-byte aligned");
    if (!ctx) return bad("null context");
    if (!n_row || !n_seq) return FRQ_OK;
    const bool ex = sinks || more.trees;
    const size_t keys = std::min(pages_pitch << shift, window ? window + sinks : SIZE_MAX);
    const Plan plan = plan_of(kv, n_row, n_head, n_seq, ex, more.trees, keys);
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
    a.c.sinks = (int)sinks;
    a.c.sink_span = sink_keys((int64_t)sinks, 32);
    a.c.tree = more.tree;
    a.c.tree_pitch = (int64_t)more.tree_pitch;
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
    // q leave the prompt kernel one wave a SIMD, and widths of an odd number of 32s
    // do not fit the LDS.  2048 rows of 8 heads over 4, the decode kernel against the
    // prompt kernel: 256 channels 288, 340 us over themselves, 72, 78 at 600 rows,
    // 1612, 1508 over 8192 tokens.  At 192 channels, 225, 202 and 1280, 676, one rule
    // for these widths costs time.)
    const bool prompts = d_first && n_row * (size_t)a.c.rep >= (size_t)plan.prompt.min_pairs &&
                         !(kv->dtype == FRQ_DT_F32 && kv->hd > 128);
    const int uncut = prompts ? plan.prompt.uncut : 0;
    a.c.max_pairs = prompts && !uncut ? plan.prompt.min_pairs - 1 : 0x7FFFFFFF;
    a.c.uncut = uncut;
    char* ws = (char*)d_ws;
    a.rec = (Record*)(ws + plan.rec_dec);
    a.part = (float*)(ws + plan.part_dec);
    a.slots = max_slots(DEC_TARGET, a.c.n_kv);
    Args b = a;
    b.c.min_pairs = plan.prompt.min_pairs;
    b.c.max_pairs = plan.prompt.max_pairs;
    b.c.tp = plan.prompt.tp;
    b.c.target = plan.prompt.target;
    b.c.even = 0;
    b.c.slots = plan.prompt.slots;
    b.c.prompt = true;
    b.c.min_chunk = plan.prompt.min_chunk;
    b.c.sink_span = sink_keys((int64_t)sinks, 64);
    b.rec = (Record*)(ws + plan.rec_prompt);
    b.part = (float*)(ws + plan.part_prompt);
    b.slots = n_row > n_seq ? max_slots(b.c.target, a.c.n_kv) : 0;
    const int64_t ga = a.c.max_pairs ? max_items(a.c) * a.c.n_kv : 0, gb = prompts ? max_items(b.c) * b.c.n_kv : 0;
    if (ga + gb > 0x7FFFFFFF) return bad("too many rows or sequences");
    const Launch la{(unsigned)ga, s}, lb{(unsigned)gb, s};
    hipError_t e = hipSuccess;
    if (n_seq > (size_t)PLAN_SEQS) {
        int32_t *pa = (int32_t*)(ws + plan.plan_dec), *pb = (int32_t*)(ws + plan.plan_prompt);
        if (ex) kv_plan_kernel<true><<<dim3(prompts ? 2 : 1), dim3(1024), 0, s>>>(a.c, b.c, pa, pb, a.err);
        else kv_plan_kernel<false><<<dim3(prompts ? 2 : 1), dim3(1024), 0, s>>>(a.c, b.c, pa, pb, a.err);
        e = hipGetLastError();
        if (e != hipSuccess) return hip_bad(e, "launch kv_plan");
        a.c.plan = pa;
        b.c.plan = pb;
    }
    const bool f32 = kv->dtype == FRQ_DT_F32, f16 = kv->dtype == FRQ_DT_F16;
    if (!ga) e = hipSuccess;
    else if (ex) e = f32 ? launch_decode_ex_f32(a, la) : f16 ? launch_decode_ex_f16(a, la) : launch_decode_ex_i8(a, la);
    else e = f32 ? launch_decode_f32(a, la) : f16 ? launch_decode_f16(a, la) : launch_decode_i8(a, la);
    if (e != hipSuccess) return hip_bad(e, "launch kv_decode");
    if (prompts) {
        if (ex) e = f32 ? launch_prompt_ex_f32(b, lb) : f16 ? launch_prompt_ex_f16(b, lb) : launch_prompt_ex_i8(b, lb);
        else e = f32 ? launch_prompt_f32(b, lb) : f16 ? launch_prompt_f16(b, lb) : launch_prompt_i8(b, lb);
        if (e != hipSuccess) return hip_bad(e, "launch kv_prompt");
    }
    if (ex) kv_join_kernel<true><<<dim3((unsigned)(ga + gb)), dim3(256), 0, s>>>(a, b, (unsigned)ga);
    else kv_join_kernel<false><<<dim3((unsigned)(ga + gb)), dim3(256), 0, s>>>(a, b, (unsigned)ga);
    e = hipGetLastError();
    return e == hipSuccess ? FRQ_OK : hip_bad(e, "launch kv_join");
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
    return std::max(plan_of(kv, n_row, n_head, n_seq, false, false, 0).bytes,
                    plan_of(kv, n_row, n_head, n_seq, true, false, 0).bytes);
}

int frq_kv_attn_dev(frq_ctx* ctx, const frq_kv* kv, const float* d_q, size_t q_pitch, size_t n_row, size_t n_head,
                    const int32_t* d_pages, size_t pages_pitch, const int32_t* d_len, const int32_t* d_first,
                    size_t n_seq, double scale, double cap, size_t window, float* d_out, size_t out_pitch, void* d_ws,
                    size_t ws_bytes) {
    return attend(ctx, kv, d_q, q_pitch, n_row, n_head, d_pages, pages_pitch, d_len, d_first, n_seq, scale, cap, window,
                  More{0, nullptr, 0, false}, d_out, out_pitch, d_ws, ws_bytes);
}

int frq_kv_attn_sink_dev(frq_ctx* ctx, const frq_kv* kv, const float* d_q, size_t q_pitch, size_t n_row, size_t n_head,
                         const int32_t* d_pages, size_t pages_pitch, const int32_t* d_len, const int32_t* d_first,
                         size_t n_seq, double scale, double cap, size_t window, size_t sinks, float* d_out,
                         size_t out_pitch, void* d_ws, size_t ws_bytes) {
    return attend(ctx, kv, d_q, q_pitch, n_row, n_head, d_pages, pages_pitch, d_len, d_first, n_seq, scale, cap, window,
                  More{sinks, nullptr, 0, false}, d_out, out_pitch, d_ws, ws_bytes);
}

int frq_kv_attn_tree_dev(frq_ctx* ctx, const frq_kv* kv, const float* d_q, size_t q_pitch, size_t n_row, size_t n_head,
                         const int32_t* d_pages, size_t pages_pitch, const int32_t* d_len, const int32_t* d_first,
                         size_t n_seq, double scale, double cap, size_t window, size_t sinks, const uint64_t* d_tree,
                         size_t tree_pitch, float* d_out, size_t out_pitch, void* d_ws, size_t ws_bytes) {
    return attend(ctx, kv, d_q, q_pitch, n_row, n_head, d_pages, pages_pitch, d_len, d_first, n_seq, scale, cap, window,
                  More{sinks, d_tree, tree_pitch, true}, d_out, out_pitch, d_ws, ws_bytes);
}

}  // extern "C"
