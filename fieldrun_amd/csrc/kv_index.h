// kv_index.h — where the rows, keys and pages of a paged attention call lie
// (plain functions, the same on the host and on the device).
//
// A call's work is cut into items: a tile of `tp` (query row, head) pairs of
// one sequence and kv head times a run of `chunk` of its keys.  Lengths and row
// offsets are device data, so every workgroup finds its own item from them:
// the chunk length follows from the whole call's keys (chunk_of), the items
// are numbered sequence after sequence, and the grid is the host's bound of
// their number (max_items).  A tile cut into several chunks leaves partial
// results in slots, at most max_slots.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define KV_HD __host__ __device__ inline
#else
#define KV_HD inline
#endif

namespace frq {
namespace kv {

constexpr int ALIGN = 32;  // a tile's first key of a window is rounded down to this

struct Call {
    const int32_t* len;    // [n_seq] cached tokens
    const int32_t* first;  // [n_seq + 1] row offsets, or null: row s is sequence s's
    int n_seq, n_row;      // sequences; rows of q
    int width, shift;      // page ids of a table row; log2 of the page
    int rep;               // query heads a kv head
    int window;            // keys seen at most (0: all)
    int n_kv;
    int tp;                // pairs a tile
    int min_pairs, max_pairs;  // the sequences served: pairs in [min, max]
    int64_t target;        // items wanted over all kv heads
    int min_chunk;         // keys a chunk at least, 64, 128 or 256
    const int32_t* plan;   // of many sequences: the chunk length and fills(), then before each 64 sequences (items, slots)
    int sinks, sink_span;  // with a window: first keys seen besides, and as a tile spans them (sink_keys; 0: none)
    const uint64_t* tree;  // bit masks of drafted tokens, a row of q each (null: rows see what lies before them)
    int64_t tree_pitch;    // words between the masks
    int even;              // items wanted where the tiles have nearly the same keys, up to target (0: target)
    int slots;             // or the items that fill the chip, up to target, for wanted() (0: target)
    int uncut;             // with a plan: drop_uncut()'s pairs (0: all that is served)
    bool prompt;           // and the launch
};

struct Seq {
    int row0, rows;  // its rows of q
    int len;         // its keys
    int ext;         // keys that a tile of it spans, at most
    int tiles;       // 0: not served
    bool bad;        // its length or offsets are out of range
};

KV_HD Seq seq_of(const Call& c, int len, int r0, int r1) {
    Seq q{r0, r1 - r0, len, 0, 0, false};
    if (r0 < 0 || r1 < r0 || r1 > c.n_row) {
        q.row0 = q.rows = q.len = 0;
        q.bad = true;
        return q;
    }
    if (len < 0 || (int64_t)len > ((int64_t)c.width << c.shift)) {
        q.len = 0;
        q.bad = true;
    }
    if (c.tree && (q.rows > q.len || (q.rows + 63) / 64 > c.tree_pitch)) {  // no room for its tree
        q.row0 = q.rows = q.len = 0;
        q.bad = true;
        return q;
    }
    const int64_t pairs = (int64_t)q.rows * c.rep;
    if (pairs < c.min_pairs || pairs > c.max_pairs) return q;
    q.tiles = (int)((pairs + c.tp - 1) / c.tp);
    // its window and its rows after the first (of a tree all, and the place
    // before it), the rounding of tile_lo, the sinks
    const int most = (c.tp - 1) / c.rep + 2, rows = c.tree ? q.rows + 1 : q.rows < most ? q.rows : most;
    const int64_t span = (int64_t)c.window + rows - 1 + ALIGN - 1 + c.sink_span;
    q.ext = c.window && span < q.len ? (int)span : q.len;
    return q;
}
KV_HD Seq seq_at(const Call& c, int s) {
    return c.first ? seq_of(c, c.len[s], c.first[s], c.first[s + 1]) : seq_of(c, c.len[s], s, s + 1);
}
KV_HD int64_t keys_of(const Seq& q) { return (int64_t)q.tiles * q.ext; }

// Keys a chunk when the call's tiles read `total` keys a kv head.  (32-bit
// divisions wherever the numbers allow: a 64-bit one is a hundred instructions
// and more, in every workgroup.)
constexpr int MOST = 0x7FFFFFFF / 64 * 64;
KV_HD int round_keys(uint32_t keys, int step) {  // up to a multiple of step, a power of two up to 256
    const uint32_t up = (keys + (uint32_t)step - 1) & ~((uint32_t)step - 1);
    return up > (uint32_t)MOST ? MOST : (int)up;
}
KV_HD int chunk_of(const Call& c, int64_t total, int64_t target) {
    const uint64_t x = (uint64_t)total * (uint64_t)c.n_kv + (uint64_t)target - 1;
    const uint64_t per = x >> 32 ? x / (uint64_t)target : (uint64_t)((uint32_t)x / (uint32_t)target);
    const int up = round_keys(per > (uint64_t)MOST ? (uint32_t)MOST : (uint32_t)per, c.min_chunk);
    return up < c.min_chunk ? c.min_chunk : up;
}
KV_HD int chunk_of(const Call& c, int64_t total) { return chunk_of(c, total, c.target); }
// The items that fill the chip less the chunks that every tile is rounded up by,
// half of them at least.
KV_HD int64_t wanted(const Call& c, int64_t tiles) {
    if (!c.slots) return c.target;
    const int64_t left = c.slots - tiles * c.n_kv;
    return left > c.slots / 2 ? left : c.slots / 2;
}
// The same where c.even is set, of `tiles` tiles of up to `most` keys.
KV_HD int chunk_of_even(const Call& c, int64_t total, int64_t tiles, int most) {
    if ((int64_t)most * tiles > total + total / 4) return chunk_of(c, total);
    if (!tiles || tiles * c.n_kv > c.even) return chunk_of(c, total, c.even);
    const uint32_t n = (uint32_t)c.even / ((uint32_t)tiles * (uint32_t)c.n_kv);  // chunks a tile: one round
    // (chunks of half the least for a few hundred keys, where a tile's latency counts: one
    // sequence of 1000 keys, 4 int8 heads of 128, 14.4 us in five chunks, 12.8 in nine; two
    // for 200 keys or sixteen for 2000 cost the joining more, 10.0 / 11.3, 12.1 / 13.1.
    // Several, 4 heads of 256: 2 f16 ones of 600 19.2 / 16.4, 4 of 1000 20.0 / 17.2, 8 int8
    // ones of 600 20.4 / 16.9; 16 and more the same but f16 of 1500, 27.3 / 29.7)
    const int least = most > 256 && most <= 12 * 128 && c.min_chunk > 128 ? 128 : c.min_chunk;
    const int up = round_keys(((uint32_t)most + n - 1) / n, least);
    return up < least ? least : up;
}
KV_HD int chunks_of(const Seq& q, int chunk) {
    const int n = (int)(((uint32_t)q.ext + (uint32_t)chunk - 1) / (uint32_t)chunk);
    return n < 1 ? 1 : n;
}
// A sequence's own chunk: its keys in n runs of equal length, whole STEPs.
constexpr int STEP = 64;
KV_HD int even_chunk(const Seq& q, int n) {
    const int up = round_keys(((uint32_t)q.ext + (uint32_t)n - 1) / (uint32_t)n, STEP);
    return up < STEP ? STEP : up;
}
// Host bounds.  Tiles: sum of ceil(rows rep / tp) <= n_row rep / tp + n_seq,
// and no more than a sequence of max_pairs has for each;
// items: sum of tiles ceil(ext / chunk) <= tiles + total / chunk and
// total / chunk <= target / n_kv; slots, over the sequences of several
// chunks only: ceil(x) < 2 x for x > 1.
KV_HD int64_t max_tiles(const Call& c) {
    const int64_t by_row = (int64_t)c.n_row * ((c.rep + c.tp - 1) / c.tp);  // no tile for less than a row
    const int64_t by_seq = (int64_t)c.n_seq * (((int64_t)c.max_pairs + c.tp - 1) / c.tp);
    const int64_t all = (int64_t)c.n_row * c.rep / c.tp + c.n_seq;
    const int64_t least = all < by_row ? all : by_row;
    return least < by_seq ? least : by_seq;
}
KV_HD int64_t max_items(const Call& c) { return max_tiles(c) + c.target / c.n_kv + 1; }
// A prompt launch that has no room for parts takes its sequences, of uncut pairs and
// more, where they fill it: their tiles' keys, of which a workgroup walks one tile's,
// come to those of LONE workgroups with the longest.  Else the decode launch does.
// (The keys without a window's rows and roundings: the same for both launches.)
constexpr int LONE = 128;
KV_HD int lone_keys(const Call& c, const Seq& q) {
    const int64_t span = (int64_t)c.window + c.sinks;
    return c.window && span < q.len ? (int)span : q.len;
}
KV_HD int64_t lone_tiles(const Call& c, const Seq& q) { return ((int64_t)q.rows * c.rep + 127) >> 7; }
KV_HD bool fills(int64_t total, int most, int n_kv) { return total > 0 && total * n_kv >= (int64_t)most * LONE; }
// What of a sequence one of both launches serves then (the decode launch's max_pairs
// and the prompt launch's min_pairs let it through).
KV_HD void drop_uncut(const Call& c, bool filled, Seq& q) {
    if (c.prompt ? !filled : filled && (int64_t)q.rows * c.rep >= c.uncut) q.tiles = 0;
}
// More sequences than this are summed once for the call, into a plan.
constexpr int PLAN_SEQS = 64;
KV_HD int64_t plan_words(int64_t n_seq) { return n_seq > PLAN_SEQS ? 2 + (n_seq + 63) / 64 * 2 : 0; }
KV_HD int64_t max_slots(int64_t target, int n_kv) { return 2 * (target / n_kv + 1); }

// The first key that the row at position pos sees (the last one is pos), and
// where the chunks of a tile begin whose first row is at pos.
KV_HD int key_lo(const Call& c, int pos) { return c.window && pos - c.window + 1 > 0 ? pos - c.window + 1 : 0; }

KV_HD int tile_lo(const Call& c, int pos) { return key_lo(c, pos) / ALIGN * ALIGN; }

// With sinks a tile takes the keys 0 .. span - 1 first, and then goes on at
// key span + gap; where its window begins no later, the keys from 0 on.
// Without, it begins at key gap.
struct Span {
    int span, gap;
};
KV_HD Span span_at(const Call& c, int pos) {
    const int lo = tile_lo(c, pos);
    if (!c.sinks) return Span{0, lo};
    return lo > c.sink_span ? Span{c.sink_span, lo - c.sink_span} : Span{0, 0};
}
KV_HD int sink_keys(int64_t sinks, int step) { return (int)((sinks + step - 1) / step * step); }  // whole tiles

// Which of the N drafted tokens from t on (t may be below 0) a mask of n tokens
// has, as bits; n 0: no mask is read.
template <int N>
KV_HD uint32_t tree_bits(const uint64_t* mask, int n, int t) {
    static_assert(N <= 16, "");
    if (n <= 0 || t <= -N || t >= n) return 0;
    const int w = t > 0 ? t >> 6 : 0, sh = t & 63;
    uint64_t m = mask[w];
    if (t < 0) {
        m <<= -t;
    } else if (sh) {
        m >>= sh;
        if (sh > 64 - N && 64 * (w + 1) < n) m |= mask[w + 1] << (64 - sh);
    }
    const int left = n - t;  // bits past the tree count for nothing
    return (uint32_t)m & ((1u << (left < N ? left : N)) - 1);
}

// A key's page id where the table holds one, else -1.
KV_HD int page_ok(int id, int64_t n_pages) { return id >= 0 && (int64_t)id < n_pages ? id : -1; }

// A slot of the cache: page and place; false for one that is not in it.
KV_HD bool slot_of(int64_t slot, int shift, int64_t n_pages, int64_t* page, int* off) {
    *page = slot >> shift;
    *off = (int)(slot & (((int64_t)1 << shift) - 1));
    return slot >= 0 && *page < n_pages;
}

}  // namespace kv
}  // namespace frq
