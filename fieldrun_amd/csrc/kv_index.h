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
    const int32_t* plan;   // of many sequences: the chunk length and 0, then before each 64 sequences (items, slots)
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
    const int64_t pairs = (int64_t)q.rows * c.rep;
    if (pairs < c.min_pairs || pairs > c.max_pairs) return q;
    q.tiles = (int)((pairs + c.tp - 1) / c.tp);
    // its window and its rows after the first, and the rounding of tile_lo
    const int most = (c.tp - 1) / c.rep + 2, rows = q.rows < most ? q.rows : most;
    const int64_t span = (int64_t)c.window + rows - 1 + ALIGN - 1;
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
KV_HD int chunk_of(const Call& c, int64_t total) {
    const uint64_t x = (uint64_t)total * (uint64_t)c.n_kv + (uint64_t)c.target - 1;
    const uint64_t per = x >> 32 ? x / (uint64_t)c.target : (uint64_t)((uint32_t)x / (uint32_t)c.target);
    const int up = round_keys(per > (uint64_t)MOST ? (uint32_t)MOST : (uint32_t)per, c.min_chunk);
    return up < c.min_chunk ? c.min_chunk : up;
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
// More sequences than this are summed once for the call, into a plan.
constexpr int PLAN_SEQS = 64;
KV_HD int64_t plan_words(int64_t n_seq) { return n_seq > PLAN_SEQS ? 2 + (n_seq + 63) / 64 * 2 : 0; }
KV_HD int64_t max_slots(int64_t target, int n_kv) { return 2 * (target / n_kv + 1); }

// The first key that the row at position pos sees (the last one is pos), and
// where the chunks of a tile begin whose first row is at pos.
KV_HD int key_lo(const Call& c, int pos) { return c.window && pos - c.window + 1 > 0 ? pos - c.window + 1 : 0; }

KV_HD int tile_lo(const Call& c, int pos) { return key_lo(c, pos) / ALIGN * ALIGN; }

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
