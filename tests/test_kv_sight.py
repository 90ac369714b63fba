"""Attention with sinks and trees without a GPU: the refusals, and the index
arithmetic of kv_index.h on the host: the chunks of a tile cover every key that
one of its rows sees once, within the bounds that the host launches by."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

import fieldrun_amd as fa
from test_kv import A, BAD_CACHES, ROOT, desc, message


def call(d=None, tree=A, tree_pitch=1, sinks=4, q=A, qp=256, n_row=3, n_head=4, pages=A, width=5, lens=A, first=None, n_seq=3,
         scale=0.1, cap=0.0, window=9, out=A, op=256, ws=A, ws_bytes=1 << 40, trees=True):
    d = C.byref(desc()) if d is None else d
    args = (None, d, q, qp, n_row, n_head, pages, width, lens, first, n_seq, scale, cap, window, sinks)
    to = (out, op, ws, ws_bytes)
    if trees:
        return fa.lib.frq_kv_attn_tree_dev(*args, tree, tree_pitch, *to)
    return fa.lib.frq_kv_attn_sink_dev(*args, *to)


@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("change,code,word", BAD_CACHES)
def test_bad_descriptors_are_refused(change, code, word, trees):
    assert call(C.byref(desc(**change)), trees=trees) == code and word in message(), message()


@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("change,word", [
    (dict(n_head=3), "n_head"), (dict(n_row=4), "one row"), (dict(qp=255), "pitch"), (dict(op=100), "pitch"),
    (dict(n_row=1 << 31, n_seq=1 << 31), "too many"), (dict(width=1 << 28), "2^31"), (dict(scale=float("nan")), "scale"),
    (dict(cap=-1.0), "cap"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(lens=None), "null"),
    (dict(pages=None), "null"), (dict(ws=A + 4), "16-byte"), ({}, "null context"), (dict(sinks=1 << 63), "null context"),
    (dict(window=0, sinks=0), "null context"), (dict(n_row=0, n_seq=0, q=None, out=None, lens=None), "null context"),
])
def test_bad_calls_are_refused(change, word, trees):
    assert call(trees=trees, **change) == fa.FRQ_ERR_ARG and word in message(), message()


@pytest.mark.parametrize("change,word", [(dict(tree=None), "null pointer"), (dict(tree_pitch=0), "tree"),
                                         (dict(tree_pitch=1 << 41), "tree"),
                                         (dict(tree=None, n_row=0, n_seq=0), "null context")])
def test_bad_trees_are_refused(change, word):
    assert call(**change) == fa.FRQ_ERR_ARG and word in message(), message()


SRC = r"""
#include "kv_index.h"
using namespace frq::kv;
struct Row { int32_t seq, tile, chunk, chunks, row0, rows, len, span, gap, ext, klen; };
extern "C" int64_t plan(const int32_t* len, const int32_t* first, int n_seq, int n_row, int rep, int window, int sinks, int step,
                        int trees, int tree_pitch, int n_kv, int tp, int64_t target, int min_chunk, Row* out, int64_t cap,
                        int64_t* bounds, int* bad) {
    Call c{len, first, n_seq, n_row, 8192, 4, rep, window, n_kv, tp, 1, 0x7FFFFFFF, target, min_chunk};
    c.sinks = sinks;
    c.sink_span = sink_keys(sinks, step);
    c.tree = trees ? (const uint64_t*)8 : nullptr;
    c.tree_pitch = tree_pitch;
    int64_t total = 0, n = 0, slots = 0;
    *bad = 0;
    for (int s = 0; s < n_seq; ++s) { const Seq q = seq_at(c, s); total += keys_of(q); *bad += q.bad; }
    const int klen = chunk_of(c, total);
    for (int s = 0; s < n_seq; ++s) {
        const Seq q = seq_at(c, s);
        const int m = chunks_of(q, klen);
        for (int t = 0; t < q.tiles; ++t)
            for (int k = 0; k < m; ++k) {
                const int base = q.len - q.rows;
                const Span sp = span_at(c, trees ? base - 1 : base + (int)((int64_t)t * tp / rep));
                if (n < cap) out[n] = Row{s, t, k, m, q.row0, q.rows, q.len, sp.span, sp.gap, q.ext, even_chunk(q, m)};
                ++n;
                if (m > 1) ++slots;
            }
    }
    bounds[0] = max_items(c);
    bounds[1] = max_slots(target, n_kv);
    bounds[2] = slots;
    return n;
}
extern "C" uint32_t bits(const uint64_t* mask, int n, int t, int of) {
    return of == 1 ? tree_bits<1>(mask, n, t) : of == 4 ? tree_bits<4>(mask, n, t) : of == 8 ? tree_bits<8>(mask, n, t)
                                                                                            : tree_bits<16>(mask, n, t);
}
"""


class Row(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("seq", "tile", "chunk", "chunks", "row0", "rows", "len", "span", "gap", "ext", "klen")]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_sight")
    (d / "plan.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "fieldrun_amd", "csrc"), str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = C.CDLL(str(d / "plan.so"))
    lib.plan.restype = C.c_int64
    lib.plan.argtypes = [C.c_void_p, C.c_void_p] + [C.c_int] * 10 + [C.c_int64, C.c_int, C.c_void_p, C.c_int64, C.c_void_p,
                                                                     C.c_void_p]
    lib.bits.restype = C.c_uint32
    lib.bits.argtypes = [C.c_void_p] + [C.c_int] * 3
    return lib


@pytest.mark.parametrize("of", [1, 4, 8, 16])
def test_bits_of_a_mask(host, of):
    """Around a tree's first and last token and its words' borders; bits past
    its tokens count for nothing, and without a tree nothing is read."""
    rng = random.Random(of)
    for n in (1, 3, 63, 64, 65, 127, 128, 129, 200):
        words = -(-n // 64)
        mask = [rng.getrandbits(64) for _ in range(words)]
        m = (C.c_uint64 * words)(*mask)  # not a word more
        for t in range(-20, n + 20):
            want = sum((0 <= t + j < n and mask[(t + j) // 64] >> (t + j) % 64 & 1) << j for j in range(of))
            assert host.bits(m, n, t, of) == want
    for t in range(-20, 20):
        assert host.bits(None, 0, t, of) == 0


def plan(host, lens, first, rep, window, sinks, step, trees, pitch=64, n_kv=4, tp=16, target=512, least=256):
    n, cap = len(lens), 200000
    out, bounds, bad = (Row * cap)(), (C.c_int64 * 3)(), C.c_int()
    cf = (C.c_int32 * (n + 1))(*first) if first else None
    m = host.plan((C.c_int32 * n)(*lens), cf, n, first[-1] if first else n, rep, window, sinks, step, int(trees), pitch, n_kv,
                  tp, target, least, out, cap, bounds, C.byref(bad))
    assert m <= cap
    return [out[i] for i in range(m)], list(bounds), bad.value


def test_chunks_cover_what_rows_see(host):
    rng = random.Random(4)
    for _ in range(400):
        n = rng.choice([1, 2, 5, 70])
        top = rng.choice([40, 700, 9000, 100000])
        trees = rng.random() < 0.5
        lens = [rng.choice([0, 1, rng.randint(0, top), top]) for _ in range(n)]
        decode = rng.random() < 0.4 and all(lens)
        rows = [1] * n if decode else [rng.choice([0, 1, rng.randint(0, 300)]) for _ in range(n)]
        if trees:
            rows = [min(a, b) for a, b in zip(rows, lens)]
        first = None if decode else [sum(rows[:i]) for i in range(n + 1)]
        window = rng.choice([0, 1, 33, 100, 4096])
        sinks = rng.choice([0, 1, 4, 33, 64, 500, 100000]) if window else 0
        rep, tp, step = rng.choice([1, 3, 7, 16]), rng.choice([16, 128]), rng.choice([32, 64])
        items, bounds, bad = plan(host, lens, first, rep, window, sinks, step, trees, tp=tp)
        assert bad == 0 and len(items) <= bounds[0] and bounds[2] <= bounds[1]
        parts = {}
        for i in items:
            parts.setdefault((i.seq, i.tile), []).append(i)
        assert len(parts) == sum(-(-r * rep // tp) for r in rows)
        for (s, t), p in parts.items():
            span, gap, base = p[0].span, p[0].gap, lens[s] - rows[s]
            assert span % step == 0 and gap % 32 == 0 and gap >= 0
            assert [x.chunk for x in p] == list(range(p[0].chunks))
            a, b = t * tp // rep, (min((t + 1) * tp, rows[s] * rep) - 1) // rep
            last = lens[s] - 1 if trees else base + b
            # the tile's keys are 0 .. span - 1 and span + gap .. last, in runs of klen
            assert p[0].chunks * p[0].klen >= last + 1 - gap
            lows = [base - 1, base] if trees else [base + a]  # the places that the first row may stand at
            for low in lows:
                lo = max(0, low - window + 1) if window else 0
                assert span + gap <= lo or (span == 0 and gap <= lo) or (span + gap == 0)
                if sinks and low >= 0 and span + gap > 0:
                    assert span >= min(sinks, lo)


def test_trees_without_room_are_told(host):
    for lens, first, pitch, want in (([70], [0, 70], 2, 0), ([70], [0, 70], 1, 1), ([69], [0, 70], 2, 1), ([64], [0, 64], 1, 0),
                                     ([0, 5], [0, 1, 3], 1, 1), ([0, 5], [0, 0, 5], 1, 0), ([5, -1], [0, 5, 7], 1, 1)):
        items, _, bad = plan(host, lens, first, 3, 0, 0, 32, True, pitch)
        assert bad == want
        assert all(i.rows <= i.len for i in items)
    assert plan(host, [5], [0, 9], 3, 0, 0, 32, False)[2] == 0  # more rows than tokens: not of trees alone


EVEN = r"""
#include "kv_index.h"
using namespace frq::kv;
extern "C" int64_t even(int n_seq, const int32_t* tiles, const int32_t* ext, int n_row, int rep, int n_kv, int tp, int64_t target,
                        int64_t even, int min_chunk, int64_t* out) {
    Call c{nullptr, nullptr, n_seq, n_row, 8192, 4, rep, 0, n_kv, tp, 1, 0x7FFFFFFF, target, min_chunk};
    c.even = even;
    int64_t total = 0, all = 0, items = 0, slots = 0;
    int most = 0;
    for (int s = 0; s < n_seq; ++s) {
        total += (int64_t)tiles[s] * ext[s];
        all += tiles[s];
        if (tiles[s] && ext[s] > most) most = ext[s];
    }
    const int klen = chunk_of_even(c, total, all, most);
    for (int s = 0; s < n_seq; ++s) {
        Seq q{0, 0, 0, ext[s], tiles[s], false};
        const int n = chunks_of(q, klen);
        items += (int64_t)tiles[s] * n;
        if (n > 1) slots += (int64_t)tiles[s] * n;
    }
    out[0] = klen;
    out[1] = items;
    out[2] = slots;
    out[3] = all + target / n_kv + 1;
    out[4] = max_slots(target, n_kv);
    return chunk_of(c, total);
}
"""


def test_chunks_of_even_tiles_keep_the_bounds(tmp_path):
    """Tiles of nearly the same keys fill one round of `even` items and no more,
    others are cut as ever; neither passes the host's bounds."""
    (tmp_path / "even.cpp").write_text(EVEN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "fieldrun_amd", "csrc"), str(tmp_path / "even.cpp"), "-o", str(tmp_path / "even.so")],
                   check=True)
    lib = C.CDLL(str(tmp_path / "even.so"))
    lib.even.restype = C.c_int64
    lib.even.argtypes = [C.c_int, C.c_void_p, C.c_void_p] + [C.c_int] * 4 + [C.c_int64] * 2 + [C.c_int, C.c_void_p]
    rng = np.random.default_rng(3)
    rounds = 0
    for i in range(3000):
        n = int(rng.integers(1, 65))
        most = int(10 ** rng.uniform(0, 9 if i % 3 == 0 else 5))
        low = most if i % 2 else max(0, int(most * rng.uniform(0.5, 1)))
        ext = rng.integers(low, most + 1, n).astype(np.int32) if i % 5 else rng.integers(0, most + 1, n).astype(np.int32)
        tiles = rng.integers(0, 4, n).astype(np.int32) if i % 4 else np.ones(n, np.int32)
        kv, step = int(rng.choice([1, 2, 4, 5, 8, 64, 600])), int(rng.choice([128, 256]))
        out = np.zeros(5, np.int64)
        plain = lib.even(n, tiles.ctypes.data, ext.ctypes.data, n, 1, kv, 16, 512, 256, step, out.ctypes.data)
        klen, items, slots, most_items, most_slots = out.tolist()
        assert klen % 64 == 0 and klen >= min(step, 128) and items <= most_items and slots <= most_slots, (i, out)
        total, top = int((tiles.astype(np.int64) * ext).sum()), int(ext[tiles > 0].max(initial=0))
        if top * int(tiles.sum()) > total + total // 4:
            assert klen == plain
        elif 0 < int(tiles.sum()) * kv <= 256:
            rounds += 1
            assert items * kv <= 256
    assert rounds > 300


WANTED = r"""
#include "kv_index.h"
using namespace frq::kv;
extern "C" int64_t items(int64_t slots, int64_t target, int64_t tiles, int n_kv) {
    Call c{};
    c.target = target;
    c.slots = slots;
    c.n_kv = n_kv;
    return wanted(c, tiles);
}
"""


def test_items_wanted_stay_within_the_target(tmp_path):
    (tmp_path / "w.cpp").write_text(WANTED)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "fieldrun_amd", "csrc"), str(tmp_path / "w.cpp"), "-o", str(tmp_path / "w.so")], check=True)
    lib = C.CDLL(str(tmp_path / "w.so"))
    lib.items.restype = C.c_int64
    lib.items.argtypes = [C.c_int64] * 3 + [C.c_int]
    for tiles in (0, 1, 20, 64, 128, 1000, 1 << 31):
        for kv in (1, 4, 65535):
            assert lib.items(0, 400, tiles, kv) == 400
            assert lib.items(512, 512, tiles, kv) == max(256, 512 - tiles * kv)


UNCUT = r"""
#include "kv_index.h"
using namespace frq::kv;
// sequences that each launch serves, and whether the prompt launch is filled
extern "C" int uncut(const int32_t* len, const int32_t* first, int n_seq, int rep, int n_kv, int window, int pairs, int* dec,
                     int* prompt) {
    Call a{len, first, n_seq, first[n_seq], 8192, 4, rep, window, n_kv, 16, 1, 0x7FFFFFFF, 512, 128};
    Call b = a;
    a.uncut = b.uncut = b.min_pairs = pairs;
    b.tp = 128;
    b.prompt = true;
    int64_t total = 0;
    int most = 0;
    for (int s = 0; s < n_seq; ++s) {
        const Seq x = seq_at(a, s), y = seq_at(b, s);  // (the launches sum their own)
        if (!y.tiles) continue;
        if (lone_tiles(a, x) != y.tiles || lone_tiles(b, y) != y.tiles || lone_keys(a, x) != lone_keys(b, y)) return -1;
        total += lone_tiles(b, y) * lone_keys(b, y);
        if (lone_keys(b, y) > most) most = lone_keys(b, y);
    }
    const bool filled = fills(total, most, n_kv);
    for (int s = 0; s < n_seq; ++s) {
        Seq x = seq_at(a, s), y = seq_at(b, s);
        drop_uncut(a, filled, x);
        drop_uncut(b, filled, y);
        dec[s] = x.tiles;
        prompt[s] = y.tiles;
    }
    return filled;
}
"""


def test_a_launch_that_cuts_no_keys_is_filled(tmp_path):
    """A batch with idle sequences: each sequence is served once, and by workgroups
    that walk all of its keys only where all of these have 128 times the longest."""
    (tmp_path / "u.cpp").write_text(UNCUT)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "fieldrun_amd", "csrc"), str(tmp_path / "u.cpp"), "-o", str(tmp_path / "u.so")], check=True)
    lib = C.CDLL(str(tmp_path / "u.so"))
    lib.uncut.argtypes = [C.c_void_p] * 2 + [C.c_int] * 5 + [C.c_void_p] * 2
    rng = np.random.default_rng(7)
    seen = [0, 0]
    for _ in range(1500):
        n = int(rng.integers(65, 400))
        rows = np.where(rng.random(n) < 10.0 ** rng.uniform(-2.5, 0), 10.0 ** rng.uniform(0, rng.choice([1.0, 2.5])), 0).astype(np.int32)
        lens = np.maximum(rows, 10.0 ** rng.uniform(0, rng.choice([2.0, 4.9]), n)).astype(np.int32)
        first = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        rep, kv, pairs = int(rng.choice([1, 4, 7, 64])), int(rng.choice([1, 2, 8, 129])), int(rng.choice([33, 129]))
        window = int(rng.choice([0, 100]))
        dec, prompt = np.zeros(n, np.int32), np.zeros(n, np.int32)
        filled = lib.uncut(lens.ctypes.data, first.ctypes.data, n, rep, kv, window, pairs, dec.ctypes.data, prompt.ctypes.data)
        large = rows.astype(np.int64) * rep >= pairs
        assert ((dec > 0) != (prompt > 0))[rows > 0].all() and not (dec + prompt)[rows == 0].any()
        assert ((prompt > 0) == (large & bool(filled))).all()
        if large.any():
            own = np.minimum(lens[large], window or 1 << 30)
            assert bool(filled) == ((-(-rows[large].astype(np.int64) * rep // 128) * own).sum() * kv >= 128 * int(own.max()))
        seen[filled] += 1
    assert min(seen) > 200, seen
    # one tree of 112 pairs beside idle sequences, many alike
    for rows, want in (([16] + [0] * 79, 0), ([16] * 64 + [0] * 16, 1), ([16] * 63 + [0] * 17, 0)):
        first = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        lens, out = np.full(80, 32768, np.int32), np.zeros((2, 80), np.int32)
        assert lib.uncut(lens.ctypes.data, first.ctypes.data, 80, 7, 2, 0, 33, out[0].ctypes.data, out[1].ctypes.data) == want


FILLED = r"""
#include "kv_index.h"
using namespace frq::kv;
extern "C" void filled(const int32_t* len, const int32_t* first, int n_seq, int rep, int n_kv, int window, int sinks, int trees,
                       int64_t want, int least, int64_t* out) {
    Call c{len, first, n_seq, first[n_seq], 1 << 17, 10, rep, window, n_kv, 128, least, 0x7FFFFFFF, want, 128};
    c.sinks = sinks;
    c.sink_span = sink_keys(sinks, 64);
    c.tree = trees ? (const uint64_t*)8 : nullptr;
    c.tree_pitch = 64;
    c.slots = want;
    int64_t total = 0, tiles = 0, items = 0, slots = 0;
    for (int s = 0; s < n_seq; ++s) { const Seq q = seq_at(c, s); total += keys_of(q); tiles += q.tiles; }
    const int klen = chunk_of(c, total, wanted(c, tiles));
    for (int s = 0; s < n_seq; ++s) {
        const Seq q = seq_at(c, s);
        const int n = q.tiles ? chunks_of(q, klen) : 1;
        items += (int64_t)q.tiles * n;
        if (n > 1) slots += (int64_t)q.tiles * n;
    }
    out[0] = items;
    out[1] = max_items(c);
    out[2] = slots;
    out[3] = max_slots(want, n_kv);
}
"""


def test_chunks_of_the_items_wanted_keep_the_bounds(tmp_path):
    """The prompt launch of calls with sinks or trees, as kernels cut it: no more
    items than its grid and records, no more parts than its workspace."""
    (tmp_path / "f.cpp").write_text(FILLED)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "fieldrun_amd", "csrc"), str(tmp_path / "f.cpp"), "-o", str(tmp_path / "f.so")], check=True)
    lib = C.CDLL(str(tmp_path / "f.so"))
    lib.filled.argtypes = [C.c_void_p] * 2 + [C.c_int] * 6 + [C.c_int64, C.c_int, C.c_void_p]
    lib.filled.restype = None
    rng, cut = np.random.default_rng(11), 0
    for i in range(4000):
        n = int(rng.choice([1, 2, 5, 20, 64, 300]))
        lens = (10.0 ** rng.uniform(0, rng.choice([2.0, 4.5, 8.0]), n)).astype(np.int32)
        rows = np.minimum(lens, 10.0 ** rng.uniform(0, rng.choice([1.0, 2.0, 3.6]), n)).astype(np.int32)
        rows[rng.random(n) < rng.choice([0.0, 0.5])] = 0
        if i % 3 == 0:
            lens[:], rows[:] = lens[0], rows[0]
        first = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        window = int(rng.choice([0, 1, 100, 4096]))
        out = np.zeros(4, np.int64)
        lib.filled(lens.ctypes.data, first.ctypes.data, n, int(rng.choice([1, 3, 7, 16])), int(rng.choice([1, 2, 4, 5, 8, 64, 600])),
                   window, int(rng.choice([0, 4, 500])) if window else 0, i % 2, int(rng.choice([256, 512])),
                   int(rng.choice([1, 33, 129])), out.ctypes.data)
        items, most_items, slots, most_slots = out.tolist()
        assert items <= most_items and slots <= most_slots, (i, out)
        cut += slots > 0
    assert cut > 500
