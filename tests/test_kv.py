"""The paged cache and the int8 norm without a GPU: every refusal that needs
none (checked before the context, so a null context shows it was reached),
and the index arithmetic of kv_index.h, compiled for the host: the items of
a call cover each (tile, key) once, within the bounds the host launches and
sizes its workspace by; bad lengths, offsets, pages and slots are told."""
import ctypes as C
import os
import random
import subprocess

import pytest

import fieldrun_amd as fa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 0x10000  # a 16-byte aligned address that is never read


def desc(kind="f16", n_pages=4, page=16, n_kv=2, hd=64, k=A, v=A, ks=None, vs=None, ps=0, ss=0):
    return fa._Kv(fa.KvCache.KINDS.get(kind, 99), n_pages, page, n_kv, hd, k, v, ks, vs, ps, ss)


def message():
    return fa.lib.frq_last_error().decode()


BAD_CACHES = [
    (dict(kind="?"), fa.FRQ_ERR_DTYPE, "dtype"),
    (dict(n_pages=0), fa.FRQ_ERR_ARG, "n_pages"), (dict(n_pages=1 << 31), fa.FRQ_ERR_ARG, "n_pages"),
    (dict(page=8), fa.FRQ_ERR_ARG, "page"), (dict(page=48), fa.FRQ_ERR_ARG, "page"),
    (dict(page=2048), fa.FRQ_ERR_ARG, "page"), (dict(n_kv=0), fa.FRQ_ERR_ARG, "n_kv"),
    (dict(n_kv=70000), fa.FRQ_ERR_ARG, "n_kv"), (dict(hd=0), fa.FRQ_ERR_ARG, "hd"),
    (dict(hd=72), fa.FRQ_ERR_ARG, "hd"), (dict(hd=272), fa.FRQ_ERR_ARG, "hd"),
    (dict(k=None), fa.FRQ_ERR_ARG, "null"), (dict(v=None), fa.FRQ_ERR_ARG, "null"),
    (dict(k=A + 8), fa.FRQ_ERR_ARG, "aligned"), (dict(v=A + 4), fa.FRQ_ERR_ARG, "aligned"),
    (dict(ps=100), fa.FRQ_ERR_ARG, "overlap"), (dict(ps=2049), fa.FRQ_ERR_ARG, "aligned"),
    (dict(kind="rowi8"), fa.FRQ_ERR_ARG, "scale"), (dict(kind="rowi8", ks=A, vs=A + 4), fa.FRQ_ERR_ARG, "aligned"),
    (dict(kind="rowi8", ks=A, vs=A, ss=16), fa.FRQ_ERR_ARG, "overlap"),
    (dict(kind="rowi8", ks=A, vs=A, ss=34), fa.FRQ_ERR_ARG, "aligned"),
]


@pytest.mark.parametrize("change,code,word", BAD_CACHES)
def test_bad_descriptors_are_refused_by_every_call(change, code, word):
    d = C.byref(desc(**change))
    for rc in (lambda: fa.lib.frq_kv_write_dev(None, d, A, A, 1 << 20, A, 1),
               lambda: fa.lib.frq_kv_read_dev(None, d, A, 1, A, A, 1 << 20),
               lambda: attn(d)):
        assert rc() == code and word in message(), message()


def attn(d=None, q=A, qp=256, n_row=3, n_head=4, pages=A, width=5, lens=A, first=None, n_seq=3, scale=0.1, cap=0.0,
         window=0, out=A, op=256, ws=A, ws_bytes=1 << 40):
    d = C.byref(desc()) if d is None else d
    return fa.lib.frq_kv_attn_dev(None, d, q, qp, n_row, n_head, pages, width, lens, first, n_seq, scale, cap, window,
                                  out, op, ws, ws_bytes)


@pytest.mark.parametrize("change,word", [
    (dict(n_head=3), "n_head"), (dict(n_head=0), "n_head"), (dict(n_row=4), "one row"), (dict(qp=255), "pitch"),
    (dict(op=100), "pitch"), (dict(n_row=1 << 31, n_seq=1 << 31), "too many"), (dict(width=1 << 28), "2^31"),
    (dict(n_row=1 << 30, n_seq=1 << 30, n_head=8, qp=512, op=512), "too many"),
    (dict(width=(1 << 27) - 63), "2^31"), (dict(scale=1e300), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(cap=-1.0), "cap"),
    (dict(cap=float("nan")), "cap"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(lens=None), "null"),
    (dict(pages=None), "null"), (dict(ws=A + 4), "16-byte"), ({}, "null context"),
])
def test_bad_attention_calls_are_refused(change, word):
    assert attn(**change) == fa.FRQ_ERR_ARG and word in message(), message()


def test_bad_rows_are_refused():
    d = C.byref(desc())
    for args, word in (((None, A, 128, A, 1), "null"), ((A, None, 128, A, 1), "null"), ((A, A, 128, None, 1), "null"),
                       ((A, A, 127, A, 1), "pitch"), ((A, A, 128, A, 1 << 40), "too many"),
                       ((A, A, 128, A, 1), "null context")):
        assert fa.lib.frq_kv_write_dev(None, d, *args) == fa.FRQ_ERR_ARG and word in message()
        k, v, pitch, slot, n = args
        assert fa.lib.frq_kv_read_dev(None, d, slot, n, k, v, pitch) == fa.FRQ_ERR_ARG and word in message()
    assert fa.lib.frq_kv_write_dev(None, None, A, A, 128, A, 1) == fa.FRQ_ERR_ARG and "null cache" in message()


@pytest.mark.parametrize("change,word", [
    (dict(k=0), "k must"), (dict(k=28673), "k must"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(x=None), "null pointer"), (dict(w=None), "null pointer"), (dict(a8=None), "null pointer"),
    (dict(sa=None), "null pointer"), (dict(a8=A + 2), "aligned"), (dict(m=1 << 31), "rows"), ({}, "null context"),
])
def test_bad_norms_are_refused(change, word):
    c = dict(x=A, y=None, w=A, eps=1e-6, m=2, k=64, s=None, a8=A, sa=A, oi=A, ov=A, **{})
    c.update(change)
    rc = fa.lib.frq_norm_quant_i8_dev(None, *c.values())
    assert rc == fa.FRQ_ERR_ARG and word in message(), message()


def test_unknown_kind():
    with pytest.raises(fa.FrqError) as e:
        fa.KvCache(None, "bf16", 1, 16, 1, 16, A, A)
    assert e.value.code == fa.FRQ_ERR_DTYPE


# ---- kv_index.h on the host ---------------------------------------------------

SRC = r"""
#include "kv_index.h"
using namespace frq::kv;
struct Row { int32_t seq, tile, chunk, chunks, row0, rows, len, lo, ext, klen; int64_t slot; };
extern "C" int64_t plan(const int32_t* len, const int32_t* first, int n_seq, int n_row, int width, int shift, int rep,
                        int window, int n_kv, int tp, int minp, int maxp, int64_t target, int min_chunk, Row* out,
                        int64_t cap, int64_t* bounds, int* bad) {
    Call c{len, first, n_seq, n_row, width, shift, rep, window, n_kv, tp, minp, maxp, target, min_chunk};
    int64_t total = 0, n = 0, slots = 0;
    *bad = 0;
    for (int s = 0; s < n_seq; ++s) { const Seq q = seq_at(c, s); total += keys_of(q); *bad += q.bad; }
    const int klen = chunk_of(c, total);
    for (int s = 0; s < n_seq; ++s) {
        const Seq q = seq_at(c, s);
        const int m = chunks_of(q, klen);
        for (int t = 0; t < q.tiles; ++t)
            for (int k = 0; k < m; ++k) {
                if (n < cap) out[n] = Row{s, t, k, m, q.row0, q.rows, q.len,
                                       tile_lo(c, q.len - q.rows + (int)((int64_t)t * tp / rep)), q.ext, even_chunk(q, m), m > 1 ? slots : -1};
                ++n;
                if (m > 1) ++slots;
            }
    }
    bounds[0] = max_items(c);
    bounds[1] = max_slots(target, n_kv);
    bounds[2] = slots;
    return n;
}
extern "C" int slot(int64_t s, int shift, int64_t n_pages, int64_t* page, int* off) { return slot_of(s, shift, n_pages, page, off); }
extern "C" int page(int id, int64_t n_pages) { return page_ok(id, n_pages); }
"""


class Row(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("seq", "tile", "chunk", "chunks", "row0", "rows", "len", "lo", "ext", "klen")
                ] + [("slot", C.c_int64)]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_index")
    (d / "plan.cpp").write_text(SRC)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "fieldrun_amd", "csrc"), str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = C.CDLL(str(d / "plan.so"))
    lib.plan.restype = C.c_int64
    lib.plan.argtypes = [C.c_void_p, C.c_void_p] + [C.c_int] * 10 + [C.c_int64, C.c_int, C.c_void_p, C.c_int64,
                                                                     C.c_void_p, C.c_void_p]
    lib.slot.argtypes = [C.c_int64, C.c_int, C.c_int64, C.c_void_p, C.c_void_p]
    lib.page.argtypes = [C.c_int, C.c_int64]
    return lib


def plan(host, lens, first, rep, n_kv=4, tp=16, window=0, width=4096, shift=5, minp=1, maxp=0x7FFFFFFF, target=1024,
         min_chunk=256, n_row=None):
    n = len(lens)
    n_row = (first[-1] if first else n) if n_row is None else n_row
    cl = (C.c_int32 * n)(*lens)
    cf = (C.c_int32 * (n + 1))(*first) if first else None
    cap = 400000
    out, bounds, bad = (Row * cap)(), (C.c_int64 * 3)(), C.c_int()
    m = host.plan(cl, cf, n, n_row, width, shift, rep, window, n_kv, tp, minp, maxp, target, min_chunk, out, cap,
                  bounds, C.byref(bad))
    assert m <= cap
    return [out[i] for i in range(m)], list(bounds), bad.value


def test_items_cover_every_tile_and_key_once(host):
    rng = random.Random(3)
    for trial in range(300):
        n = rng.choice([1, 2, 5, 64, 65, 130])
        top = rng.choice([40, 700, 9000, 131072])
        lens = [rng.choice([0, 1, rng.randint(0, top), top]) for _ in range(n)]
        decode = rng.random() < 0.5
        rows = [1] * n if decode else [rng.choice([0, 1, rng.randint(0, 300)]) for _ in range(n)]
        first = None if decode else [sum(rows[:i]) for i in range(n + 1)]
        rep, n_kv, tp = rng.choice([1, 3, 7, 8, 16, 20, 71]), rng.choice([1, 4, 8, 40]), rng.choice([16, 64, 128])
        window = rng.choice([0, 0, 1, 33, 4096])
        minp, maxp = rng.choice([(1, 0x7FFFFFFF), (1, 64), (65, 0x7FFFFFFF)])
        target, least = rng.choice([256, 512, 1024]), rng.choice([64, 128, 256])
        items, bounds, bad = plan(host, lens, first, rep, n_kv, tp, window, 8192, 4, minp, maxp, target, least)
        assert bad == 0
        assert len(items) <= bounds[0]                    # the grid holds them
        assert bounds[2] <= bounds[1]                     # and the workspace their parts
        slots = [i.slot for i in items if i.chunks > 1]
        assert len(set(slots)) == len(slots) and all(0 <= s < bounds[1] for s in slots)
        seen = {}
        for i in items:
            seen.setdefault((i.seq, i.tile), []).append(i)
        for s in range(n):
            pairs = rows[s] * rep
            served = minp <= pairs <= maxp
            tiles = [t for q, t in seen if q == s]
            assert sorted(tiles) == list(range(-(-pairs // tp) if served else 0))
        for (s, t), parts in seen.items():
            lo = parts[0].lo
            first_pos = lens[s] - rows[s] + t * tp // rep
            last_pos = lens[s] - rows[s] + (min((t + 1) * tp, rows[s] * rep) - 1) // rep
            assert lo % 32 == 0 and lo <= max(0, first_pos - window + 1 if window else 0)
            assert parts[0].klen % 64 == 0 and (parts[0].klen >= least // 2 or len(parts) == 1)
            assert [p.chunk for p in parts] == list(range(parts[0].chunks))
            assert lo + parts[0].chunks * parts[0].klen >= last_pos + 1
            assert (parts[0].chunks - 1) * parts[0].klen < max(1, parts[0].ext)


def test_bad_lengths_and_offsets_are_told(host):
    for lens, first, n_row, want in (([5, -1], None, 2, 1), ([5, 4096 * 32 + 1], None, 2, 1),
                                     ([5, 4096 * 32], None, 2, 0), ([9, 9], [0, 5, 3], 5, 1),
                                     ([9, 9], [-1, 2, 3], 5, 1), ([9, 9], [0, 2, 6], 5, 1),
                                     ([9, 9, 9], [0, 7, 2, 9], 5, 3), ([2 ** 31 - 1], None, 1, 1)):
        items, bounds, bad = plan(host, lens, first, 4, n_row=n_row)
        assert bad == want
        for i in items:  # whatever is left of them stays inside q and the table
            assert 0 <= i.row0 and i.row0 + i.rows <= n_row and 0 <= i.len <= 4096 * 32


def test_slots_and_pages(host):
    page, off = C.c_int64(), C.c_int()
    for s, ok in ((0, 1), (16 * 7 - 1, 1), (16 * 7, 0), (-1, 0), (-2 ** 63, 0), (2 ** 63 - 1, 0)):
        assert bool(host.slot(s, 4, 7, C.byref(page), C.byref(off))) == bool(ok)
        if ok:
            assert (page.value, off.value) == divmod(s, 16)
    # a slot past 2^31 in a large pool
    assert host.slot(2 ** 33 + 5, 4, 2 ** 30, C.byref(page), C.byref(off)) and page.value == 2 ** 29 and off.value == 5
    assert [host.page(i, 7) for i in (0, 6, 7, -1, 2 ** 31 - 1, -2 ** 31)] == [0, 6, -1, -1, -1, -1]


@pytest.mark.parametrize("n_seq", [2 ** 31 - 1, 2 ** 31 - 63])
def test_sequences_beyond_their_count_in_64s_are_refused(n_seq):
    """Sequences are counted in 64s in 32 bits: up to 2^31 - 64 of them."""
    assert attn(n_seq=n_seq, first=A) == fa.FRQ_ERR_ARG and "too many" in message(), message()
    assert attn(n_seq=2 ** 31 - 64, first=A) == fa.FRQ_ERR_ARG and "null context" in message(), message()
