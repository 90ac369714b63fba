"""Paged attention whose rows see more than what lies before them: a window
with sinks (frq_kv_attn_sink_dev) and trees of drafted tokens
(frq_kv_attn_tree_dev).  Held to the definition in 64 bits on the stored values,
each row over the keys of its own; the tolerance is test_gpu_kv.py's, derived
there, with the number of keys a row sees."""
import ctypes as C
import gc

import numpy as np
import pytest

import fieldrun_amd as fa
from fieldrun_amd import hip
from test_gpu_kv import Batch, Graph, put, same
from test_gpu_kv_edges import hold

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "rowi8"]


@pytest.fixture(autouse=True)
def freed():
    """A batch refers to itself: its device memory is given back here."""
    yield
    gc.collect()


def words_of(trees, pitch, junk=None):
    """Masks (lists of sets of drafted tokens, a sequence each) as words; bits
    past a sequence's rows as `junk` has them."""
    rows = [(len(t), m) for t in trees for m in t]
    out = np.zeros((len(rows), pitch), np.uint64)
    if junk is not None:
        out[:] = junk.integers(0, 1 << 63, out.shape, dtype=np.uint64) * np.uint64(2) + np.uint64(1)
    for i, (r, m) in enumerate(rows):
        for t in range(r):
            bit = np.uint64(1 << t % 64)
            out[i, t // 64] = out[i, t // 64] | bit if t in m else out[i, t // 64] & ~bit
    return out


def grow(rng, r, fan=3):
    """A tree of r drafted tokens: each sees its ancestors and itself."""
    masks = []
    for i in range(r):
        parent = rng.integers(max(0, i - 2 * fan) - 1, i) if i else -1
        masks.append((masks[parent] if parent >= 0 else set()) | {i})
    return masks


class More(Batch):
    """A Batch whose rows see sinks, or the tokens of their trees."""

    def __init__(self, *args, window=0, sinks=0, trees=None, pitch=None, junk=None, **how):
        super().__init__(*args, **how)
        self.window, self.sinks, self.trees, self.dtree = window, sinks, trees, None
        if trees is not None:
            self.decode = False
            self.pitch = pitch or max(1, -(-max(len(t) for t in trees) // 64))
            self.dtree = hip.DeviceArray.from_numpy(words_of(trees, self.pitch, junk))

    def seen(self, s, i):
        """The keys of row i of sequence s."""
        n, r = self.lens[s], self.rows[s]
        j = np.arange(n)
        if self.trees is None:
            p = n - r + i
            keep = j <= p
        else:
            p = n - r - 1 + len(self.trees[s][i])
            keep = j < n - r
        if self.window:
            keep &= (p - j < self.window) | (j < self.sinks)
        if self.trees is not None:
            keep[[n - r + t for t in self.trees[s][i]]] = True
        return np.flatnonzero(keep)

    def run(self, cap=0.0, spare=3, sync=True, fill=7.0):
        kv, hd, heads = self.p.kv, self.p.hd, self.p.kv * self.rep
        self.dq = hip.DeviceArray.from_numpy(self.q)
        self.do = hip.DeviceArray.from_numpy(np.full((self.n_row + spare, heads, hd), fill, np.float32))
        need = self.p.c.attn_ws_bytes(self.n_row, heads, len(self.lens), self.width)
        self.ws = hip.DeviceArray.from_numpy(np.full(need, 0xFF, np.uint8))
        t, n, f = self.dev
        self.call = lambda: self.p.c.attn_dev(
            self.dq.ptr, self.n_row, heads, t.ptr, self.width, n.ptr, len(self.lens), self.do.ptr,
            None if self.decode else f.ptr, cap=cap, window=self.window, sinks=self.sinks, ws_ptr=self.ws.ptr,
            ws_bytes=need, tree_ptr=self.dtree and self.dtree.ptr, tree_pitch=self.pitch if self.dtree else 1)
        self.call()
        if sync:
            self.ctx.sync()
        out = self.do.numpy()
        assert (out[self.n_row:] == fill).all()
        return out[:self.n_row]

    def want(self, cap=0.0, gone=None):
        kv, hd, rep, kind = self.p.kv, self.p.hd, self.rep, self.p.kind
        scale, u = hd ** -0.5, 2.0 ** -24
        out = np.zeros((self.n_row, kv * rep, hd))
        tol = np.zeros_like(out)
        for s in range(len(self.lens)):
            for i in range(self.rows[s]):
                keys = np.setdiff1d(self.seen(s, i), list((gone or {}).get(s, ())))
                if not len(keys):
                    continue
                r = int(self.first[s]) + i
                for h in range(kv):
                    k, v = (x[s][keys, h].astype(np.float64) for x in (self.k, self.v))
                    q = self.q[r, h * rep:(h + 1) * rep].astype(np.float64)
                    z = scale * (q @ k.T)
                    d = u * (4 * hd ** 0.5 + 8) * scale * (np.abs(q) @ np.abs(k).T).max(1)
                    if kind != "f32":
                        d += 2.0 ** -22 * scale * np.abs(q).max(1) * np.abs(k).sum(1).max()
                    if cap:
                        z = cap * np.tanh(z / cap)
                        d += 4e-7 * np.abs(z).max(1)
                    w = np.exp(z - z.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    at = slice(h * rep, (h + 1) * rep)
                    out[r, at] = w @ v
                    tol[r, at] = (np.expm1(2 * d) + 2.0 ** -21 + u * (len(keys) / 16 + 16))[:, None] * (w @ np.abs(v))
                    tol[r, at] += (2.0 ** (-126 if kind == "f32" else -35) * w.max(1) * len(keys))[:, None] * np.abs(
                        v[np.isfinite(v)]).max()
        return out, tol

    def check(self, cap=0.0):
        got = self.run(cap)
        hold(got, *self.want(cap))
        return got


# ---- windows with sinks -----------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 1), (5, 4), (16, 31), (33, 32), (40, 33), (100, 64), (64, 70), (7, 130),
                                          (1, 300), (2000, 5), (20, 100000)])
def test_sinks(ctx, kind, window, sinks):
    """Decode rows and prompt rows: windows that begin inside, at and behind the
    sinks' tiles, sinks past a sequence's end."""
    how = dict(window=window, sinks=sinks)
    More(ctx, kind, 16, 2, 3, 64, [1, 40, 300, 0, 97, 129, 33], seed=window, **how).check(cap=30.0)
    More(ctx, kind, 32, 1, 5, 128, [90, 257, 400], [60, 19, 200], seed=sinks, **how).check()
    More(ctx, kind, 64, 1, 2, 96, [3, 700, 130], [5, 1, 70], seed=sinks + 1, **how).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", range(16, 257, 16))
def test_sinks_at_every_width(ctx, kind, hd):
    More(ctx, kind, 16, 1, 3, hd, [200, 333], [1, 50], seed=hd, window=40, sinks=5).check()


@pytest.mark.parametrize("kind", KINDS)
def test_sinks_long_and_many(ctx, kind):
    """Windows cut over many workgroups, and more than 64 sequences."""
    More(ctx, kind, 64, 2, 4, 64, [30011], seed=1, window=9000, sinks=100).check()
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.choice([0, 1, 7, 40, 290], 150)]
    lens[71], lens[149] = 4001, 1200
    More(ctx, kind, 16, 1, 2, 32, lens, seed=2, window=64, sinks=9).check()
    rows = [min(n, int(x)) for n, x in zip(lens, rng.choice([0, 1, 2, 80], 150))]
    More(ctx, kind, 16, 1, 2, 32, lens, rows, seed=3, window=50, sinks=20).check()


@pytest.mark.parametrize("rows", [None, [3, 70, 1]])
def test_without_sinks_or_window_it_is_the_plain_call(ctx, rows):
    for how in (dict(window=40, sinks=0), dict(window=0, sinks=9), dict(window=0, sinks=2 ** 40), dict(window=7, sinks=2 ** 63)):
        b = More(ctx, "f16", 16, 2, 3, 64, [200, 300, 70], rows, seed=4, **how)
        got = b.run()
        b.window, b.sinks = (how["window"] if how["sinks"] < 2 ** 40 else 0), 0
        t, n, f = b.dev
        plain = hip.DeviceArray(b.q.shape, np.float32)
        call = fa.lib.frq_kv_attn_dev
        assert call(ctx.h, b.p.c._ref, b.dq.ptr, 384, b.n_row, 6, t.ptr, b.width, n.ptr, None if rows is None else f.ptr, 3,
                    64 ** -0.5, 0.0, b.window, plain.ptr, 384, b.ws.ptr, b.ws.nbytes) == 0
        ctx.sync()
        assert same(plain.numpy(), got)
        # through the entry point itself
        assert fa.lib.frq_kv_attn_sink_dev(ctx.h, b.p.c._ref, b.dq.ptr, 384, b.n_row, 6, t.ptr, b.width, n.ptr,
                                           None if rows is None else f.ptr, 3, 64 ** -0.5, 0.0, how["window"], how["sinks"],
                                           plain.ptr, 384, b.ws.ptr, b.ws.nbytes) == 0
        ctx.sync()
        assert same(plain.numpy(), got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 5), (33, 40), (20, 64)])
def test_pages_between_sinks_and_window_may_be_gone(ctx, kind, window, sinks):
    """A program frees what no later row sees; a page of a sink that is gone is
    reported, and its tokens are left out."""
    lens = [300 + i for i in range(32)] + [5, 1001, 16, 80]
    for rows in (None, [(1, 2, 50)[i % 3] for i in range(len(lens) - 4)] + [1, 60, 16, 3]):
        b = More(ctx, kind, 16, 1, 3, 64, lens, rows, seed=window, window=window, sinks=sinks)
        table = b.table.copy()
        for s, n in enumerate(lens):
            table[s, -(-sinks // 16):max(0, n - b.rows[s] - window + 1) // 16] = -1
        assert (table[:, -(-sinks // 16)] == -1).sum() >= len(lens) - 5
        put(b.dev[0], table)
        hold(b.run(), *b.want())
        table[3, 0] = b.p.n_pages
        put(b.dev[0], table)
        with pytest.raises(fa.FrqError) as e:
            b.run()
        assert e.value.code == fa.FRQ_ERR_ARG
        ctx.sync()
        hold(b.do.numpy()[:b.n_row], *b.want(gone={3: range(16)}))


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows", [None, [60, 90]])
def test_what_lies_between_sinks_and_window_may_be_anything(ctx, kind, rows):
    """Keys and values that no row sees, and some that only earlier rows see,
    infinite or NaN; a sink that is infinite reaches every row."""
    lens, w, sinks = [200, 333], 40, 5

    def poison(ks, vs):
        for k, v in zip(ks, vs):
            first = len(k) - (1 if rows is None else rows[0 if len(k) == 200 else 1]) - w + 1
            k[sinks:first], v[sinks:first:2], v[sinks + 1:first:2] = np.nan, np.inf, np.nan

    b = More(ctx, kind, 16, 2, 3, 64, lens, rows, seed=6, window=w, sinks=sinks, poison=poison)
    b.check()
    if rows is None:
        return

    def early(ks, vs):  # seen by each sequence's first rows alone
        for k, v in zip(ks, vs):
            v[len(k) - (60 if len(k) == 200 else 90) - w + 10] = np.inf

    b = More(ctx, kind, 16, 2, 3, 64, lens, rows, seed=6, window=w, sinks=sinks, poison=early)
    got = b.run()
    hit = np.zeros(b.n_row, bool)
    for s in (0, 1):
        for i in range(b.rows[s]):
            hit[b.first[s] + i] = lens[s] - rows[s] - w + 10 in b.seen(s, i)
    assert 0 < hit.sum() < b.n_row and np.isfinite(got[~hit]).all() and not np.isfinite(got[hit]).any()
    b = More(ctx, kind, 16, 2, 3, 64, lens, rows, seed=6, window=w, sinks=sinks,
             poison=lambda ks, vs: vs[0].__setitem__(2, np.inf))
    got = b.run()
    assert not np.isfinite(got[:60]).any() and np.isfinite(got[60:]).all()


# ---- trees --------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv,rep,hd,lens,rows", [
    (2, 7, 64, [211], [8]), (1, 1, 16, [1], [1]), (2, 4, 128, [300, 26, 64, 90], [26, 26, 1, 40]),
    (1, 2, 96, [700], [64]), (1, 3, 80, [130, 500], [130, 65]), (2, 1, 256, [70, 90], [63, 64]),
    (1, 8, 112, [257, 40, 33], [129, 3, 0]), (1, 16, 48, [90], [33]),
])
def test_trees(ctx, kind, kv, rep, hd, lens, rows):
    """Trees over much, little and nothing cached, in one, two and three words;
    what the masks hold past a tree's rows is anything."""
    rng = np.random.default_rng(hd + len(lens))
    trees = [grow(rng, r) for r in rows]
    More(ctx, kind, 16, kv, rep, hd, lens, rows, seed=hd, trees=trees, pitch=3, junk=rng).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rep", [1, 5])
def test_any_mask(ctx, kind, rep):
    """Any set of drafted tokens: none (a row without anything to see is
    zeros), all, later ones, not itself."""
    rng = np.random.default_rng(rep)
    lens, rows = [300, 40, 70, 70], [70, 40, 40, 5]
    trees = [[set(np.flatnonzero(rng.random(r) < p)) for _ in range(r)] for r, p in zip(rows, (0.3, 0.05, 0.9, 0.0))]
    trees[1][3] = set()
    b = More(ctx, kind, 16, 2, rep, 64, lens, rows, seed=rep, trees=trees)
    got = b.check(cap=20.0)
    assert (got[70 + 3] == 0).all() and any(not t for t in trees[1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", range(16, 257, 16))
def test_trees_at_every_width(ctx, kind, hd):
    rng = np.random.default_rng(hd)
    rows = [5, 50]
    More(ctx, kind, 16, 1, 3, hd, [200, 133], rows, seed=hd, trees=[grow(rng, r) for r in rows]).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 2), (10, 0), (33, 40), (64, 5), (300, 70)])
def test_trees_with_windows_and_sinks(ctx, kind, window, sinks):
    """A row's window ends at its depth: of two siblings' branches of unlike
    depth each sees its own of the cached tokens; pages that none sees are
    gone."""
    rng = np.random.default_rng(window)
    lens, rows = [400, 131, 45, 200], [60, 9, 45, 64]
    trees = [grow(rng, r) for r in rows]
    for i in range(20, 60):  # one deep branch
        trees[0][i] = trees[0][i - 1] | {i}
    b = More(ctx, kind, 16, 2, 3, 64, lens, rows, seed=window, trees=trees, window=window, sinks=sinks)
    b.check()
    table = b.table.copy()
    for s, n in enumerate(lens):
        low = min((k for i in range(rows[s]) for k in list(b.seen(s, i)) + [n - rows[s]] if k >= sinks), default=0)
        table[s, -(-sinks // 16):low // 16] = -1
    put(b.dev[0], table)
    hold(b.run(), *b.want())


def test_a_chain_is_a_prompt(ctx):
    """Rows that see every token before them: what frq_kv_attn_dev computes."""
    for kind in KINDS:
        lens, rows = [200, 90], [70, 4]
        chain = [[set(range(i + 1)) for i in range(r)] for r in rows]
        b = More(ctx, kind, 16, 2, 3, 64, lens, rows, seed=3, trees=chain)
        got = b.check()
        b.trees, b.dtree = None, None
        hold(b.run(), got.astype(np.float64), 2 * b.want()[1])


@pytest.mark.parametrize("kind", KINDS)
def test_trees_long_and_many(ctx, kind):
    rng = np.random.default_rng(9)
    More(ctx, kind, 64, 2, 4, 64, [20011], [64], seed=1, trees=[grow(rng, 64)]).check()
    More(ctx, kind, 64, 1, 4, 128, [9000], [12], seed=1, trees=[grow(rng, 12)]).check()
    rows = [int(x) for x in rng.choice([0, 1, 8, 70], 150)]
    lens = [r + int(x) for r, x in zip(rows, rng.choice([0, 1, 60, 200], 150))]
    More(ctx, kind, 16, 1, 2, 32, lens, rows, seed=2, trees=[grow(rng, r) for r in rows]).check()


def test_a_row_a_sequence(ctx):
    """Without row offsets every sequence drafts one token."""
    b = More(ctx, "f16", 16, 2, 3, 64, [40, 1, 300], [1, 1, 1], seed=5, trees=[[{0}], [set()], [set()]])
    got = b.check()
    assert (got[1] == 0).all()
    b.decode = True
    assert same(b.run(), got)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows", [[9], [70]])
def test_branches_keep_to_themselves(ctx, kind, rows):
    """A drafted token that is infinite or NaN reaches the rows that see it, and
    none that do not."""
    rng = np.random.default_rng(rows[0])
    trees = [grow(rng, rows[0])]
    bad = 4

    def poison(ks, vs):
        at = 300 - rows[0] + bad
        vs[0][at, :, ::2], vs[0][at, :, 1::2] = np.inf, np.nan

    clean = More(ctx, kind, 16, 2, 3, 64, [300], rows, seed=7, trees=trees).run()
    got = More(ctx, kind, 16, 2, 3, 64, [300], rows, seed=7, trees=trees, poison=poison).run()
    hit = np.array([bad in m for m in trees[0]])
    assert 0 < hit.sum() < rows[0] and not np.isfinite(got[hit]).any() and same(got[~hit], clean[~hit])

    def key(ks, vs):
        ks[0][300 - rows[0] + bad] = np.nan

    got = More(ctx, kind, 16, 2, 3, 64, [300], rows, seed=7, trees=trees, poison=key).run()
    assert not np.isfinite(got[hit]).any() and same(got[~hit], clean[~hit])


@pytest.mark.parametrize("many", [False, True])
def test_trees_out_of_range_stay_as_they_were(ctx, many):
    """More rows than tokens, or than a mask has bits."""
    rng = np.random.default_rng(2)
    lens, rows = [200, 90, 70, 300] + [9] * (80 if many else 0), [8, 70, 30, 66] + [2] * (80 if many else 0)
    trees = [grow(rng, r) for r in rows]
    b = More(ctx, "f16", 16, 2, 3, 64, lens, rows, seed=3, trees=trees)
    want, tol = b.want()
    put(b.dev[1], np.array([200, 90, 29, 300] + lens[4:], np.int32))
    with pytest.raises(fa.FrqError) as e:
        b.run()
    assert e.value.code == fa.FRQ_ERR_ARG
    ctx.sync()
    got = b.do.numpy()[:b.n_row]
    out = np.arange(b.n_row)
    out = (out >= b.first[2]) & (out < b.first[3])
    assert (got[out] == 7.0).all()
    hold(got[~out], want[~out], tol[~out])
    put(b.dev[1], np.asarray(lens, np.int32))
    b.dtree, b.pitch = hip.DeviceArray.from_numpy(words_of([t if len(t) <= 64 else [set(m) for m in t] for t in trees], 2)[:, :1]), 1
    with pytest.raises(fa.FrqError) as e:
        b.run()
    assert e.value.code == fa.FRQ_ERR_ARG
    ctx.sync()
    got = b.do.numpy()[:b.n_row]
    row = np.arange(b.n_row)
    out = ((row >= b.first[1]) & (row < b.first[2])) | ((row >= b.first[3]) & (row < b.first[4]))
    assert (got[out] == 7.0).all()
    hold(got[~out], want[~out], tol[~out])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [[5, 20], [70, 90]])
def test_pages_of_trees_out_of_range_take_no_part(ctx, kind, rows):
    rng = np.random.default_rng(8)
    lens = [300, 200]
    b = More(ctx, kind, 16, 2, 3, 64, lens, rows, seed=4, trees=[grow(rng, r) for r in rows])
    table = b.table.copy()
    table[0, 3] = -1
    table[1, [0, (200 - rows[1]) // 16 + 1]] = b.p.n_pages
    gone = {0: range(48, 64), 1: [*range(16), *range(16 * ((200 - rows[1]) // 16 + 1), 16 * ((200 - rows[1]) // 16 + 2))]}
    put(b.dev[0], table)
    runs = []
    for _ in range(2):
        with pytest.raises(fa.FrqError) as e:
            b.run(cap=20.0)
        assert e.value.code == fa.FRQ_ERR_ARG
        ctx.sync()
        runs.append(b.do.numpy()[:b.n_row])
    assert same(*runs)
    hold(runs[0], *b.want(20.0, gone))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("every", [False, True])
@pytest.mark.parametrize("window,sinks,length,rows,page", [
    (1, 0, 300, 70, 15), (10, 0, 300, 70, 15), (10, 5, 300, 70, 14), (16, 40, 131, 64, 5),  # the decode kernel
    (10, 1000, 1500, 200, 85), (190, 0, 900, 400, 32), (190, 0, 900, 400, 31),  # the prompt kernel
])
def test_pages_of_drafted_tokens_count_past_the_window(ctx, kind, every, window, sinks, length, rows, page):
    """A drafted token stays seen however deep its row, so a page id out of range
    under one is reported and its tokens left out of every row: chains longer
    than the window, and rows that see all drafted tokens."""
    trees = [[set(range(r if every else i + 1)) for i in range(r)] for r in (rows, 7)]
    rep = 3 if rows < 100 else 21 if sinks else 42
    b = More(ctx, kind, 16, 2, rep, 16, [length, 40], [rows, 7], seed=window, trees=trees, window=window, sinks=sinks)
    table = b.table.copy()
    assert (page + 1) * 16 > length - rows and page * 16 + 15 < length
    table[0, page] = b.p.n_pages
    put(b.dev[0], table)
    runs = []
    for _ in range(2):
        with pytest.raises(fa.FrqError) as e:
            b.run()
        assert e.value.code == fa.FRQ_ERR_ARG
        ctx.sync()
        runs.append(b.do.numpy()[:b.n_row])
    assert same(*runs)
    hold(runs[0], *b.want(gone={0: range(16 * page, 16 * page + 16)}))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("many", [False, True])
def test_small_sequences_beside_large_ones(ctx, kind, many):
    """Calls of many pairs a sequence, where one kernel serves them all: rows of
    sequences of a token or none, of one row or none, beside large ones; then a
    length that no table holds."""
    lens, rows = [900, 1, 40, 0, 333, 17], [200, 1, 1, 2, 90, 17]
    if many:
        lens, rows = lens + [25, 0, 3, 60] * 20, rows + [25, 1, 0, 57] * 20
    b = More(ctx, kind, 16, 2, 7, 64, lens, rows, seed=5, window=64, sinks=5)
    b.check(cap=20.0)
    want, tol = b.want()
    put(b.dev[1], np.array([900, 1, 2 ** 30, 0, 333, 17] + lens[6:], np.int32))
    with pytest.raises(fa.FrqError) as e:
        b.run()
    assert e.value.code == fa.FRQ_ERR_ARG
    ctx.sync()
    got, other = b.do.numpy()[:b.n_row], np.arange(b.n_row) != b.first[2]
    assert (got[~other] == 0.0).all()
    hold(got[other], want[other], tol[other])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4)])
def test_small_trees_beside_large_ones(ctx, kind, window, sinks):
    rng = np.random.default_rng(9)
    lens, rows = [9000, 1, 40, 0, 700, 17], [130, 1, 1, 0, 30, 17]
    trees = [grow(rng, r) for r in rows]
    More(ctx, kind, 64, 4, 7, 32, lens, rows, seed=6, trees=trees, window=window, sinks=sinks).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("trees", [False, True])
def test_batches_with_idle_sequences(ctx, kind, trees):
    """No more rows than sequences, most of them idle, sequences of a row beside
    large ones: which do or do not fill a launch that cuts no keys, also behind
    one another in a graph; and a length that no table holds."""
    rng = np.random.default_rng(12)
    for kv, rep, n, lens, rows in ((2, 7, 64, [4000, 300, 40], [16, 1, 5]), (8, 16, 200, [900, 300, 150, 7], [140, 1, 20, 2]),
                                   (8, 16, 130, [1700, 0, 95], [95, 1, 30]), (1, 140, 70, [2000, 33], [9, 1]),
                                   (8, 16, 90, [400, 50] * 5, [16, 2] * 5)):
        rows, lens = rows + [0] * (n - len(rows)), lens + [0] * (n - len(lens))
        if trees:
            rows = [min(a, b) for a, b in zip(rows, lens)]
        assert sum(rows) <= n
        More(ctx, kind, 16, kv, rep, 32, lens, rows, seed=n, window=600, sinks=9,
             trees=[grow(rng, r) for r in rows] if trees else None).check()
    n, lens, rows = 200, [700, 300, 150, 400, 40] + [0] * 195, [120, 1, 20, 30, 2] + [0] * 195
    b = More(ctx, kind, 16, 8, 16, 32, lens, rows, seed=n, window=600, sinks=9, trees=[grow(rng, r) for r in rows] if trees else None)
    b.check()
    graph, held = Graph(ctx, b.call), (list(b.k), list(b.v))
    for first in (130, 700, 2 ** 30):  # the longest and its share of the keys
        put(b.dev[1], np.array([first] + lens[1:], np.int32))
        b.lens = [first if first < 2 ** 30 else 0] + lens[1:]
        b.k, b.v = ([x[:n] for x, n in zip(y, b.lens)] for y in held)
        outs = []
        for how in (graph.replay, b.call):
            put(b.do, np.full(b.do.shape, 7.0, np.float32))
            how()
            if first < 2 ** 30:
                ctx.sync()
            else:
                with pytest.raises(fa.FrqError):
                    ctx.sync()
            outs.append(b.do.numpy()[:b.n_row])
        assert same(*outs)
        if first < 2 ** 30:
            hold(outs[0], *b.want())
        else:
            assert (outs[0][:120] == (7.0 if trees else 0.0)).all()
            b.lens[0], b.rows = 120, [120] + rows[1:]
            b.k, b.v = ([x[:n] for x, n in zip(y, b.lens)] for y in held)
            want, tol = b.want()
            hold(outs[0][120:], want[120:], tol[120:])
    graph.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [16, 128, 1024])
def test_pages_and_pitches(ctx, kind, page):
    """Strided pages of every size, rows of q and out that lie apart."""
    rng = np.random.default_rng(10)
    for lens, rows in (([1500, 90, 3], [1, 1, 1]), ([1500, 90, 40], [70, 5, 40])):
        for trees in (None, [grow(rng, r) for r in rows]):
            b = More(ctx, kind, page, 2, 3, 64, lens, rows, seed=page, pad=1, window=200, sinks=17, trees=trees)
            want = b.check()
            n, heads, wide = b.n_row, 6, 6 * 64
            q = np.full((n, wide + 5), np.nan, np.float32)
            q[:, :wide] = b.q.reshape(n, wide)
            dq, do = hip.DeviceArray.from_numpy(q), hip.DeviceArray.from_numpy(np.full((n, wide + 3), 7.0, np.float32))
            t, ln, f = b.dev
            b.p.c.attn_dev(dq.ptr, n, heads, t.ptr, b.width, ln.ptr, len(lens), do.ptr, f.ptr, window=200, sinks=17,
                           q_pitch=wide + 5, out_pitch=wide + 3, ws_ptr=b.ws.ptr, ws_bytes=b.ws.nbytes,
                           tree_ptr=b.dtree and b.dtree.ptr, tree_pitch=b.pitch if b.dtree else 1)
            ctx.sync()
            out = do.numpy()
            assert same(out[:, :wide].copy().reshape(want.shape), want) and (out[:, wide:] == 7.0).all()


@pytest.mark.parametrize("rep", [70, 130])
def test_many_heads_and_a_row_a_sequence(ctx, rep):
    More(ctx, "f16", 16, 1, rep, 32, [700, 33], [1, 1], seed=rep, window=90, sinks=4).check()
    More(ctx, "f16", 16, 1, rep, 32, [700, 33], [1, 1], seed=rep, trees=[[{0}], [{0}]]).check()


def test_captured_and_replayed(ctx):
    """A speculative step's attention in a graph, over changing trees, lengths
    and queries, with eager calls and synchronizations between."""
    rng = np.random.default_rng(3)
    lens, rows = [300, 700], [9, 60]
    b = More(ctx, "rowi8", 16, 2, 3, 64, lens, rows, seed=4, trees=[grow(rng, r) for r in rows], window=200, sinks=4)
    b.check()
    graph = Graph(ctx, b.call)
    held, last = (list(b.k), list(b.v)), None
    for i in range(4):
        b.lens = [300 - 40 * i, 700 - 100 * i]
        b.k, b.v = ([x[:n] for x, n in zip(y, b.lens)] for y in held)
        b.trees = [grow(rng, r) for r in rows]
        b.q = rng.standard_normal(b.q.shape).astype(np.float32)
        put(b.dev[1], np.array(b.lens, np.int32))
        put(b.dtree, words_of(b.trees, b.pitch))
        put(b.dq, b.q)
        outs = []
        for how in (graph.replay, b.call, graph.replay):
            put(b.do, np.full(b.do.shape, 7.0, np.float32))
            how()
            ctx.sync()
            outs.append(b.do.numpy())
        assert all(same(o, outs[0]) for o in outs[1:])
        hold(outs[0][:b.n_row], *b.want())
        assert last is None or not same(outs[0], last)
        last = outs[0]
    graph.close()


def test_calls_on_another_stream_and_without_a_workspace(ctx):
    rng = np.random.default_rng(4)
    b = More(ctx, "f16", 16, 2, 3, 64, [300, 70], [70, 1], seed=2, trees=[grow(rng, 70), [{0}]])
    want = b.check()
    other = C.c_void_p()
    hip._chk(hip._hip.hipStreamCreate(C.byref(other)), "hipStreamCreate")
    try:
        ctx.set_stream(other.value)
        assert same(b.run(), want)
    finally:
        ctx.sync()
        ctx.set_stream(None)
        hip._chk(hip._hip.hipStreamDestroy(other), "hipStreamDestroy")
    t, n, f = b.dev
    put(b.do, np.zeros(b.do.shape, np.float32))
    b.p.c.attn_dev(b.dq.ptr, b.n_row, 6, t.ptr, b.width, n.ptr, 2, b.do.ptr, f.ptr, tree_ptr=b.dtree.ptr, tree_pitch=b.pitch)
    ctx.sync()
    assert same(b.do.numpy()[:b.n_row], want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [[1, 2], [60, 90]])
def test_pages_beyond_32_bits(ctx, kind, rows):
    """Pages, and int8 steps, more than 2^32 bytes apart."""
    page, kv, hd, n_pages, rep = 256, 1, 64, 2, 3
    size = {"f32": 4, "f16": 2, "rowi8": 1}[kind]
    stride, sstride = (1 << 32) // size + 1024, (1 << 30) + 64
    k, v = (hip.DeviceArray(((stride + kv * page * hd) * size,), np.int8) for _ in "kv")
    ks = vs = None
    if kind == "rowi8":
        ks, vs = (hip.DeviceArray((sstride + kv * page,), np.float32) for _ in "kv")
    c = fa.KvCache(ctx, kind, n_pages, page, kv, hd, k.ptr, v.ptr, ks and ks.ptr, vs and vs.ptr, stride, sstride)
    rng = np.random.default_rng(5)
    for how in (dict(window=30, sinks=3), dict(trees=[grow(rng, r) for r in rows])):
        b = More(ctx, kind, page, kv, rep, hd, [200, 250], rows, seed=3, **how)  # the same data, beside it
        table = np.array([[1], [0]], np.int32)
        for s, n in enumerate(b.lens):
            dk, dv = (hip.DeviceArray.from_numpy(x[s].astype(np.float32)) for x in (b.k, b.v))
            slot = hip.DeviceArray.from_numpy(table[s, 0] * page + np.arange(n, dtype=np.int64))
            c.write_dev(dk.ptr, dv.ptr, slot.ptr, n)
            ctx.sync()
            b.k[s], b.v[s] = b.p.stored(b.k[s].astype(np.float32)), b.p.stored(b.v[s].astype(np.float32))
        q, first, lens = (hip.DeviceArray.from_numpy(x) for x in (b.q, b.first, np.asarray(b.lens, np.int32)))
        t, out = hip.DeviceArray.from_numpy(table), hip.DeviceArray(b.q.shape, np.float32)
        c.attn_dev(q.ptr, b.n_row, kv * rep, t.ptr, 1, lens.ptr, 2, out.ptr, first_ptr=first.ptr, window=b.window,
                   sinks=b.sinks, tree_ptr=b.dtree and b.dtree.ptr, tree_pitch=b.pitch if b.dtree else 1)
        ctx.sync()
        hold(out.numpy(), *b.want())
