"""The paged attention where a call is allowed and unusual: pages that are gone
or out of range, scores, caps and values of any size, entries that are not
finite.  Held to the definition in 64 bits as test_gpu_kv.py holds the rest;
its tolerance is derived there."""
import ctypes as C
import gc

import numpy as np
import pytest

import fieldrun_amd as fa
from fieldrun_amd import hip
from test_gpu_kv import Batch, put

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "rowi8"]


@pytest.fixture(autouse=True)
def freed():
    """A batch refers to itself: its device memory is given back here."""
    yield
    gc.collect()


def expect(b, gone=None, scale=None, cap=0.0, window=0):
    """Outputs and tolerances of batch b, the keys of gone ({sequence: keys})
    left out; a row that sees no key is zeros."""
    kv, hd, rep, kind = b.p.kv, b.p.hd, b.rep, b.p.kind
    scale = hd ** -0.5 if scale is None else scale
    out = np.zeros((b.n_row, kv * rep, hd))
    tol = np.zeros_like(out)
    u = 2.0 ** -24
    for s, n in enumerate(b.lens):
        for i in range(b.rows[s]):
            p = n - b.rows[s] + i
            keys = np.arange(max(0, p - window + 1) if window else 0, p + 1)
            keys = np.setdiff1d(keys, list((gone or {}).get(s, ())))
            if not len(keys):
                continue
            r = int(b.first[s]) + i
            for h in range(kv):
                k, v = (x[s][keys, h].astype(np.float64) for x in (b.k, b.v))
                q = b.q[r, h * rep:(h + 1) * rep].astype(np.float64)
                z = scale * (q @ k.T)
                d = u * (4 * hd ** 0.5 + 8) * abs(scale) * (np.abs(q) @ np.abs(k).T).max(1)
                if kind != "f32":
                    d += 2.0 ** -22 * abs(scale) * np.abs(q).max(1) * np.abs(k).sum(1).max()
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


def hold(got, want, tol):
    off = np.abs(got - want)
    bad = ~(off <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


def set_table(b, table):
    put(b.dev[0], np.ascontiguousarray(table, np.int32))


# ---- pages ----------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 16, 33])
@pytest.mark.parametrize("many", [False, True])
def test_pages_before_the_window_may_be_gone(ctx, kind, window, many):
    """A program frees the pages that no later row sees and marks them -1: no
    error and the same outputs, whatever place in its page the window begins
    at (every length mod 32), decode rows and prompt rows."""
    lens = [300 + i for i in range(32)] * (3 if many else 1) + [5, 1001, 16]
    for rows in (None, [(1, 2, 50)[i % 3] for i in range(len(lens) - 3)] + [1, 60, 16]):
        b = Batch(ctx, kind, 16, 1, 3, 64, lens, rows, seed=window)
        table = b.table.copy()
        for s, n in enumerate(lens):
            table[s, :max(0, n - b.rows[s] - window + 1) // 16] = -1
        assert (table[:, 0] == -1).sum() >= len(lens) - 3
        set_table(b, table)
        hold(b.run(window=window), *expect(b, window=window))


def seed_with(lens, page, owner):
    """A seed whose Batch of lens gives page 0 to sequence `owner` (None: to none)."""
    held = [-(-n // page) for n in lens]
    for seed in range(1000):
        at = int(np.argwhere(np.random.default_rng(seed).permutation(sum(held) + 2) == 0)[0, 0])
        who = next((s for s in range(len(lens)) if sum(held[:s]) <= at < sum(held[:s + 1])), None)
        if who == owner:
            return seed
    raise AssertionError


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("owner", [None, 0])
@pytest.mark.parametrize("rows", [None, [3, 4, 2], [40, 90, 60]])
@pytest.mark.parametrize("window,cap", [(0, 0.0), (20, 30.0)])
def test_pages_out_of_range_take_no_part(ctx, kind, owner, rows, window, cap):
    """Keys under a page id out of range are left out and reported, whatever
    page 0 holds (unwritten: NaN and infinities; another sequence's rows, here
    large ones); a row that is left without a key gets zeros."""
    lens = [200, 300, 70]

    def poison(ks, vs):
        ks[0] *= 3
        vs[0] += 1000

    b = Batch(ctx, kind, 16, 2, 3, 64, lens, rows, seed=seed_with(lens, 16, owner), poison=poison)
    assert (b.table[0] == 0).any() == (owner == 0)
    clean = b.run(window=window, cap=cap)
    hold(clean, *expect(b, window=window, cap=cap))
    table = b.table.copy()
    holes = {1: (3, 10, 17, 18), 2: (0, 1, 2, 3, 4)}
    ids = [-1, b.p.n_pages, 2 ** 31 - 1, -2 ** 31]
    for s, pages in holes.items():
        for i, p in enumerate(pages):
            table[s, p] = ids[i % 4]
    gone = {s: {j for p in pages for j in range(16 * p, 16 * p + 16)} for s, pages in holes.items()}
    set_table(b, table)
    with pytest.raises(fa.FrqError) as e:
        b.run(window=window, cap=cap)
    assert e.value.code == fa.FRQ_ERR_ARG
    ctx.sync()
    got = b.do.numpy()[:b.n_row].reshape(clean.shape)
    want, tol = expect(b, gone, window=window, cap=cap)
    hold(got, want, tol)
    assert (got[b.first[2]:] == 0).all()  # every page of it is gone
    assert np.array_equal(got[:b.first[1]], clean[:b.first[1]])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kv,rep,many", [(16, 2, 5, False), (80, 3, 20, False), (256, 1, 3, False), (48, 2, 3, True)])
def test_gone_pages_at_any_width(ctx, kind, hd, kv, rep, many):
    """Strided pages, heads of every kind of width, decode and prompt rows in one
    call, on both sides of 64 sequences; the same bits again."""
    lens = [400, 150, 90] + [7] * (80 if many else 0)
    rows = [1, 60, 2] + [1] * (len(lens) - 3)
    b = Batch(ctx, kind, 16, kv, rep, hd, lens, rows, seed=hd, pad=1)
    table = b.table.copy()
    for s, pages in ((0, (2, 24)), (1, (0, 8)), (2, (5,))):
        table[s, list(pages)] = b.p.n_pages + s
    gone = {s: {j for p in np.flatnonzero(table[s, :-(-lens[s] // 16)] >= b.p.n_pages) for j in range(16 * p, 16 * p + 16)}
            for s in range(3)}
    set_table(b, table)
    runs = []
    for _ in range(2):
        with pytest.raises(fa.FrqError) as e:
            b.run(cap=20.0)
        assert e.value.code == fa.FRQ_ERR_ARG
        ctx.sync()
        runs.append(b.do.numpy()[:b.n_row].reshape(b.n_row, kv * rep, hd))
    hold(runs[0], *expect(b, gone, cap=20.0))
    assert np.array_equal(runs[0], runs[1])


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_gone_pages_beside_values_that_are_not_finite(ctx, kind):
    """A seen value that is not finite reaches the rows that see it and no
    other, in a tile with a page out of range too."""
    def poison(ks, vs):
        vs[0][70, 0, 5] = np.inf
        vs[0][58, 0, 9] = np.nan  # in the page that goes

    b = Batch(ctx, kind, 16, 1, 3, 64, [100], [64], poison=poison)
    table = b.table.copy()
    table[0, 3] = -1  # keys 48 .. 63
    set_table(b, table)
    with pytest.raises(fa.FrqError):
        b.run()
    got = b.do.numpy()[:64].reshape(64, 3, 64)
    with np.errstate(invalid="ignore"):
        want, tol = expect(b, {0: set(range(48, 64))})
    hold(got[:34], want[:34], tol[:34])  # rows at 36 .. 69
    rest = np.delete(np.arange(64), 5)
    hold(got[34:][:, :, rest], want[34:][:, :, rest], tol[34:][:, :, rest])
    assert (got[34:, :, 5] == np.inf).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [[3, 4, 2], [60, 70, 80]])
@pytest.mark.parametrize("many", [False, True])
def test_bad_lengths_and_offsets_stay_with_their_sequences(ctx, kind, rows, many):
    """A length out of range counts as 0, its rows are zeros; rows between
    offsets out of range stay as they were; the others are right."""
    lens = [300, 90, 200] + [5] * (100 if many else 0)
    rows = rows + [1] * (len(lens) - 3)
    b = Batch(ctx, kind, 16, 1, 3, 64, lens, rows, seed=11)
    clean = b.run()
    hold(clean, *expect(b))
    at = b.first
    want, tol = expect(b)
    for change, value in (("length", b.width * 16 + 1), ("length", -1), ("offset", b.n_row + 1), ("offset", -1)):
        n, f = np.asarray(lens, np.int32), b.first.copy()
        if change == "length":
            n[1] = value
        else:
            f[2] = value  # the end of sequence 1 and the beginning of 2
        put(b.dev[1], n)
        put(b.dev[2], f)
        with pytest.raises(fa.FrqError) as e:
            b.run()
        assert e.value.code == fa.FRQ_ERR_ARG
        ctx.sync()
        got = b.do.numpy()[:b.n_row].reshape(clean.shape)
        lost = slice(at[1], at[2] if change == "length" else at[3])
        assert (got[lost] == (0.0 if change == "length" else 7.0)).all()
        # (the others' keys are cut into other runs than before: not the same bits)
        hold(*(np.delete(x, np.r_[lost], 0) for x in (got, want, tol)))
        put(b.dev[1], np.asarray(lens, np.int32))
        put(b.dev[2], b.first)
    assert np.array_equal(b.run(), clean)


def test_a_bad_index_and_a_nan_are_both_reported(ctx):
    b = Batch(ctx, "f16", 16, 1, 2, 32, [20])
    b.run()
    table = b.table.copy()
    table[0, 1] = -1
    x = hip.DeviceArray.from_numpy(np.full((1, 64), np.nan, np.float32))
    a8, sa = hip.DeviceArray((1, fa.quant_pitch(64)), np.int8), hip.DeviceArray((1,), np.float32)
    oi, ov = hip.DeviceArray((1, 32), np.uint32), hip.DeviceArray((1, 32), np.float32)
    for first in (0, 1):
        set_table(b, table)
        for i in (first, 1 - first):
            if i:
                b.call()
            else:
                ctx.quant_dev(x.ptr, 1, 64, a8.ptr, sa.ptr, oi.ptr, ov.ptr)
        codes = []
        for _ in range(2):
            with pytest.raises(fa.FrqError) as e:
                ctx.sync()
            codes.append(e.value.code)
        assert sorted(codes) == sorted([fa.FRQ_ERR_NAN, fa.FRQ_ERR_ARG])
        ctx.sync()  # each told once


# ---- sizes ----------------------------------------------------------------------

def patterned(b, rows_of, value):
    """Keys of few kinds: key j of every sequence has value(j) in channel 0 and
    zeros beside it, so that scores are exact and tie exactly."""
    for s, n in enumerate(b.lens):
        if not n:
            continue
        k = np.zeros((n, b.p.kv, b.p.hd), np.float32)
        k[:, :, 0] = np.array([value(j) for j in range(n)], np.float32)[:, None]
        j = np.arange(n)
        b.p.write(k, b.v[s].astype(np.float32), b.table[s, j // b.p.page].astype(np.int64) * b.p.page + j % b.p.page)
        b.k[s] = b.p.stored(k)
        b.v[s] = b.p.stored(b.v[s].astype(np.float32))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [None, [60, 90]])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 24 * 1.5, 2.0 ** 27, 2.0 ** 31, 2.0 ** 40 * 1.25, 2.0 ** 70, 2.0 ** 110])
def test_scores_of_any_size(ctx, kind, rows, size):
    """Scores far beyond the steps of f32 at 1: the keys that share the largest
    share the output, evenly and exactly as many as there are, over one chunk
    and several; a second head asks the other way, a third with zeros."""
    b = Batch(ctx, kind, 16, 1, 3, 64, [90, 5000], rows, seed=4)
    patterned(b, rows, lambda j: (j * 5) % 7 - 3)
    b.q[:] = 0.0
    b.q[:, 0, 0] = size
    b.q[:, 1, 0] = -size
    got = b.run()
    u = 2.0 ** -24
    for s, n in enumerate(b.lens):
        for i in range(b.rows[s]):
            p = n - b.rows[s] + i
            k0, v = b.k[s][:p + 1, 0, 0], b.v[s][:p + 1, 0].astype(np.float64)
            for h, top in ((0, k0.max()), (1, k0.min()), (2, None)):
                keys = np.flatnonzero(k0 == top) if h < 2 else np.arange(p + 1)
                want = v[keys].mean(0)
                # no score is rounded: the weights' split, sums, joining and division, as in test_gpu_kv.py
                tol = (2.0 ** -21 + u * ((p + 1) / 16 + 16)) * np.abs(v[keys]).mean(0)
                tol += 2.0 ** -35 * (p + 1) / len(keys) * np.abs(v).max() * (kind != "f32")
                assert (np.abs(got[b.first[s] + i, h] - want) <= tol).all(), (s, i, h)


@pytest.mark.parametrize("kind", ["f16", "rowi8"])
@pytest.mark.parametrize("cap", [0.0, 50.0])
def test_large_scale_and_rows_of_q(ctx, kind, cap):
    """scale times the size of q beyond f32, over keys of zeros among others."""
    b = Batch(ctx, kind, 16, 1, 2, 64, [300, 70], [70, 1], seed=2)
    patterned(b, None, lambda j: j % 3)
    b.q[:] = 0.0
    b.q[:, 0, 0] = 3e38
    b.q[:, 1, 0] = -3e38
    got = b.run(scale=1e25, cap=cap)
    for s, n in enumerate(b.lens):
        for i in range(b.rows[s]):
            p = n - b.rows[s] + i
            v, k0 = b.v[s][:p + 1, 0].astype(np.float64), b.k[s][:p + 1, 0, 0]
            for h, sign in ((0, 1), (1, -1)):
                z = sign * cap * np.sign(k0.astype(np.float64)) if cap else None
                w = np.exp(z - z.max()) if cap else 1.0 * (k0 == (k0.max() if h == 0 else k0.min()))
                w /= w.sum()
                d = 4e-7 * cap
                tol = (np.expm1(2 * d) + 2.0 ** -21 + 2.0 ** -24 * ((p + 1) / 16 + 16)) * (w @ np.abs(v))
                assert (np.abs(got[b.first[s] + i, h] - w @ v) <= tol + 2.0 ** -35 * w.max() * (p + 1) * np.abs(v).max()).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cap", [1e-300, 1e-42, 1e-38, 1e-20, 1e-9, 1e-6])
def test_tiny_caps(ctx, kind, cap):
    """A cap leaves no score larger than itself: a tiny one is the mean."""
    b = Batch(ctx, kind, 16, 1, 3, 64, [40, 700], [1, 60], seed=3)
    b.q[0, 0] = 0.0
    hold(b.run(cap=cap), *expect(b, cap=cap))
    hold(b.run(cap=cap, window=9), *expect(b, cap=cap, window=9))


@pytest.mark.parametrize("kind", ["f32", "rowi8"])
@pytest.mark.parametrize("lens,rows", [([1, 77, 3000], None), ([90, 1500], [60, 90])])
def test_values_up_to_the_largest(ctx, kind, lens, rows):
    """An average of finite values is finite: values up to 3e38, of one sign
    and of both, over one chunk and several."""
    def poison(ks, vs):
        rng = np.random.default_rng(1)
        for v in vs:
            v[:] = rng.uniform(1e38, 3e38, v.shape)
            v[:, :, ::2] *= rng.choice([-1, 1], v[:, :, ::2].shape)

    b = Batch(ctx, kind, 16, 1, 3, 64, lens, rows, seed=3, poison=poison)
    hold(b.run(), *expect(b))


@pytest.mark.parametrize("rows", [None, [60, 90]])
def test_small_values_keep_their_bits(ctx, rows):
    """f32 values down to 1e-25 (products with probabilities stay normal numbers)."""
    def poison(ks, vs):
        for v in vs:
            v *= np.float32(1e-25)

    b = Batch(ctx, "f32", 16, 1, 3, 64, [77, 1500], rows, seed=3, poison=poison)
    hold(b.run(), *expect(b))


# ---- entries that are not finite ---------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("inf", [np.inf, -np.inf])
@pytest.mark.parametrize("lens,rows", [([100, 1400], [64, 3]), ([76, 1400], None)])
@pytest.mark.parametrize("window", [0, 9])
def test_rows_that_see_an_infinite_key(ctx, kind, inf, lens, rows, window):
    """A score of +inf makes its row NaN, as the softmax is; one of -inf leaves
    the other keys' value or makes the row NaN; other rows are right."""
    def poison(ks, vs):
        ks[0][75, 0, 3] = inf
        ks[1][1398, 0, 3] = inf

    b = Batch(ctx, kind, 16, 1, 3, 64, lens, rows, seed=6, poison=poison)
    at = {0: 75, 1: 1398}
    got = b.run(window=window)
    with np.errstate(invalid="ignore"):
        want, tol = expect(b, {s: {j} for s, j in at.items()}, window=window)
    for s, n in enumerate(lens):
        for i in range(b.rows[s]):
            p, r = n - b.rows[s] + i, int(b.first[s]) + i
            for h in range(3):
                sees = at[s] <= p and not (window and p - at[s] >= window)
                if sees and b.q[r, h, 3] * inf > 0:
                    assert np.isnan(got[r, h]).all(), (s, i, h)
                elif sees and np.isnan(got[r, h]).all():
                    continue
                else:
                    assert (np.abs(got[r, h] - want[r, h]) <= tol[r, h]).all(), (s, i, h)


@pytest.mark.parametrize("lens,rows", [([100], [64]), ([75], None), ([71], None)])
@pytest.mark.parametrize("window", [0, 4])
def test_rows_that_see_an_infinite_step(ctx, lens, rows, window):
    """An infinite value gives its int8 row an infinite step over zeros: NaN in
    every channel of the rows that see it; the others are right."""
    def poison(ks, vs):
        vs[0][70, 0, 5] = np.inf

    b = Batch(ctx, "rowi8", 16, 1, 3, 64, lens, rows, seed=7, poison=poison)
    assert np.isnan(b.v[0][70, 0]).all()
    got = b.run(window=window)
    with np.errstate(invalid="ignore"):
        want, tol = expect(b, {0: {70}}, window=window)
    for i in range(b.rows[0]):
        p = lens[0] - b.rows[0] + i
        if 70 <= p and not (window and p - 70 >= window):
            assert np.isnan(got[i]).all(), i
        else:
            assert (np.abs(got[i] - want[i]) <= tol[i]).all(), i


# ---- layouts ------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [32, 64, 128, 256, 512, 1024])
def test_prompts_over_every_page_size(ctx, kind, page):
    """Decode rows and prompts in one call, lengths around the ends of pages."""
    b = Batch(ctx, kind, page, 2, 3, 64, [page - 1, page, page + 1, 2 * page + 17], [60, 1, 45, 70], seed=page)
    hold(b.run(), *expect(b))
    hold(b.run(window=40, cap=25.0), *expect(b, window=40, cap=25.0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rep,rows", [(150, None), (150, [1, 3]), (129, [2, 1]), (300, [5, 1])])
def test_many_heads_a_kv_head(ctx, kind, rep, rows):
    """More heads than a tile has pairs: a row spans several tiles."""
    b = Batch(ctx, kind, 16, 1, rep, 32, [77, 1300], rows, seed=rep)
    hold(b.run(), *expect(b))
    hold(b.run(window=20), *expect(b, window=20))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [[1, 2], [60, 90]])
def test_pages_beyond_32_bits(ctx, kind, rows):
    """Pages, and int8 steps, more than 2^32 bytes apart, written, read back and
    attended to."""
    rng = np.random.default_rng(5)
    page, kv, hd, n_pages, rep = 256, 1, 64, 2, 3
    size = {"f32": 4, "f16": 2, "rowi8": 1}[kind]
    stride, sstride = (1 << 32) // size + 1024, (1 << 30) + 64
    last = kv * page * hd
    k, v = (hip.DeviceArray(((stride * (n_pages - 1) + last) * size,), np.int8) for _ in "kv")
    ks = vs = None
    if kind == "rowi8":
        ks, vs = (hip.DeviceArray((sstride * (n_pages - 1) + kv * page,), np.float32) for _ in "kv")
    c = fa.KvCache(ctx, kind, n_pages, page, kv, hd, k.ptr, v.ptr, ks and ks.ptr, vs and vs.ptr, stride, sstride)
    b = Batch(ctx, kind, page, kv, rep, hd, [200, 250], rows, seed=3)  # the same data, beside it
    table = np.array([[1], [0]], np.int32)
    for s, n in enumerate(b.lens):
        dk, dv = (hip.DeviceArray.from_numpy(x[s].astype(np.float32)) for x in (b.k, b.v))
        slot = hip.DeviceArray.from_numpy(table[s, 0] * page + np.arange(n, dtype=np.int64))
        c.write_dev(dk.ptr, dv.ptr, slot.ptr, n)
        ok, ov = (hip.DeviceArray((n, kv, hd), np.float32) for _ in "kv")
        c.read_dev(slot.ptr, n, ok.ptr, ov.ptr)
        ctx.sync()
        b.k[s], b.v[s] = b.p.stored(b.k[s].astype(np.float32)), b.p.stored(b.v[s].astype(np.float32))
        assert np.array_equal(ok.numpy(), b.k[s]) and np.array_equal(ov.numpy(), b.v[s])
    q, first, lens = (hip.DeviceArray.from_numpy(x) for x in (b.q, b.first, np.asarray(b.lens, np.int32)))
    t, out = hip.DeviceArray.from_numpy(table), hip.DeviceArray(b.q.shape, np.float32)
    c.attn_dev(q.ptr, b.n_row, kv * rep, t.ptr, 1, lens.ptr, 2, out.ptr, first_ptr=first.ptr)
    ctx.sync()
    hold(out.numpy(), *expect(b))


def test_calls_on_another_stream(ctx):
    """On a stream of the caller's, and back on the context's own."""
    b = Batch(ctx, "f16", 16, 2, 3, 64, [300, 70], [70, 1])
    want = b.check()
    other = C.c_void_p()
    hip._chk(hip._hip.hipStreamCreate(C.byref(other)), "hipStreamCreate")
    try:
        ctx.set_stream(other.value)
        assert np.array_equal(b.run(), want)
    finally:
        ctx.sync()
        ctx.set_stream(None)
        hip._chk(hip._hip.hipStreamDestroy(other), "hipStreamDestroy")
    assert np.array_equal(b.run(), want)
