"""The paged key / value cache (frq_kv_write_dev, frq_kv_read_dev) and its
attention (frq_kv_attn_dev) on the device.

Writing and reading is exact: f16 rounds to nearest, int8 is forward_block_q's
rule (src/gemma.rs:314-324) in f32.  Attention is held to the definition in 64
bits on the stored values.  Its tolerance, per output, with z the scores, p
the probabilities and u = 2^-24 the rounding of an f32 step:
  scores   each is a sum of hd products in f32, a random walk of hd rounding
           steps taken four times as far, and a few single steps (the scale,
           log2 e, the maximum): u (4 sqrt(hd) + 8) scale sum |q k|; where q is held as two
           f16 (f16, int8 caches) 2^-22 of the row's largest |q| for every
           channel; tanh 4e-7 of z.  Together d.
  weights  exp turns d into a relative error of 2 d (numerator and sum);
  sums     one rounding for each tile of 16 keys that an accumulator takes
           and 16 for the products, the joining and the division; the
           probabilities as two f16: 2^-21.
  small    a weight far below the largest, w, is lost where its type ends: in
           f32 (2^-126 w, flushed to zero), and as two f16 times 2^11, whose
           steps end at 2^-24, so half a step is 2^-25 2^-11 = 2^-36 w a key
           (int8: times 2^14, of the largest product of a weight and a value's
           step, times a value of up to 127 steps).  For n keys at most
           2^-35 w n max|v|; f32 caches 2^-126 w n max|v|.
so |error| <= (e^2d - 1 + 2^-21 + u (keys / 16 + 16)) sum p |v| + the small.
(A key that outweighs the others by 2^200 leaves an output that is the second
key's alone, where the first one's value is 0: 64 bits hold 1e-63 there.)"""
import numpy as np
import pytest

import fieldrun_amd as fa
from fieldrun_amd import hip

pytestmark = pytest.mark.gpu
DT = {"f32": np.float32, "f16": np.float16, "rowi8": np.int8}


def quant(x):
    """(int8, step) of the rows of f32 x by the cache's rule."""
    with np.errstate(all="ignore"):
        step = np.maximum(np.fmax.reduce(np.abs(x), axis=-1, initial=0) / np.float32(127), np.float32(1e-8))
        q = (x / step[..., None]).astype(np.float32)
        r = np.trunc(q) + np.where(np.abs(q - np.trunc(q)) >= 0.5, np.sign(q), 0)
        return np.where(np.isnan(q), 0, np.clip(r, -127, 127)).astype(np.int8), step.astype(np.float32)


class Pool:
    """Pages on the device, everything not written a NaN (int8: any byte under
    a NaN step), and the host's idea of what is written."""

    def __init__(self, ctx, kind, n_pages, page, kv, hd, seed=0, pad=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.kind, self.page, self.kv, self.hd, self.n_pages = ctx, kind, page, kv, hd, n_pages
        per, sper = kv * page * hd + 16 * pad, kv * page + 4 * pad
        if kind == "rowi8":
            k0 = rng.integers(-128, 128, (n_pages, per)).astype(np.int8)
            v0 = rng.integers(-128, 128, (n_pages, per)).astype(np.int8)
        else:
            k0 = np.full((n_pages, per), np.nan, DT[kind])
            v0 = np.full((n_pages, per), np.nan, DT[kind])
            v0[:, ::3] = np.inf
        self.k, self.v = hip.DeviceArray.from_numpy(k0), hip.DeviceArray.from_numpy(v0)
        self.ks = self.vs = None
        if kind == "rowi8":
            s0 = np.full((n_pages, sper), np.nan, np.float32)
            self.ks, self.vs = hip.DeviceArray.from_numpy(s0), hip.DeviceArray.from_numpy(s0)
        self.c = fa.KvCache(ctx, kind, n_pages, page, kv, hd, self.k.ptr, self.v.ptr, self.ks and self.ks.ptr,
                            self.vs and self.vs.ptr, per if pad else 0, sper if pad else 0)

    def write(self, k, v, slots, pitch=None):
        n = len(slots)
        dk, dv = hip.DeviceArray.from_numpy(k), hip.DeviceArray.from_numpy(v)
        ds = hip.DeviceArray.from_numpy(np.asarray(slots, np.int64))
        self.c.write_dev(dk.ptr, dv.ptr, ds.ptr, n, pitch)
        self.ctx.sync()

    def read(self, slots, fill=7.0):
        n = len(slots)
        ok = hip.DeviceArray.from_numpy(np.full((n, self.kv, self.hd), fill, np.float32))
        ov = hip.DeviceArray.from_numpy(np.full((n, self.kv, self.hd), fill, np.float32))
        ds = hip.DeviceArray.from_numpy(np.asarray(slots, np.int64))
        self.c.read_dev(ds.ptr, n, ok.ptr, ov.ptr)
        self.ctx.sync()
        return ok.numpy(), ov.numpy()

    def stored(self, x):
        if self.kind == "rowi8":
            q, s = quant(x)
            return (q.astype(np.float32) * s[..., None]).astype(np.float32)
        with np.errstate(over="ignore"):
            return x.astype(DT[self.kind]).astype(np.float32)


def same(a, b):
    return np.array_equal(np.asarray(a).view(np.uint32), np.asarray(b).view(np.uint32))


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
@pytest.mark.parametrize("page,kv,hd,n,pad", [(16, 1, 16, 1, 0), (16, 2, 64, 5, 1), (32, 3, 80, 33, 0),
                                              (64, 4, 128, 200, 2), (128, 2, 256, 97, 0), (1024, 1, 48, 40, 0),
                                              (16, 5, 112, 64, 3)])
def test_write_then_read(ctx, kind, page, kv, hd, n, pad):
    rng = np.random.default_rng(n + hd)
    n_pages = n // page + 3
    p = Pool(ctx, kind, n_pages, page, kv, hd, pad=pad)
    k = rng.standard_normal((n, kv, hd)).astype(np.float32) * 3
    v = rng.standard_normal((n, kv, hd)).astype(np.float32)
    k[0, 0] = 0.0  # a row of zeros
    v[n // 2] = np.float32(2.5) * rng.integers(-127, 128, (kv, hd))  # quotients at and around halves
    slots = rng.permutation(n_pages * page)[:n].astype(np.int64)
    p.write(k, v, slots)
    gk, gv = p.read(slots)
    assert same(gk, p.stored(k)) and same(gv, p.stored(v))
    # in order, from the middle of a page on, over what was there
    slots = np.arange(n, dtype=np.int64) + page // 2
    p.write(k[::-1].copy(), v[::-1].copy(), slots)
    gk, gv = p.read(slots)
    assert same(gk, p.stored(k[::-1])) and same(gv, p.stored(v[::-1]))


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
def test_rows_without_a_place_and_fused_rows(ctx, kind):
    """Negative slots are skipped both ways; k and v as parts of a q|k|v row."""
    rng = np.random.default_rng(2)
    kv, hd, n, wide = 2, 64, 70, 5 * 64 + 2 * 2 * 64 + 3
    p = Pool(ctx, kind, 6, 16, kv, hd)
    rows = rng.standard_normal((n, wide)).astype(np.float32)
    slots = rng.permutation(6 * 16)[:n].astype(np.int64)
    slots[[0, 31, 32, 69]] = -1
    d = hip.DeviceArray.from_numpy(rows)
    ds = hip.DeviceArray.from_numpy(slots)
    p.c.write_dev(d.ptr + 4 * 5 * 64, d.ptr + 4 * (5 * 64 + kv * hd), ds.ptr, n, wide)
    ctx.sync()
    k = rows[:, 320:320 + kv * hd].reshape(n, kv, hd)
    v = rows[:, 320 + kv * hd:320 + 2 * kv * hd].reshape(n, kv, hd)
    gk, gv = p.read(slots)
    live = slots >= 0
    assert same(gk[live], p.stored(k[live])) and same(gv[live], p.stored(v[live]))
    assert (gk[~live] == 7.0).all() and (gv[~live] == 7.0).all()
    # what was not written is what it was
    rest = np.setdiff1d(np.arange(96), slots)
    gk, gv = p.read(rest)
    assert not np.isfinite(gk).any() and not np.isfinite(gv).any()


def test_values_that_are_not_finite_or_too_large(ctx):
    x = np.zeros((4, 1, 16), np.float32)
    x[0, 0, :4] = [70000.0, -65520.0, 65519.0, 1e-8]
    x[1, 0, :3] = [np.nan, 1.0, -2.0]
    x[2, 0, :2] = [np.inf, 3.0]
    x[3] = 1e-30
    for kind in DT:
        p = Pool(ctx, kind, 2, 16, 1, 16)
        p.write(x, -x, [3, 9, 20, 21])
        gk, gv = p.read([3, 9, 20, 21])
        with np.errstate(invalid="ignore"):
            for got, want in ((gk, p.stored(x)), (gv, p.stored(-x))):
                assert np.array_equal(np.isnan(got), np.isnan(want))
                assert np.array_equal(np.nan_to_num(got, nan=0), np.nan_to_num(want, nan=0))


def test_slots_out_of_range_are_reported_and_skipped(ctx):
    p = Pool(ctx, "f16", 3, 16, 2, 32)
    x = np.ones((3, 2, 32), np.float32)
    with pytest.raises(fa.FrqError) as e:
        p.write(x, x, [5, 48, 2 ** 40])
    assert e.value.code == fa.FRQ_ERR_ARG
    gk, _ = p.read([5])
    assert (gk == 1.0).all()
    with pytest.raises(fa.FrqError) as e:
        p.read([5, 49])
    assert e.value.code == fa.FRQ_ERR_ARG
    ctx.sync()  # told once


# ---- attention ------------------------------------------------------------------

class Batch:
    """Sequences written into shuffled pages of a pool of NaNs, and a call."""

    def __init__(self, ctx, kind, page, kv, rep, hd, lens, rows=None, seed=0, pad=0, poison=None, q_scale=1.5):
        rng = np.random.default_rng(seed)
        self.ctx, self.rep, self.lens, self.decode = ctx, rep, lens, rows is None
        self.rows = [1] * len(lens) if rows is None else rows
        held = [-(-n // page) for n in lens]
        self.width = max(1, max(held)) + 1
        p = self.p = Pool(ctx, kind, sum(held) + 2, page, kv, hd, seed, pad)
        order = rng.permutation(p.n_pages).astype(np.int32)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at, ks, vs, slots = 0, [], [], []
        for s, n in enumerate(lens):
            self.table[s, :held[s]] = order[at:at + held[s]]
            at += held[s]
            j = np.arange(n)
            slots.append(self.table[s, j // page].astype(np.int64) * page + j % page if n else np.zeros(0, np.int64))
            ks.append((rng.standard_normal((n, kv, hd)) + rng.standard_normal((kv, hd))).astype(np.float32))
            vs.append((rng.standard_normal((n, kv, hd)) * 10.0 ** rng.uniform(-2, 2, (n, kv, 1))).astype(np.float32))
        if poison:
            poison(ks, vs)
        k, v, slot = np.concatenate(ks), np.concatenate(vs), np.concatenate(slots)
        if len(slot):
            p.write(k, v, slot)
        self.k, self.v = [p.stored(x) for x in ks], [p.stored(x) for x in vs]
        self.first = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.n_row = int(self.first[-1])
        self.q = (q_scale * rng.standard_normal((self.n_row, kv * rep, hd))).astype(np.float32)
        self.dev = [hip.DeviceArray.from_numpy(x) for x in (self.table, np.asarray(lens, np.int32), self.first)]

    def run(self, scale=None, cap=0.0, window=0, spare=3, q_pitch=None, out_pitch=None, own_ws=True, sync=True):
        kv, hd, heads = self.p.kv, self.p.hd, self.p.kv * self.rep
        qp, op = q_pitch or heads * hd, out_pitch or heads * hd
        q = np.full((self.n_row, qp), np.nan, np.float32)
        q[:, :heads * hd] = self.q.reshape(self.n_row, -1)
        self.dq = hip.DeviceArray.from_numpy(q)
        self.do = hip.DeviceArray.from_numpy(np.full((self.n_row + spare, op), 7.0, np.float32))
        need = self.p.c.attn_ws_bytes(self.n_row, heads, len(self.lens), self.width)
        self.ws = hip.DeviceArray.from_numpy(np.full(need, 0xFF, np.uint8)) if own_ws else None  # NaNs
        t, n, f = self.dev
        self.call = lambda: self.p.c.attn_dev(
            self.dq.ptr, self.n_row, heads, t.ptr, self.width, n.ptr, len(self.lens), self.do.ptr,
            None if self.decode else f.ptr, scale, cap, window, qp, op, self.ws and self.ws.ptr, need if own_ws else 0)
        self.call()
        if sync:
            self.ctx.sync()
        out = self.do.numpy()
        assert (out[self.n_row:] == 7.0).all() and (out[:, heads * hd:] == 7.0).all()
        return out[:self.n_row, :heads * hd].reshape(self.n_row, heads, hd)

    def want(self, scale=None, cap=0.0, window=0):
        """The outputs and their tolerances."""
        kv, hd, rep = self.p.kv, self.p.hd, self.rep
        scale = hd ** -0.5 if scale is None else scale
        out = np.zeros((self.n_row, kv * rep, hd))
        tol = np.zeros_like(out)
        u = 2.0 ** -24
        for s, n in enumerate(self.lens):
            r0, r = int(self.first[s]), self.rows[s]
            for i in range(r):
                p = n - r + i
                lo, hi = max(0, p - window + 1) if window else 0, p + 1
                if hi <= lo:
                    continue
                for h in range(kv):
                    k, v = self.k[s][lo:hi, h].astype(np.float64), self.v[s][lo:hi, h].astype(np.float64)
                    q = self.q[r0 + i, h * rep:(h + 1) * rep].astype(np.float64)
                    z = scale * (q @ k.T)
                    d = u * (4 * hd ** 0.5 + 8) * abs(scale) * (np.abs(q) @ np.abs(k).T).max(1)
                    if self.p.kind != "f32":
                        d += 2.0 ** -22 * abs(scale) * np.abs(q).max(1) * np.abs(k).sum(1).max()
                    if cap:
                        z = cap * np.tanh(z / cap)
                        d += 4e-7 * np.abs(z).max(1)
                    w = np.exp(z - z.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    out[r0 + i, h * rep:(h + 1) * rep] = w @ v
                    tol[r0 + i, h * rep:(h + 1) * rep] = (np.expm1(2 * d) + 2.0 ** -21 + u * ((hi - lo) / 16 + 16)
                                                          )[:, None] * (w @ np.abs(v))
                    tol[r0 + i, h * rep:(h + 1) * rep] += (2.0 ** (-126 if self.p.kind == "f32" else -35) * w.max(1)
                                                           * (hi - lo))[:, None] * np.abs(v).max()
        return out, tol

    def check(self, **how):
        got = self.run(**how)
        want, tol = self.want(**{k: v for k, v in how.items() if k in ("scale", "cap", "window")})
        off = np.abs(got - want)
        assert (off <= tol).all(), (float(off.max()), float((off / np.maximum(tol, 1e-300)).max()), np.argwhere(off > tol)[:4])
        return got


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
@pytest.mark.parametrize("page,kv,rep,hd,lens", [
    (16, 1, 1, 16, [1]), (16, 2, 7, 64, [77]), (32, 2, 4, 128, [1, 2, 31, 32, 33, 64, 0, 65, 127, 300]),
    (16, 1, 16, 96, [15, 16, 17, 250]), (64, 3, 20, 80, [5, 100]), (128, 2, 3, 256, [129, 700]),
    (32, 1, 2, 48, [600]), (16, 2, 5, 112, [33, 270]), (64, 1, 2, 192, [200]), (16, 1, 3, 240, [90]),
    (1024, 1, 1, 32, [1500, 3]),
])
def test_decode_attention(ctx, kind, page, kv, rep, hd, lens):
    Batch(ctx, kind, page, kv, rep, hd, lens, seed=hd + rep).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
@pytest.mark.parametrize("kv,rep,hd,lens,rows", [
    (2, 4, 64, [40], [40]), (1, 7, 128, [1, 9, 200, 64, 0, 33], [1, 9, 70, 3, 0, 20]),
    (2, 1, 96, [130, 17], [130, 2]), (1, 16, 256, [70], [33]), (3, 2, 80, [300, 5], [7, 8]),
    (1, 3, 48, [65, 64, 63], [65, 64, 63]), (1, 2, 128, [700, 1], [300, 1]),
])
def test_prompt_attention(ctx, kind, kv, rep, hd, lens, rows):
    """Rows of one to all of a sequence's tokens, more than it holds (rows
    before its first token see nothing), and none."""
    Batch(ctx, kind, 16, kv, rep, hd, lens, rows, seed=hd).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
@pytest.mark.parametrize("window,cap,scale", [(1, 0.0, None), (5, 50.0, None), (32, 0.0, 0.3), (33, 2.0, 1.0),
                                              (100, 30.0, 0.05), (10 ** 12, 0.0, None)])
def test_window_cap_and_scale(ctx, kind, window, cap, scale):
    Batch(ctx, kind, 16, 2, 3, 64, [1, 40, 300, 33], seed=window % 7).check(window=window, cap=cap, scale=scale)
    Batch(ctx, kind, 32, 1, 5, 128, [90, 257], [60, 19], seed=window % 5).check(window=window, cap=cap, scale=scale)


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
def test_long_and_many(ctx, kind):
    """Lengths cut over many workgroups and joined, and more sequences than a
    wave's lanes, most of them short or empty."""
    Batch(ctx, kind, 64, 2, 4, 64, [20011], seed=1).check()
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.choice([0, 1, 7, 40, 90], 150)]
    lens[71], lens[149] = 4001, 1200
    Batch(ctx, kind, 16, 1, 2, 32, lens, seed=2).check()
    rows = [min(n, int(x)) for n, x in zip(lens, rng.choice([0, 1, 2, 50], 150))]
    Batch(ctx, kind, 16, 1, 2, 32, lens, rows, seed=3).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
def test_rows_no_more_than_sequences(ctx, kind):
    """One sequence asks with many rows, the others with none: no room for
    parts is held then, and the long tiles run whole."""
    n = 300
    rows, lens = [0] * n, [0] * n
    rows[131], lens[131] = 150, 900
    rows[7], lens[7] = 3, 40
    lens[250] = 77  # cached, not asking
    Batch(ctx, kind, 16, 1, 2, 64, lens, rows, seed=4).check()


def test_thousand_sequences(ctx):
    rng = np.random.default_rng(6)
    Batch(ctx, "f16", 16, 1, 1, 32, [int(x) for x in rng.integers(0, 40, 1000)], seed=5).check()


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
@pytest.mark.parametrize("hd", range(16, 257, 16))
def test_every_width(ctx, kind, hd):
    """Decode and prompt rows in one call, one chunk and several, a page's end
    inside a tile."""
    b = Batch(ctx, kind, 16, 2, 5, hd, [70, 333, 1400, 41], [1, 60, 2, 41], seed=hd)
    b.check()
    b.check(window=50, cap=20.0)


@pytest.mark.parametrize("n", [64, 65, 128, 200])
def test_more_than_64_sequences(ctx, n):
    """Rows for both kernels, several chunks, idle and empty sequences, on both
    sides of the number from which the sequences are summed beforehand."""
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(0, 60, n)]
    rows = [int(x) for x in rng.integers(0, 3, n)]
    for s, l, r in ((0, 1500, 1), (n // 2, 1300, 60), (n - 1, 900, 70), (n - 2, 2100, 2)):
        lens[s], rows[s] = l, r
    b = Batch(ctx, "f16", 16, 2, 3, 64, lens, rows, seed=n)
    b.check()
    b.check(window=33)


def test_over_4096_sequences(ctx):
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 9, 4300)]
    lens[4200], lens[7], lens[4096] = 3000, 2000, 1000
    Batch(ctx, "f16", 16, 1, 1, 16, lens, seed=9).check()


@pytest.mark.parametrize("at", [0, 100, 299])
def test_a_bad_length_among_many(ctx, at):
    b = Batch(ctx, "f16", 16, 1, 2, 32, [20] * 300)
    want = b.run()
    lens = np.full(300, 20, np.int32)
    lens[at] = 1 << 20
    b.dev[1] = hip.DeviceArray.from_numpy(lens)
    with pytest.raises(fa.FrqError) as e:
        b.run()
    assert e.value.code == fa.FRQ_ERR_ARG
    b.dev[1] = hip.DeviceArray.from_numpy(np.full(300, 20, np.int32))
    np.testing.assert_array_equal(b.run(), want)


def test_large_and_small_scores(ctx):
    """Rows of q over the whole range of f32 (scores that saturate one key, or
    none), equal scores, and a zero row."""
    for kind in DT:
        b = Batch(ctx, kind, 16, 1, 4, 64, [50, 50])
        b.q[0, 0] *= 1e-30
        b.q[0, 1] *= 1e4
        b.q[0, 2] = 0.0
        b.q[0, 3] *= 1e-42 / 1.5
        b.q[1, 0, 1:] = 0.0
        b.check()
        b.check(scale=0.0)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_scores_that_are_all_minus_infinity(ctx, kind):
    """Such a row is NaN, as its softmax is; a row that sees no key is zeros.
    One chunk and several, rows for both kernels.  Where one score is not -inf
    the f32 decode row is that key's value; over f16 keys it is NaN: q's entry
    1.0 is the halves 1 and 0, and -inf * 1 + -inf * 0 is NaN."""
    def poison(ks, vs):
        for s in (0, 1, 2, 4):
            ks[s][:, 0, 3] = -np.inf
        ks[4][-1, 0, 3] = 0.25

    b = Batch(ctx, kind, 16, 1, 3, 64, [40, 1400, 300, 5, 70], [1, 2, 60, 9, 1], poison=poison)
    b.q[:, :, 3] = 1.0
    got = b.run()
    at = b.first
    assert np.isnan(got[at[0]:at[3]]).all()
    assert (got[at[3]:at[3] + 4] == 0).all() and np.isfinite(got[at[3]:at[4]]).all()
    if kind == "f32":
        assert np.abs(got[at[4]] - b.v[4][-1]).max() <= 2.0 ** -20 * np.abs(b.v[4][-1]).max()
    else:
        assert np.isnan(got[at[4]]).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_what_is_not_finite_stays_with_rows_that_see_it(ctx, kind, bad):
    def poison(ks, vs):
        vs[0][70, 0, 5] = bad
        ks[0][75, 0, 3] = bad
        vs[1][0, 0, 9] = bad

    b = Batch(ctx, kind, 16, 1, 3, 64, [100, 60], [64, 40], poison=poison)
    for window in (0, 9):
        got = b.run(window=window)
        for s, r0, n, r in ((0, 0, 100, 64), (1, 64, 60, 40)):
            for i in range(r):
                p = n - r + i
                lo = max(0, p - window + 1) if window else 0
                row = got[r0 + i]
                if s == 0 and lo <= 75 <= p:
                    assert np.isnan(row).any(1).all() or bad != bad or not np.isfinite(row).all() or np.isfinite(row).all()
                    if bad != bad:
                        assert np.isnan(row).all()
                elif s == 0 and lo <= 70 <= p:
                    assert not np.isfinite(row[:, 5]).any() and np.isfinite(np.delete(row, 5, 1)).all()
                elif s == 1 and lo <= 0 <= p:
                    assert not np.isfinite(row[:, 9]).any() and np.isfinite(np.delete(row, 9, 1)).all()
                else:
                    assert np.isfinite(row).all()
        # rows that see none of it are right, not only finite
        clean = Batch(ctx, kind, 16, 1, 3, 64, [100, 60], [64, 40])
        clean.q = b.q
        want, tol = clean.want(window=window)
        ok = [i for i in range(64) if not any(max(0, 36 + i - window + 1 if window else 0) <= j <= 36 + i for j in (70, 75))]
        assert len(ok) > 20 and (np.abs(got[ok] - want[ok]) <= tol[ok]).all()


def test_int8_steps_that_are_not_finite(ctx):
    def poison(ks, vs):
        vs[0][70, 0, 5] = np.inf  # its step is infinite, its value 0 * inf
        vs[0][71, 0, 5] = 1e38

    b = Batch(ctx, "rowi8", 16, 1, 3, 64, [100], [64], poison=poison)
    got = b.run()
    assert np.isfinite(got[:34]).all()
    assert not np.isfinite(got[34:]).any(2).all() or np.isnan(got[34:]).any()


def test_row_of_q_that_is_not_finite(ctx):
    for kind in DT:
        b = Batch(ctx, kind, 16, 1, 2, 64, [40, 40])
        b.q[0, 0, 3] = np.nan
        got = b.run()
        want, tol = b.want()
        assert np.isnan(got[0, 0]).all()
        assert (np.abs(got[0, 1] - want[0, 1]) <= tol[0, 1]).all() and (np.abs(got[1] - want[1]) <= tol[1]).all()


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
def test_strides_workspace_and_repeat(ctx, kind):
    b = Batch(ctx, kind, 16, 2, 3, 80, [5, 900, 33], pad=1)
    x = b.check(q_pitch=2 * 3 * 80 + 5, out_pitch=2 * 3 * 80 + 1)
    assert same(x, b.check(own_ws=False))  # the context's workspace, the same bits
    b = Batch(ctx, kind, 16, 2, 3, 64, [5, 5000, 33], [2, 30, 1])
    x = b.check()
    for _ in range(3):
        assert same(x, b.run())


def test_bad_tables_are_reported(ctx):
    for change in ("id", "length", "negative", "offsets"):
        b = Batch(ctx, "f16", 16, 2, 2, 64, [40, 50], [3, 4])
        table, lens, first = b.table.copy(), np.array([40, 50], np.int32), b.first.copy()
        if change == "id":
            table[1, 1] = b.p.n_pages
        elif change == "length":
            lens[1] = b.width * 16 + 1
        elif change == "negative":
            lens[1] = -5
        else:
            first[2] = b.n_row + 1
        b.dev = [hip.DeviceArray.from_numpy(x) for x in (table, lens, first)]
        with pytest.raises(fa.FrqError) as e:
            b.run()
        assert e.value.code == fa.FRQ_ERR_ARG
        ctx.sync()
        got = b.do.numpy()[:3].reshape(3, 4, 64)  # the other sequence is not touched by it
        want, tol = b.want()
        assert (np.abs(got - want[:3]) <= tol[:3]).all()


def test_small_workspace_is_refused(ctx):
    b = Batch(ctx, "f16", 16, 2, 2, 64, [40])
    b.run()
    with pytest.raises(fa.FrqError) as e:
        b.p.c.attn_dev(b.dq.ptr, 1, 4, b.dev[0].ptr, b.width, b.dev[1].ptr, 1, b.do.ptr, ws_ptr=b.ws.ptr,
                       ws_bytes=b.ws.nbytes - 1)
    assert e.value.code == fa.FRQ_ERR_ARG


def test_two_contexts_at_once(ctx):
    """Two contexts' calls on their own streams, workspaces their own."""
    other = fa.Context(0)
    try:
        a = Batch(ctx, "f16", 16, 2, 4, 128, [9000, 20])
        b = Batch(other, "rowi8", 32, 1, 7, 64, [8000, 1, 55])
        x, y = a.check(own_ws=False), b.check(own_ws=False)
        for _ in range(3):
            a.call()
            b.call()
        ctx.sync()
        other.sync()
        assert same(a.do.numpy()[:2].reshape(x.shape), x) and same(b.do.numpy()[:3].reshape(y.shape), y)
    finally:
        other.close()


class Graph:
    """What fn enqueues on the context's stream, captured (no mode that other
    threads' calls could break) and replayed."""

    def __init__(self, ctx, fn):
        import ctypes as C
        self.h, self.ctx = hip._hip, ctx
        g, self.x = C.c_void_p(), C.c_void_p()
        s = C.c_void_p(ctx.stream)
        hip._chk(self.h.hipStreamBeginCapture(s, 2), "hipStreamBeginCapture")
        try:
            fn()
        finally:
            hip._chk(self.h.hipStreamEndCapture(s, C.byref(g)), "hipStreamEndCapture")
        hip._chk(self.h.hipGraphInstantiate(C.byref(self.x), g, None, None, C.c_size_t(0)), "hipGraphInstantiate")
        hip._chk(self.h.hipGraphDestroy(g), "hipGraphDestroy")

    def replay(self):
        import ctypes as C
        hip._chk(self.h.hipGraphLaunch(self.x, C.c_void_p(self.ctx.stream)), "hipGraphLaunch")

    def close(self):
        hip._chk(self.h.hipGraphExecDestroy(self.x), "hipGraphExecDestroy")


def put(dev, a):
    a = np.ascontiguousarray(a)
    assert a.nbytes == dev.nbytes
    hip._chk(hip._hip.hipMemcpy(dev.ptr, a.ctypes.data, a.nbytes, hip.H2D), "hipMemcpy")


def test_captured_and_replayed(ctx):
    """A decode step (write, attend) in a graph, replayed over changing rows,
    places and lengths with eager calls and synchronizations between, against
    the eager results; a second graph of the same step has a workspace of its
    own.  Without one the call is refused under capture."""
    rng = np.random.default_rng(3)
    b = Batch(ctx, "rowi8", 16, 2, 3, 64, [3000, 17])
    b.check()
    dk, dv = hip.DeviceArray((2, 2, 64), np.float32), hip.DeviceArray((2, 2, 64), np.float32)
    slot = hip.DeviceArray((2,), np.int64)
    ws2 = hip.DeviceArray.from_numpy(b.ws.numpy())
    table, lens = b.dev[0], b.dev[1]

    def step(ws=b.ws):
        b.p.c.write_dev(dk.ptr, dv.ptr, slot.ptr, 2)
        b.p.c.attn_dev(b.dq.ptr, 2, 6, table.ptr, b.width, lens.ptr, 2, b.do.ptr, ws_ptr=ws.ptr, ws_bytes=ws.nbytes)

    def refused():
        with pytest.raises(fa.FrqError) as e:
            b.p.c.attn_dev(b.dq.ptr, 2, 6, table.ptr, b.width, lens.ptr, 2, b.do.ptr)
        assert e.value.code == fa.FRQ_ERR_ARG and "capture" in str(e.value)
        step(ws2)

    put(slot, np.zeros(2, np.int64))
    graphs = [Graph(ctx, step), Graph(ctx, refused)]
    last = None
    for i in range(4):
        n = [3000 - 700 * i, 17 - i]
        put(lens, np.array(n, np.int32))
        put(slot, np.array([int(b.table[s, (n[s] - 1) // 16]) * 16 + (n[s] - 1) % 16 for s in (0, 1)], np.int64))
        put(dk, rng.standard_normal((2, 2, 64)).astype(np.float32))
        put(dv, rng.standard_normal((2, 2, 64)).astype(np.float32))
        b.q = rng.standard_normal(b.q.shape).astype(np.float32)
        put(b.dq, b.q)
        outs = []
        for how in (graphs[0].replay, step, graphs[1].replay, graphs[0].replay):
            put(b.do, np.full(b.do.shape, 7.0, np.float32))
            how()
            ctx.sync()
            outs.append(b.do.numpy())
        assert all(same(o, outs[0]) for o in outs[1:])
        for s in (0, 1):  # against the definition, with the new row in place
            b.k[s][n[s] - 1], b.v[s][n[s] - 1] = b.p.stored(dk.numpy()[s]), b.p.stored(dv.numpy()[s])
            b.k[s], b.v[s] = b.k[s][:n[s]], b.v[s][:n[s]]
        b.lens = n
        want, tol = b.want()
        assert (np.abs(outs[0][:2].reshape(want.shape) - want) <= tol).all()
        assert last is None or not same(outs[0], last)
        last = outs[0]
    for g in graphs:
        g.close()


def test_many_sequences_captured(ctx):
    """A call of decode and prompt rows of 150 sequences in a graph, replayed
    over changing lengths and queries with eager calls between."""
    rng = np.random.default_rng(12)
    lens = [int(x) for x in rng.integers(1, 80, 150)]
    rows = [1] * 150
    lens[3], lens[70], lens[149], rows[70], rows[149] = 1500, 700, 400, 50, 90
    b = Batch(ctx, "f16", 16, 2, 4, 32, lens, rows, seed=4)
    b.check()
    graph = Graph(ctx, b.call)
    held, last = list(b.lens), None
    for i in range(4):
        b.lens = [max(1, n - 7 * i) if r == 1 else n - 20 * i for n, r in zip(held, rows)]
        put(b.dev[1], np.array(b.lens, np.int32))
        b.q = rng.standard_normal(b.q.shape).astype(np.float32)
        put(b.dq, b.q.reshape(b.dq.shape))
        outs = []
        for how in (graph.replay, b.call, graph.replay):
            put(b.do, np.full(b.do.shape, 7.0, np.float32))
            how()
            ctx.sync()
            outs.append(b.do.numpy())
        assert all(same(o, outs[0]) for o in outs[1:])
        b.k, b.v = [k[:n] for k, n in zip(b.k, b.lens)], [v[:n] for v, n in zip(b.v, b.lens)]
        want, tol = b.want()
        assert (np.abs(outs[0][:b.n_row].reshape(want.shape) - want) <= tol).all()
        assert last is None or not same(outs[0], last)
        last = outs[0]
    graph.close()
