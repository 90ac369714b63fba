"""frq_kv_append_dev on the device: fused rows with biases, head norms and the
rotation, against the formulas in numpy's 64 bits.

Tolerances: the results are formed in 64 bits and rounded to f32 once, so q is
off by half a step, 2^-24 of its value (below the normal numbers 2^-150), and
what 64 bits leave: 2^-48 of the head's terms, some 30 operations of 2^-53 each
(the angle's own rounding is the same on both sides).  Keys and values then
take frq_kv_write_dev's rounding: the bytes have to be those that call writes for
the f32 rows that an f32 cache holds."""
import ctypes as C

import numpy as np
import pytest

import fieldrun_amd as fa
from fieldrun_amd import hip
from test_gpu_kv import Graph, Pool, put, same

pytestmark = pytest.mark.gpu
up = hip.DeviceArray.from_numpy


class Rows:
    """Fused rows, what is done to them, and the call."""

    def __init__(self, ctx, kv, rep, hd, n, rot, pairs=False, bias=True, qn=False, kn=False, far=5000, seed=0, extra=0,
                 eps=1e-6):
        rng = np.random.default_rng(seed)
        self.ctx, self.kv, self.heads, self.hd, self.n, self.rot, self.pairs, self.eps = (
            ctx, kv, kv * rep, hd, n, rot, pairs, eps)
        self.wide = (self.heads + 2 * kv) * hd
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.x = f(n, self.wide + extra) * np.exp(rng.uniform(-3, 3, (n, 1))).astype(np.float32)
        self.bias = f(self.wide) if bias else None
        self.qn, self.kn = (1 + f(hd) / 4 if qn else None), (1 + f(hd) / 4 if kn else None)
        self.pos = rng.integers(-far // 4, far, n).astype(np.int32)
        self.freq = 1e4 ** (-2.0 * np.arange(rot // 2) / max(1, rot))
        self.keep = [None if a is None else up(a) for a in (self.bias, self.qn, self.kn)]
        self.dx, self.dpos, self.dfreq = up(self.x), up(self.pos), up(self.freq)
        at = [a and a.ptr for a in self.keep]
        self.how = fa.Rotary(rot, self.dfreq.ptr if rot else None, pairs, at[0], at[1], at[2], eps)

    def call(self, pool, slots, q_pitch=None, spare=2):
        """q's rows; keys and values are in the pool."""
        qp = q_pitch or self.heads * self.hd
        self.dq = up(np.full((self.n + spare, qp), 7.0, np.float32))
        self.ds = up(np.asarray(slots, np.int64))
        pool.c.append_dev(self.dx.ptr, self.heads, self.dpos.ptr if self.rot else None, self.ds.ptr, self.n, self.dq.ptr,
                          self.how, self.x.shape[1], qp)
        self.ctx.sync()
        q = self.dq.numpy()
        assert (q[self.n:] == 7.0).all() and (q[:, self.heads * self.hd:] == 7.0).all()
        return q[:self.n, :self.heads * self.hd].reshape(self.n, self.heads, self.hd)

    def want(self):
        """(n, heads + 2 kv, hd) in 64 bits, and the size of each head's terms."""
        x = self.x[:, :self.wide].astype(np.float64)
        if self.bias is not None:
            x = x + self.bias
        x = x.reshape(self.n, -1, self.hd)
        size = np.abs(x).max(-1, keepdims=True)
        for lo, hi, gain in ((0, self.heads, self.qn), (self.heads, self.heads + self.kv, self.kn)):
            if gain is not None:
                f = gain / np.sqrt((x[:, lo:hi] ** 2).mean(-1, keepdims=True) + self.eps)
                x[:, lo:hi] *= f
                size[:, lo:hi] *= np.abs(f).max(-1, keepdims=True)
        half, t = self.rot // 2, self.pos[:, None, None].astype(np.float64) * self.freq
        c, s = np.cos(t), np.sin(t)
        y = x.copy()
        ia, ib = (slice(0, self.rot, 2), slice(1, self.rot, 2)) if self.pairs else (slice(0, half), slice(half, self.rot))
        qk = slice(0, self.heads + self.kv)
        a, b = x[:, qk, ia], x[:, qk, ib]
        y[:, qk, ia], y[:, qk, ib] = a * c - b * s, b * c + a * s
        return y, size


def check_rows(got, want, size):
    tol = 2.0 ** -24 * np.abs(want) * (1 + 2.0 ** -20) + 2.0 ** -48 * size + 2.0 ** -150
    off = np.abs(got - want)
    assert (off <= tol).all(), (float(off.max()), np.argwhere(off > tol)[:4])


def raw(pool):
    return [a.numpy().view(np.uint8) for a in (pool.k, pool.v, pool.ks, pool.vs) if a is not None]


def check(r, kind, page, pad=0, q_pitch=None, seed=0, skip=()):
    rng = np.random.default_rng(seed)
    n_pages = r.n // page + 3
    slots = rng.permutation(n_pages * page)[:r.n].astype(np.int64)
    slots[list(skip)] = -1
    if r.n > 40:  # a prompt's rows lie in order
        slots[:33] = np.setdiff1d(np.arange(n_pages * page), slots[33:])[:33]
    p = [Pool(r.ctx, k, n_pages, page, r.kv, r.hd, seed, pad) for k in ("f32", kind, kind)]
    q = r.call(p[0], slots, q_pitch)
    want, size = r.want()
    check_rows(q, want[:, :r.heads], size[:, :r.heads])
    live = slots >= 0
    k, v = p[0].read(slots)
    check_rows(k[live], want[live, r.heads:r.heads + r.kv], size[live, r.heads:r.heads + r.kv])
    check_rows(v[live], want[live, r.heads + r.kv:], 0 * size[live, r.heads + r.kv:])
    assert same(r.call(p[1], slots, q_pitch), q)
    p[2].write(np.where(live[:, None, None], k, 0), np.where(live[:, None, None], v, 0), slots)
    for a, b in zip(raw(p[1]), raw(p[2])):  # all of the pool, what was not written too
        assert np.array_equal(a, b)


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
@pytest.mark.parametrize("page,kv,rep,hd,n,rot,pairs,bias,qn,kn", [
    (16, 1, 1, 16, 1, 16, False, False, False, False), (16, 2, 7, 64, 1, 64, False, True, False, False),
    (32, 5, 3, 80, 61, 32, True, False, True, True), (16, 3, 2, 48, 9, 8, False, True, True, False),
    (64, 4, 7, 128, 200, 128, False, True, False, True), (16, 1, 4, 256, 33, 256, True, True, True, True),
    (128, 2, 1, 240, 70, 120, False, False, False, False), (16, 2, 3, 112, 40, 0, False, True, True, True),
    (16, 8, 4, 192, 17, 192, False, False, True, True), (1024, 1, 16, 32, 300, 32, False, True, False, False),
])
def test_rows(ctx, kind, page, kv, rep, hd, n, rot, pairs, bias, qn, kn):
    check(Rows(ctx, kv, rep, hd, n, rot, pairs, bias, qn, kn, seed=hd + n), kind, page, seed=n)


@pytest.mark.parametrize("hd", range(16, 257, 16))
def test_every_width_and_turn(ctx, hd):
    for i, rot in enumerate(sorted({8, hd // 16 * 8, hd - 8, hd})):
        check(Rows(ctx, 2, 2, hd, 5, rot, bool(i % 2), i < 2, i > 1, i > 1, seed=rot), "f16", 16)


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
def test_strides_and_rows_without_a_place(ctx, kind):
    """Odd pitches, padded pages, rows that have no slot (their q is made all
    the same)."""
    check(Rows(ctx, 2, 3, 64, 70, 64, extra=3, seed=1), kind, 16, pad=2, q_pitch=6 * 64 + 5, skip=(40, 55, 69))


@pytest.mark.parametrize("n", [1, 63, 1030, 9000])
def test_many_rows(ctx, n):
    """Every split of rows and heads over workgroups."""
    check(Rows(ctx, 1, 2, 64, n, 64, seed=n), "rowi8", 64)
    check(Rows(ctx, 2, 8, 16, n, 16, True, False, True, True, seed=n), "f16", 16)


def test_far_positions(ctx):
    r = Rows(ctx, 1, 2, 64, 6, 64, seed=3)
    r.pos = np.array([0, 131071, 2 ** 30, -2 ** 30, -1, 999999937], np.int32)
    put(r.dpos, r.pos)
    check(r, "f32", 16)


@pytest.mark.parametrize("pairs", [False, True])
def test_in_place(ctx, pairs):
    """q into the fused rows themselves: keys' and values' columns stay."""
    for n in (1, 50, 700):
        r = Rows(ctx, 2, 3, 128, n, 64, pairs, extra=1, seed=n)
        slots = np.arange(n, dtype=np.int64) + 3
        p = Pool(ctx, "f16", n // 16 + 2, 16, 2, 128)
        q = r.call(p, slots)
        before = raw(p)
        p.c.append_dev(r.dx.ptr, r.heads, r.dpos.ptr, r.ds.ptr, n, r.dx.ptr, r.how, r.x.shape[1], r.x.shape[1])
        ctx.sync()
        x = r.dx.numpy()
        assert same(x[:, :r.heads * 128].reshape(q.shape), q) and same(x[:, r.heads * 128:], r.x[:, r.heads * 128:])
        assert all(np.array_equal(a, b) for a, b in zip(raw(p), before))


def test_slots_out_of_range_are_reported_and_skipped(ctx):
    r = Rows(ctx, 2, 2, 32, 5, 32, seed=4)
    p, ref = Pool(ctx, "f32", 2, 16, 2, 32), Pool(ctx, "f32", 2, 16, 2, 32)
    q = r.call(ref, [3, -1, 9, -1, 31])
    with pytest.raises(fa.FrqError) as e:
        r.call(p, [3, 32, 9, 2 ** 40, 31])
    assert e.value.code == fa.FRQ_ERR_ARG
    assert all(np.array_equal(a, b) for a, b in zip(raw(p), raw(ref)))
    assert same(r.dq.numpy()[:5].reshape(q.shape), q)
    ctx.sync()  # told once


def test_no_rows(ctx):
    r = Rows(ctx, 1, 1, 16, 1, 16)
    p = Pool(ctx, "f16", 1, 16, 1, 16)
    p.c.append_dev(None, 1, None, None, 0, None, r.how)
    ctx.sync()


def test_what_is_not_finite_stays_in_its_head(ctx):
    for pairs in (False, True):
        r = Rows(ctx, 2, 2, 64, 4, 32, pairs, seed=6, qn=True, kn=True)
        clean = r.call(Pool(ctx, "f32", 1, 16, 2, 64), [0, 1, 2, 3])
        r.x[1, 5], r.x[2, 64 + 40], r.x[3, 3 * 64 + 1] = np.nan, np.inf, 3e38
        put(r.dx, r.x)
        p = Pool(ctx, "f32", 1, 16, 2, 64)
        q = r.call(p, [0, 1, 2, 3])
        touched = np.zeros((4, 4), bool)
        touched[1, 0] = touched[2, 1] = touched[3, 3] = True
        assert same(q[~touched], clean[~touched])
        assert np.isnan(q[1, 0]).all()  # the norm takes it to all of the head
        assert np.isfinite(q[3, 3]).all()  # whose square 64 bits hold


def test_captured_and_replayed(ctx):
    """In a graph, over changing rows, positions and slots, with eager calls
    and synchronizations between, on a caller's stream too."""
    r = Rows(ctx, 2, 3, 64, 9, 64, qn=True, kn=True, seed=8)
    p = Pool(ctx, "rowi8", 4, 16, 2, 64)
    r.call(p, np.arange(9))
    step = lambda: p.c.append_dev(r.dx.ptr, r.heads, r.dpos.ptr, r.ds.ptr, 9, r.dq.ptr, r.how)  # noqa: E731
    graph = Graph(ctx, step)
    rng = np.random.default_rng(1)
    for i in range(4):
        r.x = rng.standard_normal(r.x.shape).astype(np.float32)
        r.pos = rng.integers(0, 4000, 9).astype(np.int32)
        put(r.dx, r.x)
        put(r.dpos, r.pos)
        put(r.ds, rng.permutation(64)[:9].astype(np.int64))
        outs = []
        for how in (graph.replay, step, graph.replay):
            put(r.dq, np.zeros(r.dq.shape, np.float32))
            how()
            ctx.sync()
            outs.append([r.dq.numpy().view(np.uint8)] + raw(p))
        for o in outs[1:]:
            assert all(np.array_equal(a, b) for a, b in zip(o, outs[0]))
        want, size = r.want()
        check_rows(r.dq.numpy()[:9].reshape(9, r.heads, 64), want[:, :r.heads], size[:, :r.heads])
    graph.close()


def test_slots_beyond_32_bits(ctx):
    """A pool of over 2^32 bytes a matrix: rows into its last pages."""
    free, _ = hip.mem_info()
    page, kv, hd, n_pages = 1024, 1, 256, 4200  # 4200 * 1024 * 256 * 4 B = 4.4 GB
    if free < 3 * n_pages * page * kv * hd * 4:
        pytest.skip("needs 13 GB")
    k, v = hip.DeviceArray((n_pages * page * kv * hd,), np.float32), hip.DeviceArray((n_pages * page * kv * hd,), np.float32)
    c = fa.KvCache(ctx, "f32", n_pages, page, kv, hd, k.ptr, v.ptr)
    r = Rows(ctx, kv, 2, hd, 40, hd, seed=9)
    slots = np.arange(40, dtype=np.int64) + n_pages * page - 45
    ds, dq = up(slots), hip.DeviceArray((40, 2 * hd), np.float32)
    ok, ov = hip.DeviceArray((40, kv, hd), np.float32), hip.DeviceArray((40, kv, hd), np.float32)
    c.append_dev(r.dx.ptr, 2, r.dpos.ptr, ds.ptr, 40, dq.ptr, r.how)
    c.read_dev(ds.ptr, 40, ok.ptr, ov.ptr)
    ctx.sync()
    want, size = r.want()
    check_rows(ok.numpy(), want[:, 2:3], size[:, 2:3])
    check_rows(ov.numpy(), want[:, 3:], 0 * size[:, 3:])


def test_another_stream_and_two_contexts_at_once(ctx):
    r = Rows(ctx, 2, 3, 64, 70, 64, qn=True, seed=11)
    p, slots = Pool(ctx, "rowi8", 6, 16, 2, 64), np.arange(70)
    q, pages = r.call(p, slots), raw(p)
    other = fa.Context(0)
    s = Rows(other, 2, 3, 64, 70, 64, qn=True, seed=11)
    o = Pool(other, "rowi8", 6, 16, 2, 64)
    stream = C.c_void_p()
    hip._chk(hip._hip.hipStreamCreate(C.byref(stream)), "hipStreamCreate")
    try:
        other.set_stream(stream.value)
        assert same(s.call(o, slots), q)
        for _ in range(10):
            for x, c in ((r, p), (s, o)):
                c.c.append_dev(x.dx.ptr, x.heads, x.dpos.ptr, x.ds.ptr, 70, x.dq.ptr, x.how)
        ctx.sync()
        other.sync()
        for x, c in ((r, p), (s, o)):
            assert same(x.dq.numpy()[:70].reshape(q.shape), q)
            assert all(np.array_equal(a, b) for a, b in zip(raw(c), pages))
    finally:
        other.sync()
        other.set_stream(None)
        hip._chk(hip._hip.hipStreamDestroy(stream), "hipStreamDestroy")
        other.close()
