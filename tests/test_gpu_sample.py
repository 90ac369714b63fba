"""frq_sample_dev on the device against the definition in numpy's 64 bits, token
for token.

Weights are whole numbers of 2^-s of a largest one between 1/2 and 1 (s = 62 -
log2 n, up to 50), and none below half a step.  So a cut or a draw could only
come out differently where a sum lies within the two sides' roundings of its
bound: n 2^-s of the largest weight here, n 2^-53 there; the inputs are fixed.
Sums of equal weights are exact on both sides, so that ties are cut alike.  The
share is rounded to f32 once, 2^-24 of itself (or half of the smallest number),
and holds half a step of its own weight and n of them in the sum, which is 1/2
or more: 2^-s (1 + n share)."""
import ctypes as C

import numpy as np
import pytest

import fieldrun_amd as fa
from fieldrun_amd import hip
from test_gpu_kv import Graph, put, same

pytestmark = pytest.mark.gpu
up = hip.DeviceArray.from_numpy


def bits(n):
    return min(50, 62 - (n - 1).bit_length())


def choose(x, temp=1.0, k=0, p=1.0, mp=0.0, u=0.5):
    """(token, share) of one row."""
    x = x.astype(np.float64)
    if temp == 0:
        return int(np.argmax(x)), 1.0
    n = len(x)
    temp = np.float64(np.float32(temp))
    w = np.exp((x - x.max()) / temp)
    lead = x.max() / temp * np.log2(np.e)
    w[w < 2.0 ** (-bits(n) - 1) * 2.0 ** min(1, np.ceil(lead) - lead)] = 0
    by = np.argsort(-x, kind="stable")
    if 0 < k < n:
        by = by[:k]
    s = np.cumsum(w[by])
    p = float(np.float32(p))
    if p < 1:
        before = np.concatenate([[0.0], s[:-1]])
        by = by[(before < p * s[-1]) | (np.arange(len(by)) == 0)]
    by = np.sort(by[w[by] >= float(np.float32(mp))])
    s = np.cumsum(w[by])
    i = int((s <= min(max(float(u), 0.0), 1 - 2.0 ** -24) * s[-1]).sum())
    t = by[i]
    return int(t), float(w[t] / s[-1])


class Call:
    def __init__(self, ctx, x, temp=None, k=None, p=None, mp=None, u=0.5, pad=0, own_ws=True):
        self.ctx, (self.m, self.n) = ctx, x.shape
        self.x, self.pitch = x, self.n + pad
        wide = np.full((self.m, self.pitch), np.nan, np.float32)
        wide[:, :self.n] = x
        row = lambda v, t: None if v is None else np.broadcast_to(np.asarray(v, t), (self.m,)).copy()  # noqa: E731
        self.par = {"temp": row(temp, np.float32), "topk": row(k, np.int32), "topp": row(p, np.float32),
                    "minp": row(mp, np.float32)}
        self.u = row(u, np.float32)
        self.dx, self.du = up(wide), up(self.u)
        self.dpar = {a: None if v is None else up(v) for a, v in self.par.items()}
        self.token = up(np.full(self.m + 2, 77, np.int64))
        self.prob = up(np.full(self.m + 2, 7.0, np.float32))
        need = ctx.sample_ws_bytes(self.m, self.n)
        assert need > 0
        self.ws = up(np.full(need, 0xFF, np.uint8)) if own_ws else None

    def __call__(self):
        self.ctx.sample_dev(self.dx.ptr, self.m, self.n, self.du.ptr, self.token.ptr,
                            **{a + "_ptr": d and d.ptr for a, d in self.dpar.items()}, prob_ptr=self.prob.ptr,
                            pitch=self.pitch, ws_ptr=self.ws and self.ws.ptr, ws_bytes=self.ws.nbytes if self.ws else 0)

    def run(self):
        self()
        self.ctx.sync()
        t, p = self.token.numpy(), self.prob.numpy()
        assert (t[self.m:] == 77).all() and (p[self.m:] == 7.0).all()
        return t[:self.m], p[:self.m]

    def want(self):
        g = lambda a, r, d: d if self.par[a] is None else self.par[a][r]  # noqa: E731
        return [choose(self.x[r], g("temp", r, 1.0), int(g("topk", r, 0)), g("topp", r, 1.0), g("minp", r, 0.0), self.u[r])
                for r in range(self.m)]

    def check(self):
        t, p = self.run()
        want = self.want()
        off = [(r, t[r], w[0]) for r, w in enumerate(want) if t[r] != w[0]]
        assert not off, off[:5]
        share = np.array([w[1] for w in want])
        tol = 2.0 ** -24 * share * (1 + 2.0 ** -20) + 2.0 ** -bits(self.n) * (1 + self.n * share) + 2.0 ** -150
        assert (np.abs(p - share) <= tol).all(), (np.abs(p - share) / tol).max()
        return t, p


def rows(rng, m, n, kind):
    if kind == "peaked":  # shares fall with a power of the rank
        x = -rng.uniform(1, 3, (m, 1)) * np.log(1 + np.argsort(rng.random((m, n)), 1)) + 0.3 * rng.standard_normal((m, n)) + 18
    elif kind == "flat":
        x = 2.5 * rng.standard_normal((m, n))
    elif kind == "tied":  # few different values
        x = np.round(2 * rng.standard_normal((m, n)))
    elif kind == "equal":
        x = np.full((m, n), -3.25)
    elif kind == "masked":  # of all but some the probability is zero
        x = np.where(rng.random((m, n)) < 0.9, -np.inf, 3 * rng.standard_normal((m, n)))
        x[:, n // 2] = 1.0
    elif kind == "wide":
        x = rng.standard_normal((m, n)) * 10.0 ** rng.uniform(-3, 4, (m, 1)) * rng.choice([-1, 1], (m, 1))
    return x.astype(np.float32)


KINDS = ["peaked", "flat", "tied", "equal", "masked", "wide"]
MODES = [dict(), dict(k=40), dict(p=0.9), dict(mp=0.05), dict(k=200, p=0.95), dict(k=50, p=0.8, mp=0.02), dict(p=0.999, mp=1e-4),
         dict(temp=0.0), dict(k=1), dict(p=0.0), dict(mp=1.0)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n", [(1, 1), (3, 2), (5, 31), (4, 257), (7, 1000), (2, 2049), (9, 5003), (3, 20011), (2, 152064)])
def test_tokens(ctx, kind, m, n):
    rng = np.random.default_rng(n + len(kind))
    x = rows(rng, m, n, kind)
    for i, mode in enumerate(MODES):
        how = dict(mode)
        how.setdefault("temp", [0.7, 1.0, 1.3][i % 3])
        Call(ctx, x, u=rng.random(m), pad=i % 3, **how).check()


@pytest.mark.parametrize("n", [511, 512, 513, 2047, 2048, 4096, 8191, 8192, 8193, 16385])
def test_widths_about_the_kernels_own(ctx, n):
    """Rows that fit a launch and rows one longer, with and without room for all
    of them in order, as few and many, also those that miss every alignment."""
    for i, kind in enumerate(KINDS):
        rng = np.random.default_rng(n + i)
        m = [2, 5, 33][i % 3]
        for mode in MODES[i % 2::2]:
            Call(ctx, rows(rng, m, n, kind), u=rng.random(m), pad=1 + 2 * (i % 2), **mode).check()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_their_own_parameters(ctx, kind):
    """Rows of every mode in one call, and each alone: the same bits, however
    the rows are cut."""
    rng = np.random.default_rng(7)
    m, n = 40, 9001
    modes = [MODES[i % len(MODES)] for i in range(m)]
    how = dict(temp=[d.get("temp", rng.uniform(0.3, 2)) for d in modes], k=[d.get("k", 0) for d in modes],
               p=[d.get("p", 1.0) for d in modes], mp=[d.get("mp", 0.0) for d in modes], u=rng.random(m))
    x = rows(rng, m, n, kind)
    t, p = Call(ctx, x, **how).check()
    for r in (0, 5, 11, 39):
        one = Call(ctx, x[r:r + 1], **{a: [v[r]] for a, v in how.items()})
        t1, p1 = one.run()
        assert t1[0] == t[r] and same(p1, p[r:r + 1])
    many = np.concatenate([x] * 30)  # 1200 rows: a workgroup a row
    tm, pm = Call(ctx, many, **{a: np.tile(np.asarray(v, np.float64), 30) for a, v in how.items()}).run()
    assert np.array_equal(tm, np.tile(t, 30)) and same(pm, np.tile(p, 30))


def test_large_sets(ctx):
    """Cuts in bins of more elements than the list holds: many equal values,
    all the same weight, and dense ones, with both bounds falling there."""
    rng = np.random.default_rng(3)
    for n in (5003, 152064):
        x = np.concatenate([rows(rng, 2, n, "equal"), rows(rng, 2, n, "tied"),
                            (1e-3 * rng.standard_normal((2, n))).astype(np.float32)])
        for k in (0, 3000, n - 1, n // 2):
            for p in (1.0, 0.5, 0.9, 1e-6):
                Call(ctx, x, k=k, p=p, temp=[0.5, 1, 2, 0.1, 1, 3], u=rng.random(6)).check()


@pytest.mark.parametrize("n", [100, 50257])
def test_numbers_at_their_ends(ctx, n):
    rng = np.random.default_rng(n)
    x = np.repeat(rows(rng, 1, n, "peaked"), 8, 0)
    u = np.array([0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, 2.0 ** -149, 0.5, np.inf], np.float32)
    for mode in (dict(), dict(k=9), dict(p=0.7), dict(mp=0.1)):
        t, _ = Call(ctx, x, u=u, **mode).check()
        assert t[0] == t[4] == t[5] and t[1] == t[2] == t[3] == t[7]


def test_tokens_rise_with_the_number(ctx):
    """Inverse sampling: the tokens of a row over rising numbers rise, and their
    shares are how often each comes."""
    rng = np.random.default_rng(2)
    m, n = 1000, 300
    x = np.repeat(rows(rng, 1, n, "flat"), m, 0)
    t, p = Call(ctx, x, u=(np.arange(m) + 0.5) / m, p=0.9).check()
    assert (np.diff(t) >= 0).all()
    for v in np.unique(t):
        assert abs((t == v).mean() - p[t == v][0]) <= 1.0 / m + 1e-6


@pytest.mark.parametrize("temp", [1e-30, 1e-6, 1e-2, 50.0, 1e6, 1e30])
def test_temperatures(ctx, temp):
    rng = np.random.default_rng(4)
    for kind in ("peaked", "flat", "tied", "masked"):
        x = rows(rng, 6, 3001, kind)
        for mode in (dict(), dict(k=30), dict(p=0.9), dict(k=100, p=0.5, mp=0.01)):
            Call(ctx, x, temp=temp, u=rng.random(6), **mode).check()


def test_logits_of_any_size(ctx):
    rng = np.random.default_rng(5)
    for scale in (1e-38, 1e-20, 1e10, 1e30, 3e38):
        x = (rng.uniform(-1, 1, (4, 2000)) * scale).astype(np.float32)
        x[1, 7] = -x[1].min()
        x[2] = np.float32(scale)
        x[3, ::2], x[3, 1::2] = 0.0, -0.0  # equal
        for mode in (dict(), dict(k=30), dict(p=0.5)):
            Call(ctx, x, u=rng.random(4), **mode).check()


def test_rows_without_a_token(ctx):
    """NaN, an infinite maximum, nothing but -inf: -1 and an error, the other
    rows as ever; told once."""
    rng = np.random.default_rng(6)
    x = rows(rng, 8, 5003, "flat")
    good = Call(ctx, x, p=0.9, u=0.3).check()
    x[1, 4000], x[3], x[5, 17], x[6, 3] = np.nan, -np.inf, np.inf, np.nan
    c = Call(ctx, x, p=0.9, u=0.3, temp=[1, 1, 1, 1, 1, 1, 0, 1])
    c()
    with pytest.raises(fa.FrqError) as e:
        ctx.sync()
    assert e.value.code == fa.FRQ_ERR_NAN
    ctx.sync()
    t, p = c.token.numpy()[:8], c.prob.numpy()[:8]
    bad = np.isin(np.arange(8), [1, 3, 5, 6])
    assert (t[bad] == -1).all() and (p[bad] == 0).all()
    assert np.array_equal(t[~bad], good[0][~bad]) and same(p[~bad], good[1][~bad])


def test_parameters_that_are_none(ctx):
    rng = np.random.default_rng(8)
    x = rows(rng, 7, 300, "flat")
    good = Call(ctx, x, k=20, temp=1.0, p=0.9, mp=0.01, u=0.3).check()
    nan = np.nan
    c = Call(ctx, x, k=20, temp=[1, -1, np.inf, nan, 1, 1, 1], p=[0.9] * 4 + [nan, 0.9, 0.9], mp=[0.01] * 5 + [nan, 0.01],
             u=[0.3] * 6 + [nan])
    c()
    with pytest.raises(fa.FrqError) as e:
        ctx.sync()
    assert e.value.code == fa.FRQ_ERR_ARG and "sampling" in str(e.value)
    ctx.sync()
    assert c.token.numpy()[:7].tolist() == [good[0][0]] + [-1] * 6
    # out of the range of a bound: no bound, or the first alone
    t, _ = Call(ctx, x, k=-5, p=7.0, mp=-1.0, u=0.3).run()
    assert np.array_equal(t, Call(ctx, x, u=0.3).check()[0])
    t, _ = Call(ctx, x, p=-3.0, mp=9.0, u=0.3).run()
    assert np.array_equal(t, x.argmax(1))


def test_repeat_strides_and_no_shares(ctx):
    rng = np.random.default_rng(9)
    x = rows(rng, 33, 4099, "peaked")
    u = rng.random(33)
    c = Call(ctx, x, k=100, p=0.9, u=u, pad=5)
    t, p = c.check()
    for other in (c, Call(ctx, x, k=100, p=0.9, u=u), Call(ctx, x, k=100, p=0.9, u=u, own_ws=False)):
        a, b = other.run()
        assert np.array_equal(a, t) and same(b, p)
    ctx.sample_dev(c.dx.ptr, 33, 4099, c.du.ptr, c.token.ptr, topk_ptr=c.dpar["topk"].ptr, topp_ptr=c.dpar["topp"].ptr,
                   pitch=c.pitch)
    ctx.sync()
    assert np.array_equal(c.token.numpy()[:33], t)
    ctx.sample_dev(None, 0, 5, None, None)  # no rows
    with pytest.raises(fa.FrqError) as e:
        ctx.sample_dev(c.dx.ptr, 33, 4099, c.du.ptr, c.token.ptr, pitch=c.pitch, ws_ptr=c.ws.ptr, ws_bytes=c.ws.nbytes - 256)
    assert e.value.code == fa.FRQ_ERR_ARG and "workspace" in str(e.value)


def test_captured_and_replayed(ctx):
    """In a graph, over changing logits, parameters and numbers, with eager
    calls and synchronizations between; without a workspace it is refused."""
    rng = np.random.default_rng(10)
    x = rows(rng, 5, 9001, "peaked")
    c = Call(ctx, x, temp=1.0, k=50, p=0.9, mp=0.0, u=0.5)
    c.check()

    def step():
        with pytest.raises(fa.FrqError) as e:
            ctx.sample_dev(c.dx.ptr, 5, 9001, c.du.ptr, c.token.ptr)
        assert "capture" in str(e.value)
        c()

    graph, last = Graph(ctx, step), None
    for i in range(5):
        c.x = rows(rng, 5, 9001, KINDS[i])
        c.u = rng.random(5).astype(np.float32)
        c.par["temp"] = rng.choice([0.0, 0.5, 1.0], 5).astype(np.float32)
        c.par["topk"] = rng.choice([0, 7, 3000], 5).astype(np.int32)
        put(c.dx, c.x)
        put(c.du, c.u)
        for a in ("temp", "topk"):
            put(c.dpar[a], c.par[a])
        outs = []
        for how in (graph.replay, c, graph.replay, graph.replay):
            put(c.token, np.full(7, 77, np.int64))
            how()
            ctx.sync()
            outs.append(c.token.numpy())
        assert all(np.array_equal(o, outs[0]) for o in outs[1:])
        assert outs[0][:5].tolist() == [w[0] for w in c.want()]
        assert last is None or not np.array_equal(outs[0], last)
        last = outs[0]
    graph.close()


def test_another_stream_and_two_contexts_at_once(ctx):
    rng = np.random.default_rng(11)
    x = rows(rng, 20, 30011, "flat")
    c = Call(ctx, x, p=0.9, u=rng.random(20))
    t, p = c.check()
    other = fa.Context(0)
    d = Call(other, x[::-1].copy(), p=0.9, u=c.u[::-1].copy())
    ctx.sync()
    for _ in range(10):
        c()
        d()
    ctx.sync()
    other.sync()
    assert np.array_equal(c.token.numpy()[:20], t) and np.array_equal(d.token.numpy()[:20], t[::-1])
    s = C.c_void_p()
    hip._chk(hip._hip.hipStreamCreate(C.byref(s)), "hipStreamCreate")
    try:
        other.set_stream(s.value)
        assert np.array_equal(d.run()[0], t[::-1])
    finally:
        other.sync()
        other.set_stream(None)
        hip._chk(hip._hip.hipStreamDestroy(s), "hipStreamDestroy")
        other.close()


def test_the_widest_rows(ctx):
    rng = np.random.default_rng(12)
    n = 1 << 24
    x = (2 * rng.standard_normal((1, n))).astype(np.float32)
    for mode in (dict(p=0.9), dict(k=100), dict(mp=0.01), dict(temp=0.0)):
        Call(ctx, x, u=0.6, **mode).check()


@pytest.mark.parametrize("n", [3001, 20011, 40009])
@pytest.mark.parametrize("temp", [1e-45, 1e-30, 1e-3, 0.1, 40.0, 1e6, 3e38])
def test_temperatures_over_several_chunks(ctx, n, temp):
    rng = np.random.default_rng(n)
    for kind in KINDS:
        x = rows(rng, 4, n, kind)
        for mode in (dict(), dict(k=30), dict(p=0.9), dict(k=5000, p=0.99), dict(k=100, p=0.5, mp=0.01)):
            Call(ctx, x, temp=temp, u=rng.random(4), **mode).check()


@pytest.mark.parametrize("n", [2000, 20011])
def test_logits_of_any_size_over_several_chunks(ctx, n):
    rng = np.random.default_rng(15)
    for scale in (1e-44, 1e-38, 1e-20, 1e10, 1e30, 3e38):
        x = (rng.uniform(-1, 1, (5, n)) * scale).astype(np.float32)
        x[1, n - 7] = -x[1].min()
        x[2] = np.float32(scale)
        x[3, ::2], x[3, 1::2] = 0.0, -0.0  # equal
        x[4] = np.float32(-scale)
        x[4, n - 1] = np.float32(-scale / 2)
        for mode in (dict(), dict(k=30), dict(p=0.5), dict(k=3000, p=0.9), dict(mp=0.5)):
            Call(ctx, x, u=rng.random(5), **mode).check()


@pytest.mark.parametrize("n", [8192, 70001])
def test_chunks_far_below_the_row(ctx, n):
    """Chunks of -inf alone, of the type's lowest value, of weights that are none,
    and one element that stands above all others, in the first chunk or the last."""
    rng = np.random.default_rng(16)
    x = rows(rng, 8, n, "flat")
    x[0, :n // 2] = -np.inf
    x[1, n // 3:] = -np.inf
    x[2, 5000:] = np.finfo(np.float32).min
    x[3, :n - 9] -= 1000
    x[4, 11:] -= 30
    x[5, n - 1] = 200
    x[6, 0] = 40
    x[7] = -np.inf
    x[7, [0, n // 2, n - 1]] = [-3, -2, -3]
    for mode in MODES:
        Call(ctx, x, u=rng.random(8), pad=1, **mode).check()


@pytest.mark.parametrize("n", [900, 50021])
def test_rows_and_parameters_that_are_none(ctx, n):
    """As above in a row of one launch and of several chunks, beside good ones."""
    rng = np.random.default_rng(17)
    x = rows(rng, 9, n, "peaked")
    how = dict(k=40, p=0.9, mp=0.001, u=rng.random(9))
    good = Call(ctx, x, **how).check()
    y, nan = x.copy(), np.nan
    y[1, n - 1], y[2, 0], y[3, n // 2], y[4] = nan, np.inf, nan, -np.inf
    bad = np.arange(9) >= 1
    bad[[5, 8]] = False
    c = Call(ctx, y, temp=[1, 1, 1, 0, 1, 1, -0.5, nan, 1], **how)
    c()
    with pytest.raises(fa.FrqError) as e:
        ctx.sync()
    assert e.value.code == fa.FRQ_ERR_NAN  # of both the NaN first
    with pytest.raises(fa.FrqError) as e:
        ctx.sync()
    assert e.value.code == fa.FRQ_ERR_ARG
    ctx.sync()
    t, p = c.token.numpy()[:9], c.prob.numpy()[:9]
    assert (t[bad] == -1).all() and (p[bad] == 0).all()
    assert np.array_equal(t[~bad], good[0][~bad]) and same(p[~bad], good[1][~bad])


def test_short_rows_captured_and_replayed(ctx):
    rng = np.random.default_rng(18)
    c = Call(ctx, rows(rng, 7, 2000, "peaked"), temp=1.0, k=50, p=0.9, u=0.5)
    c.check()
    graph = Graph(ctx, c)
    for i in range(5):
        c.x, c.u = rows(rng, 7, 2000, KINDS[i]), rng.random(7).astype(np.float32)
        put(c.dx, c.x)
        put(c.du, c.u)
        for how in (graph.replay, c, graph.replay):
            put(c.token, np.full(9, 77, np.int64))
            how()
            ctx.sync()
            assert c.token.numpy()[:7].tolist() == [w[0] for w in c.want()]
    graph.close()
