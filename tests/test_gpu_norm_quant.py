"""frq_norm_quant_i8_dev: residual, RMS norm and the int8 rows of the next
linear in one call.  The sum is exact; n is the 64-bit norm rounded once
(an order of the 64-bit sum moves it by 2^-50 or so, so it lands on the same
f32); the int8 rows, steps and outliers are frq_quant_i8_dev's for n, byte for
byte.  A run through the next linear equals the two steps apart."""
import numpy as np
import pytest

import fieldrun_amd as fa
from fieldrun_amd import hip, synth

pytestmark = pytest.mark.gpu


def quantise(ctx, n):
    m, k = n.shape
    kp = fa.quant_pitch(k)
    d = hip.DeviceArray.from_numpy(n)
    a8, sa = hip.DeviceArray((m, kp), np.int8), hip.DeviceArray((m,), np.float32)
    oi, ov = hip.DeviceArray((m, 32), np.uint32), hip.DeviceArray((m, 32), np.float32)
    ctx.quant_dev(d.ptr, m, k, a8.ptr, sa.ptr, oi.ptr, ov.ptr)
    ctx.sync()
    return a8.numpy(), sa.numpy(), oi.numpy(), ov.numpy()


class Call:
    def __init__(self, ctx, x, y, w, eps=1e-6, alias=None, keep_sum=True, nan=False):
        m, k = x.shape
        self.dx, self.dw = hip.DeviceArray.from_numpy(x), hip.DeviceArray.from_numpy(w)
        self.dy = None if y is None else hip.DeviceArray.from_numpy(y)
        s = self.dx if alias == "x" else self.dy if alias == "y" else hip.DeviceArray.from_numpy(np.full((m, k), 7, np.float32))
        kp = fa.quant_pitch(k)
        self.a8, self.sa = hip.DeviceArray.from_numpy(np.full((m + 1, kp), 77, np.int8)), hip.DeviceArray((m,), np.float32)
        self.oi, self.ov = hip.DeviceArray((m, 32), np.uint32), hip.DeviceArray((m, 32), np.float32)
        ctx.norm_quant_dev(self.dx.ptr, self.dy and self.dy.ptr, self.dw.ptr, eps, m, k, s.ptr if keep_sum else None,
                           self.a8.ptr, self.sa.ptr, self.oi.ptr, self.ov.ptr)
        if nan:
            with pytest.raises(fa.FrqError) as e:
                ctx.sync()
            assert e.value.code == fa.FRQ_ERR_NAN
        else:
            ctx.sync()
        self.sum = s.numpy()
        a8 = self.a8.numpy()
        assert (a8[m] == 77).all()  # the row behind the last
        self.parts = a8[:m], self.sa.numpy(), self.oi.numpy(), self.ov.numpy()


def norm(s, w, eps):
    s = s.astype(np.float64)
    return (s * (1.0 / np.sqrt((s * s).sum(1, keepdims=True) / s.shape[1] + eps)) * w.astype(np.float64)).astype(np.float32)


def data(m, k, seed):
    rng = np.random.default_rng(seed)
    return (synth.activations(m, k, seed), rng.standard_normal((m, k)).astype(np.float32),
            (1 + 0.2 * rng.standard_normal(k)).astype(np.float32))


@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (2, 32), (5, 33), (1, 64), (13, 1027), (4, 1024), (2, 1025), (3, 2304),
                                 (1, 3584), (17, 4096), (2, 4099), (3, 8190), (2, 9216), (1, 18944), (2, 20481),
                                 (1, 28672)])
@pytest.mark.parametrize("residual", [True, False])
def test_matches_norm_then_quant(ctx, m, k, residual):
    x, y, w = data(m, k, m * 7 + k)
    s = (x + y).astype(np.float32) if residual else x
    c = Call(ctx, x, y if residual else None, w)
    assert np.array_equal(c.sum, s)
    for got, want in zip(c.parts, quantise(ctx, norm(s, w, 1e-6))):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("alias", ["x", "y"])
def test_sum_in_place(ctx, alias):
    x, y, w = data(5, 900, 3)
    a, b = Call(ctx, x, y, w, alias=alias), Call(ctx, x, y, w, keep_sum=False)
    assert np.array_equal(a.sum, x + y) and (b.sum == 7).all()
    for p, q in zip(a.parts, b.parts):
        assert np.array_equal(p, q)


def test_rows_with_equal_magnitudes(ctx):
    """Constant, alternating and zero rows (the selection's slow path, ties by
    the lowest channel), at widths with a tail past the last multiple of 4."""
    for k in (1027, 4096, 4097, 5000):
        w = np.ones(k, np.float32)
        x = np.ones((4, k), np.float32)
        x[1, ::2] = -1
        x[2] = 0.0
        x[3] = 0.0
        x[3, k - 3:] = 5.0
        c = Call(ctx, x, None, w)
        for got, want in zip(c.parts, quantise(ctx, norm(x, w, 1e-6))):
            assert np.array_equal(got, want)


def test_small_and_large_rows(ctx):
    x, y, w = data(6, 1500, 9)
    x *= np.array([1e-20, 1e-38, 1e15, 3e37, 1e-3, 1e30], np.float32)[:, None]
    y[:] = 0
    # row 3 overflows: activations reach 12 and 3e37 * 12 > 2^128, so the row
    # holds infinities, its norm inf / inf NaN, which is reported
    assert np.isinf(x[3]).any() and np.isfinite(np.delete(x, 3, 0)).all()
    c = Call(ctx, x, y, w, eps=0.0, nan=True)
    with np.errstate(invalid="ignore"):
        n = norm(x, w, 0.0)
    n[3] = 0.0
    for got, want in zip(c.parts, quantise(ctx, n)):
        assert np.array_equal(np.delete(got, 3, 0), np.delete(want, 3, 0))
    assert (c.parts[0][3] == 0).all() and c.parts[1][3] == 1.0  # the placeholders


def test_nan_rows_are_reported(ctx):
    for k in (40, 4096, 20000):
        x, y, w = data(3, k, 5)
        x[1, 7] = np.nan
        with pytest.raises(fa.FrqError) as e:
            Call(ctx, x, y, w)
        assert e.value.code == fa.FRQ_ERR_NAN
        ctx.sync()


@pytest.mark.parametrize("m", [1, 5, 40])
def test_feeds_the_int8_linear(ctx, m):
    """x, y -> norm -> int8 linear: mm_q_dev on the call's rows against mm_dev
    on the norm's f32 rows (the same sums: to the bit up to 16 rows, beyond
    that within the GEMM's bound of its correction)."""
    k, n = 896, 512
    x, y, w = data(m, k, 11)
    wt, scale = synth.int8_weight(n, k, 4)
    weight = ctx.upload_i8(wt, scale)
    c = Call(ctx, x, y, w)
    out = hip.DeviceArray((m, n), np.float32)
    weight.mm_q_dev(c.a8.ptr, c.sa.ptr, c.oi.ptr, c.ov.ptr, m, out.ptr)
    ctx.sync()
    want = weight.mm(norm(x + y, w, 1e-6))
    got = out.numpy()
    assert np.array_equal(got, want) if m <= 16 else np.abs(got - want).max() <= 1e-5 * np.abs(want).max()


@pytest.mark.parametrize("k", [1, 7, 32])
def test_nan_in_rows_of_outliers_alone(ctx, k):
    """Up to 32 channels nothing is selected: a NaN goes through as an outlier,
    unreported, as frq_quant_i8_dev hands it on."""
    x, y, w = data(3, k, 5)
    x[1, k // 2] = np.nan
    c = Call(ctx, x, None, w)
    with np.errstate(invalid="ignore"):
        want = quantise(ctx, norm(x, w, 1e-6))
    for got, exp in zip(c.parts, want):
        assert np.array_equal(got, exp, equal_nan=got.dtype.kind == "f")
    assert np.isnan(c.parts[3][1, :k]).all()
