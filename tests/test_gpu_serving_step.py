"""The operators of a serving step together, as a program runs them on device
pointers: residual + norm + int8 rows (frq_norm_quant_i8_dev), the q|k|v int8
linear on those rows (frq_mm_i8_q_dev), the new tokens' keys and values from
the fused rows into the paged cache (frq_kv_write_dev), attention with q from
the same rows (frq_kv_attn_dev), the output linear (frq_mm_dev), into the next
layer's residual.  Three sequences: their prompts in one ragged call, then
steps in which a sequence ends and its pages go to a new one whose prompt runs
beside the others' decode rows.  Every operator's output is checked on the
inputs it was given: sums and int8 rows exact, linears against Weight.mm,
attention against the definition in 64 bits (its tolerance as derived in
test_gpu_kv.py)."""
import numpy as np
import pytest

from fieldrun_amd import hip, quant_pitch, synth
from test_gpu_kv import Pool, put
from test_gpu_norm_quant import norm, quantise

pytestmark = pytest.mark.gpu
D, KV, REP, HD, PAGE, PAGES, TABLE, LAYERS, EPS = 256, 2, 3, 64, 16, 24, 8, 2, 1e-6
HEADS, WIDE = KV * REP, (KV * REP + 2 * KV) * HD


class Layer:
    def __init__(self, ctx, kind, seed):
        rng = np.random.default_rng(seed)
        self.w = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
        self.dw = hip.DeviceArray.from_numpy(self.w)
        self.qkv = ctx.upload_i8(*synth.int8_weight(WIDE, D, seed))
        self.o = ctx.upload_i8(*synth.int8_weight(D, HEADS * HD, seed + 1))
        self.pool = Pool(ctx, kind, PAGES, PAGE, KV, HD, seed)
        self.k, self.v = {}, {}  # sequence -> rows, as stored


def attend(q, k, v, kind):
    """(outputs, tolerances) of one row (heads, hd) over all of k, v."""
    u, out, tol = 2.0 ** -24, np.zeros((HEADS, HD)), np.zeros((HEADS, HD))
    for h in range(HEADS):
        kh, vh, qh = (x.astype(np.float64) for x in (k[:, h // REP], v[:, h // REP], q[h]))
        z = HD ** -0.5 * (kh @ qh)
        d = u * (4 * HD ** 0.5 + 8) * HD ** -0.5 * (np.abs(kh) @ np.abs(qh)).max()
        if kind != "f32":
            d += 2.0 ** -22 * HD ** -0.5 * np.abs(qh).max() * np.abs(kh).sum(1).max()
        w = np.exp(z - z.max())
        w /= w.sum()
        out[h] = w @ vh
        tol[h] = (np.expm1(2 * d) + 2.0 ** -21 + u * (len(z) / 16 + 16)) * (w @ np.abs(vh))
        tol[h] += 2.0 ** (-126 if kind == "f32" else -35) * w.max() * len(z) * np.abs(vh).max()
    return out, tol


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
def test_serving_steps(ctx, kind):
    rng = np.random.default_rng(8)
    layers = [Layer(ctx, kind, 50 + i) for i in range(LAYERS)]
    free = list(rng.permutation(PAGES))
    seqs = {}  # name -> [length, pages]

    def step(asks):
        """asks: {sequence: new tokens}; one call of every operator a layer."""
        slots, table, lens, first = [], np.full((len(asks), TABLE), -1, np.int32), [], [0]
        for i, (s, r) in enumerate(asks.items()):
            n, pages = seqs.setdefault(s, [0, []])
            while len(pages) * PAGE < n + r:
                pages.append(free.pop())
            slots += [pages[j // PAGE] * PAGE + j % PAGE for j in range(n, n + r)]
            seqs[s][0] = n + r
            table[i, :len(pages)] = pages
            lens.append(n + r)
            first.append(first[-1] + r)
        m = first[-1]
        up = hip.DeviceArray.from_numpy
        x = up(rng.standard_normal((m, D)).astype(np.float32))
        y = up(np.zeros((m, D), np.float32))
        slot, tab, ln, fi = (up(np.asarray(a, t)) for a, t in ((slots, np.int64), (table, np.int32),
                                                               (lens, np.int32), (first, np.int32)))
        kp = quant_pitch(D)
        a8, sa = hip.DeviceArray((m, kp), np.int8), hip.DeviceArray((m,), np.float32)
        oi, ov = hip.DeviceArray((m, 32), np.uint32), hip.DeviceArray((m, 32), np.float32)
        decode = first[-1] == len(asks)
        for l in layers:
            before, res = x.numpy(), y.numpy()
            fused, att = hip.DeviceArray((m, WIDE), np.float32), hip.DeviceArray((m, HEADS * HD), np.float32)
            out = hip.DeviceArray((m, D), np.float32)
            ctx.norm_quant_dev(x.ptr, y.ptr, l.dw.ptr, EPS, m, D, x.ptr, a8.ptr, sa.ptr, oi.ptr, ov.ptr)
            l.qkv.mm_q_dev(a8.ptr, sa.ptr, oi.ptr, ov.ptr, m, fused.ptr)
            l.pool.c.write_dev(fused.ptr + 4 * HEADS * HD, fused.ptr + 4 * (HEADS + KV) * HD, slot.ptr, m, WIDE)
            l.pool.c.attn_dev(fused.ptr, m, HEADS, tab.ptr, TABLE, ln.ptr, len(asks), att.ptr,
                              first_ptr=None if decode else fi.ptr, q_pitch=WIDE)
            l.o.mm_dev(att.ptr, m, out.ptr)
            ctx.sync()
            # each on the inputs it was given
            total = x.numpy()
            assert np.array_equal(total, before + res)
            n = norm(total, l.w, EPS)
            for got, want in zip((a8.numpy(), sa.numpy(), oi.numpy(), ov.numpy()), quantise(ctx, n)):
                assert np.array_equal(got, want)
            f = fused.numpy()
            want = l.qkv.mm(n)
            assert np.array_equal(f, want) if m <= 16 else np.abs(f - want).max() <= 1e-5 * np.abs(want).max()
            q, k, v = (f[:, a:b].reshape(m, -1, HD) for a, b in ((0, HEADS * HD), (HEADS * HD, (HEADS + KV) * HD),
                                                                  ((HEADS + KV) * HD, WIDE)))
            for i, (s, r) in enumerate(asks.items()):
                a, b = first[i], first[i + 1]
                old = lens[i] - r
                l.k[s] = np.concatenate([l.k[s], l.pool.stored(k[a:b])]) if old else l.pool.stored(k[a:b])
                l.v[s] = np.concatenate([l.v[s], l.pool.stored(v[a:b])]) if old else l.pool.stored(v[a:b])
                for j in range(r):
                    o, tol = attend(q[a + j], l.k[s][:old + j + 1], l.v[s][:old + j + 1], kind)
                    assert (np.abs(att.numpy()[a + j].reshape(HEADS, HD) - o) <= tol).all(), (s, j)
            want = l.o.mm(att.numpy())
            got = out.numpy()
            assert np.array_equal(got, want) if m <= 16 else np.abs(got - want).max() <= 1e-5 * np.abs(want).max()
            put(y, got)

    step({"a": 37, "b": 1, "c": 18})
    for _ in range(3):
        step({"a": 1, "b": 1, "c": 1})
    free.extend(seqs.pop("b")[1])  # ends; its pages are used again, whatever they hold
    step({"a": 1, "d": 45, "c": 1})
    step({"c": 1, "d": 1, "a": 1})
    got = layers[0].pool.read([seqs["d"][1][j // PAGE] * PAGE + j % PAGE for j in range(46)])
    assert np.array_equal(got[0], layers[0].k["d"]) and np.array_equal(got[1], layers[0].v["d"])
