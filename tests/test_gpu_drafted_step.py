"""The operators of an answer together, as a program runs them on device
pointers: residual + norm + int8 rows, the q|k|v int8 linear on them, those rows
made ready and appended in place (frq_kv_append_dev), attention with q from the
same rows over a window with sinks (frq_kv_attn_sink_dev) or, for drafted tokens,
over their trees (frq_kv_attn_tree_dev), the output linear, the logits, and a
token of each row by settings of its own (frq_sample_dev), whose embedding is the
next step's input.  Prompts, steps, a step of drafted trees, the rows of the
branch that was taken moved to the front, and a step after it.

Every operator's output is checked on the inputs it was given: appended rows
against the formulas in 64 bits (test_gpu_kv_append.py's tolerance, then half a
step of the cache's type), attention against the definition over the stored rows
(test_gpu_kv.py's), tokens by the definition on the logits, one by one."""
import numpy as np
import pytest

import fieldrun_amd as fa
from fieldrun_amd import hip, quant_pitch, synth
from test_gpu_kv import Graph, Pool, put, same
from test_gpu_kv_append import Rows, check_rows
from test_gpu_kv_sight import grow, words_of
from test_gpu_sample import choose
from test_gpu_serving_step import attend

pytestmark = pytest.mark.gpu
D, KV, REP, HD, PAGE, PAGES, TABLE, VOCAB, EPS = 256, 2, 3, 64, 16, 30, 10, 601, 1e-6
HEADS, WIDE, ROT = KV * REP, (KV * REP + 2 * KV) * HD, 48
WINDOW, SINKS = 30, 4
up = hip.DeviceArray.from_numpy


class Layer:
    def __init__(self, ctx, kind, seed, pairs):
        rng = np.random.default_rng(seed)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.w, self.bias, self.qn, self.kn = 1 + f(D) / 8, f(WIDE) / 4, 1 + f(HD) / 4, 1 + f(HD) / 4
        self.freq = 1e4 ** (-2.0 * np.arange(ROT // 2) / ROT)
        self.dev = [up(a) for a in (self.w, self.bias, self.qn, self.kn, self.freq)]
        p = [a.ptr for a in self.dev]
        self.pairs, self.how = pairs, fa.Rotary(ROT, p[4], pairs, p[1], p[2], p[3], EPS)
        self.qkv = ctx.upload_i8(*synth.int8_weight(WIDE, D, seed))
        self.o = ctx.upload_i8(*synth.int8_weight(D, HEADS * HD, seed + 1))
        self.pool = Pool(ctx, kind, PAGES, PAGE, KV, HD, seed)
        self.k, self.v = {}, {}  # sequence -> rows, as stored

    def ready(self, x, pos):
        """The fused rows x as they should be appended, and their terms' sizes."""
        r = Rows.__new__(Rows)
        r.x, r.wide, r.n, r.hd, r.heads, r.kv, r.rot, r.pos = x, WIDE, len(x), HD, HEADS, KV, ROT, np.asarray(pos, np.int32)
        r.bias, r.qn, r.kn, r.eps, r.freq, r.pairs = self.bias, self.qn, self.kn, EPS, self.freq, self.pairs
        return r.want()


def check_stored(got, want, size, kind):
    if kind == "f32":
        return check_rows(got, want, size)
    near = 2.0 ** -24 * np.abs(want) + 2.0 ** -48 * size  # before the cache's rounding
    if kind == "f16":
        tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 2 * near
    else:  # half of the row's step, the step's and the product's roundings
        tol = np.abs(want).max(-1, keepdims=True) / 127 * (0.5 + 2.0 ** -14) + 2 * near
    assert (np.abs(got - want) <= tol).all()


class Engine:
    def __init__(self, ctx, kind, seed=1):
        self.ctx, self.kind, self.rng = ctx, kind, np.random.default_rng(seed)
        self.layers = [Layer(ctx, kind, 70 + i, bool(i)) for i in range(2)]
        self.table = self.rng.standard_normal((VOCAB, D)).astype(np.float32)
        self.head = ctx.upload_rows("f32", self.table / 8)
        self.free, self.seqs = list(self.rng.permutation(PAGES)), {}  # name -> [length, pages]

    def slots(self, s, a, b):
        pages = self.seqs[s][1]
        return [int(pages[j // PAGE]) * PAGE + j % PAGE for j in range(a, b)]

    def step(self, asks, trees=None):
        """asks: {sequence: new tokens}; trees: {sequence: what each sees of
        them}.  Returns the sequences' sampled tokens, a row each."""
        ctx, kind = self.ctx, self.kind
        table, lens, first, slots, pos = np.full((len(asks), TABLE), -1, np.int32), [], [0], [], []
        for i, (s, new) in enumerate(asks.items()):
            n, pages = self.seqs.setdefault(s, [0, []])
            r = len(new)
            while len(pages) * PAGE < n + r:
                pages.append(self.free.pop())
            self.seqs[s][0] = n + r
            slots += self.slots(s, n, n + r)
            pos += [n + len(t) - 1 for t in trees[s]] if trees else list(range(n, n + r))
            table[i, :len(pages)] = pages
            lens.append(n + r)
            first.append(first[-1] + r)
        m = first[-1]
        x = up(self.table[np.concatenate(list(asks.values()))])
        y = up(np.zeros((m, D), np.float32))
        slot, tab, ln, fi, ps = (up(np.asarray(a, t)) for a, t in (
            (slots, np.int64), (table, np.int32), (lens, np.int32), (first, np.int32), (pos, np.int32)))
        masks = [trees[s] for s in asks] if trees else None
        tree = up(words_of(masks, 1, np.random.default_rng(3))) if trees else None
        kp = quant_pitch(D)
        a8, sa = hip.DeviceArray((m, kp), np.int8), hip.DeviceArray((m,), np.float32)
        oi, ov = hip.DeviceArray((m, 32), np.uint32), hip.DeviceArray((m, 32), np.float32)
        for l in self.layers:
            fused, att, out = (hip.DeviceArray((m, w), np.float32) for w in (WIDE, HEADS * HD, D))
            ctx.norm_quant_dev(x.ptr, y.ptr, l.dev[0].ptr, EPS, m, D, x.ptr, a8.ptr, sa.ptr, oi.ptr, ov.ptr)
            l.qkv.mm_q_dev(a8.ptr, sa.ptr, oi.ptr, ov.ptr, m, fused.ptr)
            ctx.sync()
            rows = fused.numpy()
            l.pool.c.append_dev(fused.ptr, HEADS, ps.ptr, slot.ptr, m, fused.ptr, l.how, q_pitch=WIDE)
            l.pool.c.attn_dev(fused.ptr, m, HEADS, tab.ptr, TABLE, ln.ptr, len(asks), att.ptr, first_ptr=fi.ptr,
                              q_pitch=WIDE, window=WINDOW, sinks=SINKS, tree_ptr=tree and tree.ptr)
            l.o.mm_dev(att.ptr, m, out.ptr)
            ctx.sync()
            # each on the inputs it was given
            want, size = l.ready(rows, pos)
            f = fused.numpy().reshape(m, -1, HD)
            check_rows(f[:, :HEADS], want[:, :HEADS], size[:, :HEADS])
            assert same(f[:, HEADS:], rows.reshape(m, -1, HD)[:, HEADS:])  # q's place alone was written
            k, v = l.pool.read(slots)
            check_stored(k, want[:, HEADS:HEADS + KV], size[:, HEADS:HEADS + KV], kind)
            check_stored(v, want[:, HEADS + KV:], size[:, HEADS + KV:], kind)
            got = att.numpy().reshape(m, HEADS, HD)
            for i, s in enumerate(asks):
                a, b = first[i], first[i + 1]
                old = lens[i] - (b - a)
                for mine, new in ((l.k, k), (l.v, v)):
                    mine[s] = np.concatenate([mine[s][:old], new[a:b]]) if old else new[a:b]
                for j in range(b - a):
                    p, own = (pos[a + j], [old + t for t in trees[s][j]]) if trees else (old + j, range(old, old + j + 1))
                    seen = [t for t in range(old) if p - t < WINDOW or t < SINKS]
                    seen = sorted(seen + [t for t in own if trees or p - t < WINDOW or t < SINKS])
                    o, tol = attend(f[a + j], l.k[s][seen], l.v[s][seen], kind)
                    assert (np.abs(got[a + j] - o) <= tol).all(), (s, j)
            put(y, out.numpy())
        ctx.norm_quant_dev(x.ptr, y.ptr, self.layers[0].dev[0].ptr, EPS, m, D, x.ptr, a8.ptr, sa.ptr, oi.ptr, ov.ptr)
        logits = up(np.full((m, VOCAB + 3), np.nan, np.float32))
        for r in range(m):
            self.head.rowdot_f32_dev(x.ptr + 4 * D * r, logits.ptr + 4 * (VOCAB + 3) * r)
        par = [self.rng.choice(c, m).astype(t) for c, t in (([0.0, 0.7, 1.0, 1.4], np.float32), ([0, 1, 20, 100], np.int32),
                                                            ([1.0, 0.9, 0.5], np.float32), ([0.0, 0.05], np.float32))]
        u = self.rng.random(m).astype(np.float32)
        dev, du, token = [up(a) for a in par], up(u), up(np.full(m + 1, 77, np.int64))
        ctx.sample_dev(logits.ptr, m, VOCAB, du.ptr, token.ptr, *(d.ptr for d in dev), pitch=VOCAB + 3)
        ctx.sync()
        z, t = logits.numpy()[:, :VOCAB], token.numpy()
        assert t[m] == 77
        for r in range(m):
            assert t[r] == choose(z[r], *(float(a[r]) if a.dtype != np.int32 else int(a[r]) for a in par), u[r])[0], r
        return {s: t[first[i]:first[i + 1]] for i, s in enumerate(asks)}

    def keep(self, s, n, branch):
        """Of the tokens drafted from place n on, those of a branch stay."""
        src, dst = [self.slots(s, n + t, n + t + 1)[0] for t in branch], self.slots(s, n, n + len(branch))
        for l in self.layers:
            k, v = l.pool.read(src)
            l.pool.write(k, v, dst)
            k, v = l.pool.read(dst)
            l.k[s], l.v[s] = np.concatenate([l.k[s][:n], k]), np.concatenate([l.v[s][:n], v])
        self.seqs[s][0] = n + len(branch)


@pytest.mark.parametrize("kind", ["f32", "f16", "rowi8"])
def test_prompts_steps_and_drafts(ctx, kind):
    e = Engine(ctx, kind)
    rng = np.random.default_rng(5)
    asks = {s: rng.integers(0, VOCAB, n) for s, n in (("a", 61), ("b", 1), ("c", 34))}
    for _ in range(3):
        asks = {s: t[-1:] for s, t in e.step(asks).items()}
    drafts = {s: np.concatenate([t, rng.integers(0, VOCAB, n)]) for (s, t), n in zip(asks.items(), (11, 4, 0))}
    trees = {s: grow(rng, len(t)) for s, t in drafts.items()}
    at = {s: e.seqs[s][0] for s in drafts}
    got = e.step(drafts, trees)
    for s in drafts:
        branch = sorted(max(trees[s], key=len))
        e.keep(s, at[s], branch)
        asks[s] = got[s][branch[-1]:branch[-1] + 1]
    for _ in range(2):
        asks = {s: t[-1:] for s, t in e.step(asks).items()}
    assert e.seqs["b"][0] == 3 + len(max(trees["b"], key=len)) + 2


def test_a_step_captured_and_replayed(ctx):
    """Append, attention over a window with sinks, logits and token in one graph,
    replayed over growing sequences with eager steps and synchronizations between;
    a tree's step in another, with the same workspaces, the graphs in turn."""
    rng = np.random.default_rng(4)
    l = Layer(ctx, "f16", 90, False)
    head = ctx.upload_rows("f32", rng.standard_normal((VOCAB, HEADS * HD)).astype(np.float32) / 4)
    base, r = 70, 5
    m = 2 * r
    pages = np.stack([rng.permutation(15)[:TABLE], 15 + rng.permutation(15)[:TABLE]]).astype(np.int32)
    tab = up(pages)
    place = lambda s, j: int(pages[s, j // PAGE]) * PAGE + j % PAGE  # noqa: E731
    fused, q, att = (hip.DeviceArray((m, w), np.float32) for w in (WIDE, HEADS * HD, HEADS * HD))
    logits, token, u = hip.DeviceArray((m, VOCAB), np.float32), hip.DeviceArray((m,), np.int64), up(rng.random(m).astype(np.float32))
    topk = up(np.full(m, 30, np.int32))
    pos, slot, ln, fi = up(np.zeros(m, np.int32)), up(np.zeros(m, np.int64)), up(np.zeros(2, np.int32)), up(np.array([0, r, m], np.int32))
    masks = up(np.zeros((m, 1), np.uint64))
    wa = hip.DeviceArray((l.pool.c.attn_ws_bytes(m, HEADS, 2, TABLE),), np.uint8)
    ws = hip.DeviceArray((ctx.sample_ws_bytes(m, VOCAB),), np.uint8)

    def step(tree):
        l.pool.c.append_dev(fused.ptr, HEADS, pos.ptr, slot.ptr, m, q.ptr, l.how)
        l.pool.c.attn_dev(q.ptr, m, HEADS, tab.ptr, TABLE, ln.ptr, 2, att.ptr, first_ptr=fi.ptr, window=WINDOW, sinks=SINKS,
                          ws_ptr=wa.ptr, ws_bytes=wa.nbytes, tree_ptr=masks.ptr if tree else None)
        for i in range(m):
            head.rowdot_f32_dev(att.ptr + 4 * HEADS * HD * i, logits.ptr + 4 * VOCAB * i)
        ctx.sample_dev(logits.ptr, m, VOCAB, u.ptr, token.ptr, topk_ptr=topk.ptr, ws_ptr=ws.ptr, ws_bytes=ws.nbytes)

    # what was cached before
    put(ln, np.array([base, base], np.int32))
    for s in (0, 1):
        l.pool.write(rng.standard_normal((base, KV, HD)).astype(np.float32), rng.standard_normal((base, KV, HD)).astype(np.float32),
                     [place(s, j) for j in range(base)])
    put(slot, np.array([place(s, base + j) for s in (0, 1) for j in range(r)], np.int64))
    step(False)
    ctx.sync()
    graphs = [Graph(ctx, lambda: step(False)), Graph(ctx, lambda: step(True))]
    last = None
    for i in range(4):
        n = base + r * i
        put(fused, rng.standard_normal((m, WIDE)).astype(np.float32))
        put(u, rng.random(m).astype(np.float32))
        put(slot, np.array([place(s, n + j) for s in (0, 1) for j in range(r)], np.int64))
        trees = [grow(rng, r) for _ in range(2)]
        put(masks, words_of(trees, 1))
        put(ln, np.array([n + r, n + r], np.int32))
        for tree in (False, True):
            put(pos, np.array([n + (len(trees[s][j]) - 1 if tree else j) for s in (0, 1) for j in range(r)], np.int32))
            outs = []
            for how in (graphs[tree].replay, lambda: step(tree), graphs[tree].replay):
                put(att, np.full((m, HEADS * HD), 7.0, np.float32))
                put(token, np.full(m, -7, np.int64))
                how()
                ctx.sync()
                outs.append((att.numpy(), token.numpy()))
            for a, t in outs[1:]:
                assert same(a, outs[0][0]) and np.array_equal(t, outs[0][1])
            z, un = logits.numpy(), u.numpy()
            assert [choose(z[j], 1.0, 30, u=un[j])[0] for j in range(m)] == list(outs[0][1])
            assert last is None or not same(outs[0][0], last)
            last = outs[0][0]
    for g in graphs:
        g.close()
