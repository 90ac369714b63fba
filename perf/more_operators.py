"""The measured cases of a serving step's remaining operators: fused q | k | v
rows rotated and appended to the paged cache, attention over a window with
sinks and over a tree of drafted tokens, and sampling.

listed() names the cases, draw(rng) gives further ones of the same ranges.
A case is a dict of plain values with a "kind":

  append  KvCache.append_dev: "rows" fused rows of kv * rep query heads and kv
          key and value heads of hd channels; bias ("bias"), an RMS norm of
          every query and key head ("norm"), the first rot channels turned
          (neighbours where "pairs", else halves), q out in f32, k and v into
          their slots of the pages ("dtype" f32, f16, or rowi8: int8 with a
          scale per token and head, read back in f32 by KvCache.read_dev)
  sink    KvCache.attn_dev with sinks: "seqs" sequences of len_lo .. len_hi
          cached tokens, the last rows_lo .. rows_hi of each asking (0: one
          row each, a decode step), each row seeing the last "window" tokens
          and the sequence's first "sinks"
  tree    KvCache.attn_dev with a tree: the last rows_lo .. rows_hi tokens are
          drafted ones, each seeing what was cached before ("window" 0: all of
          it) and its own ancestors; branches of up to "fan" children
  sample  Context.sample_dev: "rows" rows of "vocab" logits, each row with
          its temperature, top-k, top-p and min-p ("mix" greedy, topk, topp,
          minp, plain, or all: a row of any kind) and its random number

Where `own` is false, run() computes the same from elementary torch
operations.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6


def listed():
    return [
        # one token of one sequence (Qwen2.5-0.5B's heads and biases): the launch latency
        {"name": "append_token", "kind": "append", "dtype": "f16", "page": 16, "kv": 2, "rep": 7, "hd": 64, "rows": 1,
         "bias": True, "norm": False, "rot": 64, "pairs": False, "far": 2000},
        # a decode batch with normed heads, part of an unusual width turned, neighbours paired, far positions
        {"name": "append_batch", "kind": "append", "dtype": "f32", "page": 32, "kv": 5, "rep": 3, "hd": 80, "rows": 61,
         "bias": False, "norm": True, "rot": 32, "pairs": True, "far": 131072},
        # a long prompt into an int8 cache (Qwen2.5-7B's heads and biases)
        {"name": "append_prompt_i8", "kind": "append", "dtype": "rowi8", "page": 64, "kv": 4, "rep": 7, "hd": 128,
         "rows": 8192, "bias": True, "norm": False, "rot": 128, "pairs": False, "far": 8192},
        # a step of one conversation long past its window, on the small model
        {"name": "sink_token", "kind": "sink", "dtype": "f16", "page": 16, "kv": 2, "rep": 7, "hd": 64, "seqs": 1,
         "len_lo": 3001, "len_hi": 3001, "rows_lo": 0, "rows_hi": 0, "window": 1020, "sinks": 4, "cap": 0.0},
        # a serving batch of long conversations over an f32 cache (Gemma-2-2b's heads, window and cap)
        {"name": "sink_batch_f32", "kind": "sink", "dtype": "f32", "page": 32, "kv": 4, "rep": 2, "hd": 256, "seqs": 16,
         "len_lo": 5000, "len_hi": 20000, "rows_lo": 0, "rows_hi": 0, "window": 4096, "sinks": 5, "cap": 50.0},
        # a chunk of a long prompt
        {"name": "sink_prompt", "kind": "sink", "dtype": "f16", "page": 64, "kv": 4, "rep": 7, "hd": 128, "seqs": 1,
         "len_lo": 8192, "len_hi": 8192, "rows_lo": 2048, "rows_hi": 2048, "window": 1024, "sinks": 4, "cap": 0.0},
        # a few drafted tokens after a short context on the small model
        {"name": "tree_short", "kind": "tree", "dtype": "f16", "page": 16, "kv": 2, "rep": 7, "hd": 64, "seqs": 1,
         "len_lo": 211, "len_hi": 211, "rows_lo": 8, "rows_hi": 8, "fan": 2, "window": 0, "sinks": 0, "cap": 0.0},
        # a serving batch over an int8 cache, trees of different sizes (Qwen2.5-7B's heads)
        {"name": "tree_batch_i8", "kind": "tree", "dtype": "rowi8", "page": 64, "kv": 4, "rep": 7, "hd": 128, "seqs": 16,
         "len_lo": 40, "len_hi": 6001, "rows_lo": 5, "rows_hi": 26, "fan": 4, "window": 0, "sinks": 0, "cap": 0.0},
        # one large tree over a long context
        {"name": "tree_long", "kind": "tree", "dtype": "f16", "page": 64, "kv": 8, "rep": 4, "hd": 128, "seqs": 1,
         "len_lo": 32768, "len_hi": 32768, "rows_lo": 64, "rows_hi": 64, "fan": 4, "window": 0, "sinks": 0, "cap": 0.0},
        # the token of one sequence (Qwen2.5-7B's vocabulary)
        {"name": "sample_token", "kind": "sample", "rows": 1, "vocab": 152064, "mix": "topk"},
        # a batch at GPT-2's vocabulary, its kept tokens by their share
        {"name": "sample_small", "kind": "sample", "rows": 9, "vocab": 50257, "mix": "topp"},
        # a serving batch, every request with settings of its own
        {"name": "sample_batch", "kind": "sample", "rows": 64, "vocab": 152064, "mix": "all"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "sink", "sink prompt", "tree", "tree", "sample", "sample"])
    if kind == "sample":
        vocab = rng.choice([50257, 152064, _log(rng, 100, 200000), _log(rng, 100, 200000)])
        rows = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 256)])
        return {"kind": "sample", "rows": max(1, min(rows, 64 * 152064 // vocab)), "vocab": vocab,
                "mix": rng.choice(["greedy", "topk", "topp", "minp", "plain", "all", "all"])}
    c = {"kind": kind.split()[0], "dtype": rng.choice(["f32", "f16", "rowi8"]), "page": rng.choice([16, 32, 64, 128]),
         "kv": rng.choice([1, 2, 3, 4, 5, 8]), "rep": rng.choice([1, 2, 3, 4, 5, 7, 8]),
         "hd": rng.choice([16, 48, 64, 64, 80, 96, 128, 128, 128, 192, 256])}
    if kind == "append":
        width = (c["rep"] + 2) * c["kv"] * c["hd"]
        c["rows"] = max(1, min(rng.choice([1, rng.randint(2, 64), _log(rng, 65, 8192)]), 8192 * 36 * 128 // width))
        c["bias"], c["norm"], c["pairs"] = rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.3
        c["rot"] = rng.choice([c["hd"], c["hd"], c["hd"] // 16 * 8, 8 * rng.randint(1, c["hd"] // 8)])
        c["far"] = c["rows"] + _log(rng, 1, 131072)
        return c
    c["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    width = c["kv"] * c["rep"] * c["hd"]
    if kind == "tree":
        c["seqs"] = rng.choice([1, rng.randint(2, 16), rng.randint(17, 32)])
        c["rows_hi"] = rng.choice([rng.randint(2, 16), rng.randint(17, 64), rng.randint(65, 130)])
        most = 64 * 32768 * 4096 // (c["seqs"] * c["rows_hi"] * width)
        c["len_hi"] = c["rows_hi"] + max(1, min(_log(rng, 20, 32768), most, 8 * 32768 // c["seqs"]))
        c["rows_lo"] = rng.choice([1, c["rows_hi"]])
        c["fan"] = rng.choice([1, 2, 4, 8])
        c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 4096)])
        c["sinks"] = rng.choice([0, rng.randint(1, 64)]) if c["window"] else 0
        c["len_lo"] = rng.choice([c["rows_hi"], max(c["rows_hi"], c["len_hi"] // 2), c["len_hi"]])
        return c
    c["window"], c["sinks"] = _log(rng, 16, 4096), rng.choice([1, 4, rng.randint(2, 64), rng.randint(65, 200)])
    if kind == "sink":
        c["seqs"] = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 64)])
        c["len_hi"] = max(2, min(_log(rng, 200, 65536), 16 * 20000 * 1024 // (c["seqs"] * c["kv"] * c["hd"])))
        c["rows_lo"] = c["rows_hi"] = 0
    else:
        c["seqs"] = rng.choice([1, 1, rng.randint(2, 8)])
        c["len_hi"] = _log(rng, 20, 8192)
        c["rows_hi"] = min(rng.choice([rng.randint(2, 9), _log(rng, 10, 2048)]), c["len_hi"])
        most = 2048 * 8192 * 3584 // (c["seqs"] * width)
        c["rows_hi"] = max(1, min(c["rows_hi"], most // c["len_hi"]))
        c["rows_lo"] = rng.choice([1, c["rows_hi"]])
    c["len_lo"] = rng.choice([1, max(1, c["len_hi"] // 2), c["len_hi"]])
    return c


# ---- inputs -----------------------------------------------------------------

def _own_rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """(cached tokens, asking rows) of each sequence: the case's own, no
    matter what the seed is."""
    rng = _own_rng(case)
    n = case["seqs"]
    lens = [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(n)]
    lens[0] = case["len_hi"]
    rng.shuffle(lens)
    if case["rows_hi"] == 0:
        return lens, [1] * n
    rows = [min(x, rng.randint(case["rows_lo"], case["rows_hi"])) for x in lens]
    at = lens.index(max(lens))
    rows[at] = min(lens[at], case["rows_hi"])
    return lens, rows


def _trees(case):
    """The masks of every drafted token (bit t: it sees the tree's token t,
    itself among them), of trees grown a token at a time."""
    rng = _own_rng(case)
    masks = []
    for r in _lengths(case)[1]:
        own_masks, children = [], [0] * r
        for i in range(r):
            open_ = [j for j in range(max(0, i - 3 * case["fan"]), i) if children[j] < case["fan"]]
            parent = rng.choice(open_) if open_ and i else -1
            if parent >= 0:
                children[parent] += 1
            own_masks.append((own_masks[parent] if parent >= 0 else 0) | 1 << i)
        masks.append(own_masks)
    return masks


def _quantise_rows(x):
    """int8 and step of each row of f32 x (last axis), the cache's rule:
    step = max(max|x| / 127, 1e-8), values round(x / step), half away."""
    step = (x.abs().amax(-1).double() / 127.0).float().clamp_min(1e-8)
    q = (x.double() / step.double()[..., None]).float()
    return (torch.sign(q) * torch.floor(q.abs().double() + 0.5).float()).clamp(-127, 127).to(torch.int8), step


def _pools(case, g, n_pages):
    """The pages of a cache in use: keys (pages, kv, page, hd), values
    (pages, kv, hd, page), and the int8 steps of each token and head."""
    kv, page, hd = case["kv"], case["page"], case["hd"]
    offset = torch.randn(kv, 1, hd, generator=g, device="cuda")
    k = torch.randn(n_pages, kv, page, hd, generator=g, device="cuda") + offset
    v = torch.randn(n_pages, kv, page, hd, generator=g, device="cuda")
    if case["dtype"] == "rowi8":
        (k, ks), (v, vs) = _quantise_rows(k), _quantise_rows(v)
        return k, v.transpose(2, 3).contiguous(), ks, vs
    t = torch.float16 if case["dtype"] == "f16" else torch.float32
    return k.to(t), v.to(t).transpose(2, 3).contiguous(), None, None


_ctx = None


def _context():
    """The program's one context (device 0, its own stream), and torch's view
    of that stream."""
    global _ctx
    if _ctx is None:
        import fieldrun_amd as fa
        c = fa.Context(0)
        _ctx = c, torch.cuda.ExternalStream(c.stream)
    return _ctx


def _take_stream():
    """The program has one stream: the context's, which waits for no other,
    becomes torch's current one.  So inputs are there when a call reads them,
    what torch does with the outputs comes behind the call, and freed memory is
    not given away under it."""
    stream = _context()[1]
    if torch.cuda.current_stream() != stream:
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)


def _handle(case, k, v, ks, vs):
    import fieldrun_amd as fa
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return fa.KvCache(_context()[0], case["dtype"], k.shape[0], case["page"], case["kv"], case["hd"],
                      at(k), at(v), at(ks), at(vs))


def _prepare_sample(case, g, rng):
    m, n = case["rows"], case["vocab"]
    # tokens' shares fall with a power of their rank, steeper in surer places, in random order
    fall = torch.tensor([rng.uniform(0.9, 3.0) for _ in range(m)], device="cuda")
    rank = torch.rand(m, n, generator=g, device="cuda").argsort(1).float() + 1.0
    x = 18.0 - fall[:, None] * rank.log() + 0.3 * torch.randn(m, n, generator=g, device="cuda")
    temp, topk, topp, minp = [], [], [], []
    for _ in range(m):
        kind = case["mix"] if case["mix"] != "all" else rng.choice(["greedy", "topk", "topp", "minp", "plain", "both"])
        temp.append(0.0 if kind == "greedy" else 1.0 if kind == "plain" else rng.uniform(0.5, 1.3))
        topk.append(rng.choice([20, 40, 50, rng.randint(1, 200)]) if kind in ("topk", "both") else 0)
        topp.append(rng.choice([0.8, 0.9, 0.95]) if kind in ("topk", "topp", "both") else 1.0)
        minp.append(rng.choice([0.02, 0.05, 0.1]) if kind in ("minp", "both") else 0.0)
    f = dict(dtype=torch.float32, device="cuda")
    return {"kind": "sample", "x": x, "temp": torch.tensor(temp, **f),
            "topk": torch.tensor(topk, dtype=torch.int32, device="cuda"), "topp": torch.tensor(topp, **f),
            "minp": torch.tensor(minp, **f), "u": torch.rand(m, generator=g, device="cuda"),
            "token": torch.empty(m, dtype=torch.int64, device="cuda"), "prob": torch.empty(m, device="cuda")}


def prepare(case, seed):
    if own:
        _take_stream()
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    if case["kind"] == "sample":
        state = _prepare_sample(case, g, random.Random(int(seed)))
        if own:
            need = _context()[0].sample_ws_bytes(case["rows"], case["vocab"])
            state["ws"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
        return state
    kv, page, hd = case["kv"], case["page"], case["hd"]
    heads = kv * case["rep"]
    if case["kind"] == "append":
        rows, rot = case["rows"], case["rot"]
        n_pages = (rows + page - 1) // page + 9
        k, v, ks, vs = _pools(case, g, n_pages)
        pages = torch.randperm(n_pages, generator=g, device="cuda")
        if rows <= 64:  # a token of each of so many sequences
            slot = torch.randperm(n_pages * page, generator=g, device="cuda")[:rows].contiguous()
            pos = torch.randint(0, case["far"], (rows,), generator=g, device="cuda")
        else:  # the tokens of a prompt, in order, from the middle of a page
            at = torch.arange(rows, device="cuda") + page // 2 + 1
            slot = pages[at // page] * page + at % page
            pos = torch.arange(rows, device="cuda") + (case["far"] - rows)
        wide = (heads + 2 * kv) * hd
        near = lambda n, s: 1.0 + s * torch.randn(n, generator=g, device="cuda")  # noqa: E731
        state = {"kind": "append", "slot": slot, "pos": pos.to(torch.int32), "page": page, "heads": heads, "rot": rot,
                 "pairs": case["pairs"], "qkv": torch.randn(rows, wide, generator=g, device="cuda"),
                 "bias": 0.5 * torch.randn(wide, generator=g, device="cuda") if case["bias"] else None,
                 "qn": near(hd, 0.2) if case["norm"] else None, "kn": near(hd, 0.2) if case["norm"] else None,
                 "freq": 1e6 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / rot),
                 "q": torch.empty(rows, heads, hd, device="cuda"),
                 "out_k": torch.empty(rows, kv, hd, device="cuda"), "out_v": torch.empty(rows, kv, hd, device="cuda")}
        state.update(k=k, v=v, ks=ks, vs=vs)
        if own:
            import fieldrun_amd as fa
            at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
            state["handle"] = _handle(case, k, v, ks, vs)
            state["how"] = fa.Rotary(rot, state["freq"].data_ptr(), pairs=case["pairs"], bias_ptr=at(state["bias"]),
                                     q_norm_ptr=at(state["qn"]), k_norm_ptr=at(state["kn"]), eps=EPS)
        return state
    lens, rows = _lengths(case)
    held = [(x + page - 1) // page for x in lens]
    n_pages, width = sum(held) + 3, max(held)
    k, v, ks, vs = _pools(case, g, n_pages)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    n = sum(rows)
    first = [sum(rows[:s]) for s in range(len(rows) + 1)]
    words = 0
    if case["kind"] == "tree":
        words = (max(rows) + 63) // 64
        flat = [m >> 64 * w & (1 << 64) - 1 for masks in _trees(case) for m in masks for w in range(words)]
        mask = torch.tensor([w - (1 << 64) if w >> 63 else w for w in flat], dtype=torch.int64, device="cuda")
    state = {"kind": case["kind"], "page": page, "rep": case["rep"], "cap": case["cap"], "window": case["window"],
             "sinks": case["sinks"], "decode": case["rows_hi"] == 0, "most": max(rows), "words": words,
             "span": max(lens) if not case["window"] else min(max(lens), case["window"] + max(rows)),
             "q": 1.5 * torch.randn(n, heads, hd, generator=g, device="cuda"), "table": table,
             "tree": mask.reshape(n, words) if words else None,
             "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
             "first": torch.tensor(first, dtype=torch.int32, device="cuda"), "out": torch.empty(n, heads, hd, device="cuda")}
    state.update(k=k, v=v, ks=ks, vs=vs, handle=_handle(case, k, v, ks, vs) if own else None)
    if own:
        need = state["handle"].attn_ws_bytes(n, heads, case["seqs"], width)
        state["ws"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    return state


# ---- the plain forms ----------------------------------------------------------

def _plain_append(s):
    rows, kv, hd, heads = s["qkv"].shape[0], s["k"].shape[1], s["k"].shape[3], s["heads"]
    x = s["qkv"].double() if s["bias"] is None else s["qkv"].double() + s["bias"].double()
    x = x.reshape(rows, heads + 2 * kv, hd)
    qk, v = x[:, :heads + kv], x[:, heads + kv:].float()
    if s["qn"] is not None:
        gain = torch.cat([s["qn"].expand(heads, hd), s["kn"].expand(kv, hd)]).double()
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * gain
    angle = s["pos"].double()[:, None] * s["freq"]
    c, i = angle.cos()[:, None], angle.sin()[:, None]
    half, rot = s["rot"] // 2, s["rot"]
    if s["pairs"]:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack([a * c - b * i, b * c + a * i], -1).flatten(-2)
    else:
        a, b = qk[..., :half], qk[..., half:rot]
        turned = torch.cat([a * c - b * i, b * c + a * i], -1)
    qk = torch.cat([turned, qk[..., rot:]], -1).float()
    q, k = qk[:, :heads].contiguous(), qk[:, heads:]
    page, off = s["slot"] // s["page"], s["slot"] % s["page"]
    if s["ks"] is None:
        s["k"][page, :, off] = k.to(s["k"].dtype)
        s["v"][page, :, :, off] = v.to(s["v"].dtype)
        return {"q": q, "k": s["k"], "v": s["v"]}
    s["k"][page, :, off], s["ks"][page, :, off] = _quantise_rows(k)
    s["v"][page, :, :, off], s["vs"][page, :, off] = _quantise_rows(v)
    return {"q": q, "k": s["k"][page, :, off].float() * s["ks"][page, :, off][..., None],
            "v": s["v"][page, :, :, off].float() * s["vs"][page, :, off][..., None]}


def _plain_attn(s):
    """Over the tokens that some row of a sequence may see: its first ones
    (sinks), then those from the oldest window's beginning on."""
    lens, first, page = s["lens"].long(), s["first"].long(), s["page"]
    seqs, most, dev = lens.shape[0], s["most"], lens.device
    kv, hd, rep = s["k"].shape[1], s["k"].shape[3], s["rep"]
    rows = first[1:] - first[:-1]
    base = lens - rows
    low = (base - s["window"]).clamp_min(s["sinks"]) if s["window"] else torch.zeros_like(lens)
    key = torch.cat([torch.arange(s["sinks"], device=dev).expand(seqs, -1),
                     low[:, None] + torch.arange(s["span"], device=dev)], 1)  # (seqs, keys)
    held = key < lens[:, None]
    at = torch.where(held, key, 0)
    pg, off = s["table"].clamp_min(0).long().gather(1, at // page), at % page
    k, v = s["k"][pg, :, off].float(), s["v"][pg, :, :, off].float()  # (seqs, keys, kv, hd)
    if s["ks"] is not None:
        k = k * s["ks"][pg, :, off][..., None]
        v = v * s["vs"][pg, :, off][..., None]
    keys = key.shape[1]
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.permute(0, 2, 1, 3).contiguous()
    i = torch.arange(most, device=dev)
    of_q = (first[:-1, None] + i).clamp_max(max(0, s["q"].shape[0] - 1))
    q = s["q"][of_q].reshape(seqs, most, kv, rep, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv, rep * most, hd)
    score = torch.matmul(q, k).reshape(seqs, kv, rep, most, keys) * hd ** -0.5
    if s["cap"]:
        score = s["cap"] * torch.tanh(score / s["cap"])
    if s["tree"] is None:
        pos = base[:, None] + i  # the rows' places
        seen = key[:, None] <= pos[..., None]
    else:
        t = torch.arange(64 * s["words"], device=dev)
        bits = (s["tree"][:, t // 64] >> (t % 64) & 1).bool()[of_q]  # (seqs, most, drafted)
        pos = base[:, None] - 1 + bits.sum(-1)
        draft = key - base[:, None]
        mine = bits.gather(2, draft.clamp(0, 64 * s["words"] - 1)[:, None].expand(-1, most, -1))
        seen = (draft < 0)[:, None] | mine & (draft >= 0)[:, None]
    if s["window"]:
        near = (key[:, None] > pos[..., None] - s["window"]) | (key < s["sinks"])[:, None]
        seen = seen & (near if s["tree"] is None else near | (draft >= 0)[:, None])
    seen = seen & held[:, None]
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    o = torch.matmul(p.reshape(seqs, kv, rep * most, keys), v).reshape(seqs, kv, rep, most, hd)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, most, kv * rep, hd)
    r = torch.arange(s["q"].shape[0], device=dev)
    of = torch.searchsorted(first[1:].contiguous(), r, right=True)  # each row's sequence
    return o[of, r - first[of]]


def _plain_sample(s):
    x, n = s["x"], s["x"].shape[1]
    greedy = s["temp"] == 0
    temp = torch.where(greedy, 1.0, s["temp"]).double()[:, None]
    z, order = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
    w = torch.exp((z.double() - z[:, :1].double()) / temp)
    place = torch.arange(n, device=x.device)
    keep = (s["topk"][:, None] <= 0) | (place < s["topk"][:, None])
    keep &= ~greedy[:, None] | (place == 0)
    w = torch.where(keep, w, 0.0)
    before = torch.cumsum(w, 1) - w
    p = s["topp"].double()[:, None]
    keep = (p >= 1) | (place == 0) | (before < p * w.sum(1, keepdim=True))
    keep &= (w >= s["minp"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))  # in the tokens' own order
    total = torch.cumsum(w, 1)
    token = (total <= s["u"].double()[:, None] * total[:, -1:]).sum(1)
    return {"token": token, "prob": (w.gather(1, token[:, None])[:, 0] / total[:, -1]).float()}


# ---- one pass -----------------------------------------------------------------

def run(state):
    s = state
    if s["kind"] == "append":
        if not own:
            return _plain_append(s)
        h, rows, slot = s["handle"], s["qkv"].shape[0], s["slot"].data_ptr()
        h.append_dev(s["qkv"].data_ptr(), s["heads"], s["pos"].data_ptr(), slot, rows, s["q"].data_ptr(), s["how"])
        if s["ks"] is None:
            return {"q": s["q"], "k": s["k"], "v": s["v"]}
        h.read_dev(slot, rows, s["out_k"].data_ptr(), s["out_v"].data_ptr())  # what the bytes stand for
        return {"q": s["q"], "k": s["out_k"], "v": s["out_v"]}
    if s["kind"] == "sample":
        if not own:
            return _plain_sample(s)
        at = {name + "_ptr": s[name].data_ptr() for name in ("temp", "topk", "topp", "minp", "prob")}
        _context()[0].sample_dev(s["x"].data_ptr(), s["x"].shape[0], s["x"].shape[1], s["u"].data_ptr(),
                                 s["token"].data_ptr(), **at, ws_ptr=s["ws"].data_ptr(), ws_bytes=s["ws"].numel())
        return {"token": s["token"], "prob": s["prob"]}
    if not own:
        return _plain_attn(s)
    q, table, ws = s["q"], s["table"], s["ws"]
    s["handle"].attn_dev(q.data_ptr(), q.shape[0], q.shape[1], table.data_ptr(), table.shape[1], s["lens"].data_ptr(),
                         table.shape[0], s["out"].data_ptr(), first_ptr=None if s["decode"] else s["first"].data_ptr(),
                         cap=s["cap"], window=s["window"], sinks=s["sinks"],
                         tree_ptr=None if s["tree"] is None else s["tree"].data_ptr(), tree_pitch=s["words"],
                         ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------

def _size(case):
    return {"f32": 4, "f16": 2, "rowi8": 1}[case["dtype"]]


def _seen(case, n, r, masks):
    """(tokens that some of the sequence's r rows see, pairs of a row and a
    token that it sees)"""
    window, sinks, base = case["window"] or n, case["sinks"], n - r
    if case["kind"] == "sink":
        last = [base + i for i in range(r)]  # a row's last token
        pairs = sum(min(p + 1, window + sinks) for p in last)
        return min(n, window + r - 1 + sinks), pairs
    depth = [bin(m).count("1") for m in masks]
    old = [min(base, max(0, window - d) + min(sinks, base)) for d in depth]  # of the cached ones
    return min(n, max(old, default=0) + r), sum(old) + sum(depth)


def work(case):
    if case["kind"] == "sample":
        m, n = case["rows"], case["vocab"]
        # the logits read; a maximum, a difference, a weight and a sum for each
        return {"bytes": 4 * m * n + 32 * m, "flops": 8 * m * n}
    kv, hd, size = case["kv"], case["hd"], _size(case)
    heads = kv * case["rep"]
    token = 2 * kv * (hd * size + (4 if size == 1 else 0))
    if case["kind"] == "append":
        m = case["rows"]
        back = token + 8 * kv * hd if size == 1 else 0  # int8 rows read back
        return {"bytes": m * (4 * (2 * heads + 2 * kv) * hd + token + back + 12), "flops": 8 * m * (heads + kv) * hd}
    lens, rows = _lengths(case)
    trees = _trees(case) if case["kind"] == "tree" else [None] * len(lens)
    seen = [_seen(case, n, r, t) for n, r, t in zip(lens, rows, trees)]
    return {"bytes": sum(a for a, _ in seen) * token + 8 * sum(rows) * heads * hd,
            "flops": 4 * sum(b for _, b in seen) * heads * hd}


# ---- the same values in 64 bits, from the definitions ---------------------------

def _rounded(x):
    """What an int8 row of the cache stands for, row by row in 64 bits; the
    step and the quotients are the rule's f32 values."""
    step = torch.maximum((x.abs().max(-1, keepdim=True).values.double() / 127).to(torch.float32),
                         torch.tensor(1e-8, device=x.device))
    q = (x.double() / step.double()).to(torch.float32).double()
    low = torch.trunc(q)
    q = low + torch.where((q - low).abs() >= 0.5, torch.sign(q), torch.zeros_like(q))
    return q.clamp(-127.0, 127.0) * step.double()


def _exact_append(case, s):
    kv, hd, heads, rot, page = case["kv"], case["hd"], s["heads"], case["rot"], case["page"]
    x = s["qkv"].double()
    if s["bias"] is not None:
        x += s["bias"].double()
    x = x.reshape(-1, heads + 2 * kv, hd)
    for h in range(heads + kv):
        if s["qn"] is not None:
            gain = s["qn"] if h < heads else s["kn"]
            x[:, h] /= torch.sqrt((x[:, h] ** 2).sum(1, keepdim=True) / hd + EPS)
            x[:, h] *= gain.double()
    for j in range(rot // 2):  # one plane of the rotation at a time, as a complex number
        a, b = (2 * j, 2 * j + 1) if case["pairs"] else (j, j + rot // 2)
        turn = torch.polar(torch.ones_like(s["pos"], dtype=torch.float64), s["pos"].double() * s["freq"][j])
        z = torch.complex(x[:, :heads + kv, a], x[:, :heads + kv, b]) * turn[:, None]
        x[:, :heads + kv, a], x[:, :heads + kv, b] = z.real, z.imag
    q, k, v = x[:, :heads], x[:, heads:heads + kv].float(), x[:, heads + kv:].float()
    if case["dtype"] == "rowi8":
        return {"q": q, "k": _rounded(k), "v": _rounded(v)}
    pool_k, pool_v = s["k"].double(), s["v"].double()
    for i, slot in enumerate(s["slot"].tolist()):
        pool_k[slot // page, :, slot % page] = k[i].to(s["k"].dtype).double()
        pool_v[slot // page, :, :, slot % page] = v[i].to(s["v"].dtype).double()
    return {"q": q, "k": pool_k, "v": pool_v}


def _exact_sample(case, s):
    token, prob = [], []
    for r in range(case["rows"]):
        x, t = s["x"][r].double(), float(s["temp"][r])
        if t == 0.0:
            token.append(int((x == x.max()).nonzero()[0, 0]))
            prob.append(1.0)
            continue
        w = torch.exp(x / t - x.max() / t)
        by = torch.from_numpy(np.argsort(-x.cpu().numpy(), kind="stable")).to(x.device)
        if int(s["topk"][r]) > 0:
            by = by[:int(s["topk"][r])]
        share = w[by] / w[by].sum()
        if float(s["topp"][r]) < 1.0:
            cut = torch.cumsum(share, 0)
            count = 1 + int((cut[:-1] < float(s["topp"][r])).sum())
            by = by[:count]
        by = by[w[by] >= float(s["minp"][r]) * w.max()].sort().values
        share = torch.cumsum(w[by] / w[by].sum(), 0)
        i = int((share <= float(s["u"][r])).sum())
        token.append(int(by[min(i, len(by) - 1)]))
        prob.append(float(w[token[-1]] / w[by].sum()))
    return {"token": torch.tensor(token, device="cuda"), "prob": torch.tensor(prob, dtype=torch.float64, device="cuda")}


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "sample":
        return _exact_sample(case, s)
    if s["kind"] == "append":
        return _exact_append(case, s)
    lens, rows = _lengths(case)
    trees = _trees(case) if s["kind"] == "tree" else [None] * len(lens)
    page, hd, rep, kv = case["page"], case["hd"], case["rep"], case["kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, r, masks) in enumerate(zip(lens, rows, trees)):
        held = s["table"][i, :(n + page - 1) // page].long()
        j = torch.arange(n, device="cuda")[None]
        pos = torch.arange(n - r, n, device="cuda")[:, None]
        hidden = j > pos
        if masks is not None:
            tree = [[m >> t & 1 for t in range(r)] for m in masks]
            hidden = torch.zeros(r, n, dtype=torch.bool, device="cuda")
            hidden[:, n - r:] = torch.tensor(tree, device="cuda") == 0
            pos = n - r - 1 + torch.tensor([[sum(t)] for t in tree], device="cuda")
        if case["window"]:
            old = (pos - j >= case["window"]) & (j >= case["sinks"])
            if masks is not None:
                old = old & (j < n - r)
            hidden = hidden | old
        for h in range(kv):
            k = s["k"][held, h].double()
            v = s["v"][held, h].double()
            if s["ks"] is not None:
                k = k * s["ks"][held, h].double()[:, :, None]
                v = v * s["vs"][held, h].double()[:, None, :]
            k = k.reshape(-1, hd)[:n]
            v = v.transpose(1, 2).reshape(-1, hd)[:n]
            for e in range(h * rep, (h + 1) * rep):
                z = s["q"][at:at + r, e].double() @ k.T.contiguous() / math.sqrt(hd)
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                out[at:at + r, e] = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ v
        at += r
    return out
