"""The measured cases of the paged key / value cache, the attention that reads
it, and the norm that feeds the int8 linears.

listed() names the cases, draw(rng) gives further ones of the same ranges.
A case is a dict of plain values with a "kind":

  cache  KvCache.write_dev + read_dev: "rows" tokens' keys and values written
         into their slots of the pages ("dtype" f32, f16 or rowi8: int8 with a
         scale per token and head), and the same slots read back in f32
  attn   KvCache.attn_dev: "seqs" sequences ("idle" of them empty) of len_lo
         .. len_hi cached tokens, the last rows_lo .. rows_hi of each asking
         (0: one row each, a decode step), kv heads of width hd read by rep
         query heads each; "window" 0: all earlier tokens, "cap" 0: no cap
  norm   Context.norm_quant_dev: rows of k: residual added ("residual"), RMS
         norm, and the outlier-aware int8 rows that the int8 linear takes

Where `own` is false, run() computes the same from elementary torch
operations.
"""
import math
import random

import torch

own = False

OUTLIERS = 32  # outlier channels of an int8 row
EPS = 1e-6


def listed():
    return [
        # one token of one sequence appended (Qwen2.5-0.5B's 2 heads of 64): the launch latencies
        {"name": "cache_token", "kind": "cache", "dtype": "f16", "page": 16, "kv": 2, "hd": 64, "rows": 1},
        # a decode step of a ragged batch at a head width that is no power of two
        {"name": "cache_batch", "kind": "cache", "dtype": "f32", "page": 32, "kv": 5, "hd": 80, "rows": 61},
        # a long prompt quantised as it is written (Qwen2.5-7B's 4 heads of 128)
        {"name": "cache_prompt_i8", "kind": "cache", "dtype": "rowi8", "page": 64, "kv": 4, "hd": 128, "rows": 8192},
        # the first answer token after a short prompt on the small model
        {"name": "decode_short", "kind": "attn", "dtype": "f16", "page": 16, "kv": 2, "rep": 7, "hd": 64, "seqs": 1,
         "idle": 0, "len_lo": 77, "len_hi": 77, "rows_lo": 0, "rows_hi": 0, "window": 0, "cap": 0.0},
        # a serving batch over an int8 cache, ragged, with unused places (Qwen2.5-7B's heads)
        {"name": "decode_batch_i8", "kind": "attn", "dtype": "rowi8", "page": 64, "kv": 4, "rep": 7, "hd": 128,
         "seqs": 48, "idle": 3, "len_lo": 1, "len_hi": 6001, "rows_lo": 0, "rows_hi": 0, "window": 0, "cap": 0.0},
        # sixteen sequences at Gemma-2-2b's heads, soft cap and window, over an f32 cache
        {"name": "decode_window_f32", "kind": "attn", "dtype": "f32", "page": 32, "kv": 4, "rep": 2, "hd": 256,
         "seqs": 16, "idle": 0, "len_lo": 3000, "len_hi": 7000, "rows_lo": 0, "rows_hi": 0, "window": 4096,
         "cap": 50.0},
        # one sequence with a very long context
        {"name": "decode_long", "kind": "attn", "dtype": "f16", "page": 64, "kv": 8, "rep": 4, "hd": 128, "seqs": 1,
         "idle": 0, "len_lo": 131071, "len_hi": 131071, "rows_lo": 0, "rows_hi": 0, "window": 0, "cap": 0.0},
        # a chunk of a long prompt over what is cached of it
        {"name": "prompt_chunk", "kind": "attn", "dtype": "f16", "page": 64, "kv": 4, "rep": 7, "hd": 128, "seqs": 1,
         "idle": 0, "len_lo": 8192, "len_hi": 8192, "rows_lo": 2048, "rows_hi": 2048, "window": 0, "cap": 0.0},
        # prompts of several users at once, some behind a shared beginning, int8 cache
        {"name": "prompt_ragged_i8", "kind": "attn", "dtype": "rowi8", "page": 32, "kv": 4, "rep": 7, "hd": 128,
         "seqs": 7, "idle": 1, "len_lo": 90, "len_hi": 1501, "rows_lo": 1, "rows_hi": 900, "window": 0, "cap": 0.0},
        # a decode step's row before gate|up (Qwen2.5-7B)
        {"name": "norm_token", "kind": "norm", "rows": 1, "k": 3584, "residual": True},
        # a decode batch at a width that is no multiple of four
        {"name": "norm_batch_odd", "kind": "norm", "rows": 13, "k": 1027, "residual": True},
        # a long prompt's rows
        {"name": "norm_prompt", "kind": "norm", "rows": 4096, "k": 4096, "residual": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "decode", "decode", "decode", "prompt", "prompt", "norm"])
    if kind == "norm":
        k = _log(rng, 40, 18944)
        if rng.random() < 0.7:
            k = max(64, k // 32 * 32)
        rows = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 4096)])
        return {"kind": "norm", "rows": max(1, min(rows, 4096 * 4096 // k)), "k": k, "residual": rng.random() < 0.7}
    c = {"kind": "cache" if kind == "cache" else "attn", "dtype": rng.choice(["f32", "f16", "rowi8"]),
         "page": rng.choice([16, 32, 64, 128]), "kv": rng.choice([1, 2, 3, 4, 5, 8]),
         "hd": rng.choice([16, 48, 64, 64, 80, 96, 128, 128, 128, 192, 256])}
    if kind == "cache":
        c["rows"] = max(1, min(rng.choice([1, rng.randint(2, 64), _log(rng, 65, 8192)]),
                               8192 * 512 // (c["kv"] * c["hd"])))
        return c
    c["rep"] = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
    c["cap"] = rng.choice([0.0, 0.0, 30.0, 50.0])
    if kind == "decode":
        c["seqs"] = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 128)])
        c["idle"] = rng.choice([0, 0, c["seqs"] // 4])
        c["len_hi"] = max(2, min(_log(rng, 20, 131072), 8 * 131072 // (c["seqs"] * c["kv"]) * 32 // c["hd"]))
        c["rows_lo"] = c["rows_hi"] = 0
    else:
        c["seqs"] = rng.choice([1, 1, rng.randint(2, 8)])
        c["idle"] = rng.choice([0, 0, c["seqs"] // 3])
        c["len_hi"] = _log(rng, 20, 4096)
        c["rows_hi"] = min(rng.choice([rng.randint(2, 9), _log(rng, 10, 2048)]), c["len_hi"])
        most = 2048 * 7000 * 28 * 128 // (c["seqs"] * c["kv"] * c["rep"] * c["hd"])
        c["rows_hi"] = max(1, min(c["rows_hi"], most // c["len_hi"]))
        c["rows_lo"] = rng.choice([1, c["rows_hi"]])
    c["len_lo"] = rng.choice([1, max(1, c["len_hi"] // 2), c["len_hi"]])
    c["window"] = rng.choice([0, 0, _log(rng, 1, 4096)])
    return c


# ---- inputs -----------------------------------------------------------------

def _lengths(case):
    """(cached tokens, asking rows) of each sequence: the case's own, no
    matter what the seed is."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n, idle = case["seqs"], case["idle"]
    lens = [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(n)]
    lens[0] = case["len_hi"]
    rng.shuffle(lens)
    for s in rng.sample(range(n), idle):
        lens[s] = 0
    if case["rows_hi"] == 0:
        return lens, [1] * n
    rows = [min(x, rng.randint(case["rows_lo"], case["rows_hi"])) for x in lens]
    at = lens.index(max(lens))
    rows[at] = min(lens[at], case["rows_hi"])
    return lens, rows


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


def prepare(case, seed):
    if own:
        _take_stream()
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    if case["kind"] == "norm":
        m, k = case["rows"], case["k"]
        x = torch.randn(m, k, generator=g, device="cuda")
        x[:, torch.randperm(k, generator=g, device="cuda")[:max(1, k // 100)]] *= 20.0
        pitch = (k + 127) // 128 * 128
        return {"kind": "norm", "x": x, "w": 1.0 + 0.2 * torch.randn(k, generator=g, device="cuda"),
                "y": torch.randn(m, k, generator=g, device="cuda") if case["residual"] else None,
                "sum": torch.empty(m, k, device="cuda"), "a8": torch.empty(m, pitch, dtype=torch.int8, device="cuda"),
                "sa": torch.empty(m, device="cuda"),
                "index": torch.empty(m, OUTLIERS, dtype=torch.int32, device="cuda"),
                "outlier": torch.empty(m, OUTLIERS, device="cuda")}
    kv, page, hd = case["kv"], case["page"], case["hd"]
    if case["kind"] == "cache":
        rows = case["rows"]
        used = (rows + page - 1) // page
        n_pages = used + 9
        k, v, ks, vs = _pools(case, g, n_pages)
        pages = torch.randperm(n_pages, generator=g, device="cuda")
        if rows <= 64:  # a token of each of so many sequences
            slot = torch.randperm(n_pages * page, generator=g, device="cuda")[:rows].contiguous()
        else:  # the tokens of a prompt, in order, from the middle of a page
            at = torch.arange(rows, device="cuda") + page // 2 + 1
            slot = pages[at // page] * page + at % page
        state = {"kind": "cache", "slot": slot, "page": page,
                 "new_k": torch.randn(rows, kv, hd, generator=g, device="cuda"),
                 "new_v": torch.randn(rows, kv, hd, generator=g, device="cuda"),
                 "out_k": torch.empty(rows, kv, hd, device="cuda"), "out_v": torch.empty(rows, kv, hd, device="cuda")}
    else:
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
        n, heads = sum(rows), kv * case["rep"]
        first = [sum(rows[:s]) for s in range(len(rows) + 1)]
        state = {"kind": "attn", "page": page, "rep": case["rep"], "cap": case["cap"], "window": case["window"],
                 "decode": case["rows_hi"] == 0, "q": 1.5 * torch.randn(n, heads, hd, generator=g, device="cuda"),
                 "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
                 "first": torch.tensor(first, dtype=torch.int32, device="cuda"), "most": max(rows),
                 "out": torch.empty(n, heads, hd, device="cuda")}
    state.update(k=k, v=v, ks=ks, vs=vs, handle=_handle(case, k, v, ks, vs) if own else None)
    if own and state["kind"] == "attn":
        need = state["handle"].attn_ws_bytes(state["q"].shape[0], heads, case["seqs"], width)
        state["ws"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    return state


# ---- the plain forms ----------------------------------------------------------

def _plain_cache(s):
    page, off = s["slot"] // s["page"], s["slot"] % s["page"]
    k, v, ks, vs = s["k"], s["v"], s["ks"], s["vs"]
    if ks is None:
        k[page, :, off] = s["new_k"].to(k.dtype)
        v[page, :, :, off] = s["new_v"].to(v.dtype)
        return {"k": k[page, :, off].float(), "v": v[page, :, :, off].float()}
    k[page, :, off], ks[page, :, off] = _quantise_rows(s["new_k"])
    v[page, :, :, off], vs[page, :, off] = _quantise_rows(s["new_v"])
    return {"k": k[page, :, off].float() * ks[page, :, off][..., None],
            "v": v[page, :, :, off].float() * vs[page, :, off][..., None]}


def _plain_attn(s):
    table, lens, first = s["table"].clamp_min(0).long(), s["lens"].long(), s["first"].long()
    seqs, keys = table.shape[0], table.shape[1] * s["page"]
    kv, hd, rep, most = s["k"].shape[1], s["k"].shape[3], s["rep"], s["most"]
    k, v = s["k"][table].float(), s["v"][table].float()  # (seqs, pages, kv, page, hd), (seqs, pages, kv, hd, page)
    if s["ks"] is not None:
        k = k * s["ks"][table][..., None]
        v = v * s["vs"][table][..., None, :]
    k = k.permute(0, 2, 4, 1, 3).reshape(seqs, kv, hd, keys)
    v = v.permute(0, 2, 1, 4, 3).reshape(seqs, kv, keys, hd)
    rows = first[1:] - first[:-1]
    i = torch.arange(most, device=k.device)
    at = (first[:-1, None] + i).clamp_max(max(0, s["q"].shape[0] - 1))
    q = s["q"][at].reshape(seqs, most, kv, rep, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kv, rep * most, hd)
    score = torch.matmul(q, k).reshape(seqs, kv, rep, most, keys) * hd ** -0.5
    if s["cap"]:
        score = s["cap"] * torch.tanh(score / s["cap"])
    pos = (lens - rows)[:, None] + i  # the rows' places
    j = torch.arange(keys, device=k.device)
    seen = (j <= pos[..., None]) & (j < lens[:, None, None])
    if s["window"]:
        seen &= j > pos[..., None] - s["window"]
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    o = torch.matmul(p.reshape(seqs, kv, rep * most, keys), v).reshape(seqs, kv, rep, most, hd)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, most, kv * rep, hd)
    r = torch.arange(s["q"].shape[0], device=k.device)
    of = torch.searchsorted(first[1:].contiguous(), r, right=True)  # each row's sequence
    return o[of, r - first[of]]


def _plain_norm(s):
    x = s["x"] if s["y"] is None else s["x"] + s["y"]
    m, k = x.shape
    wide = x.double()
    n = (wide * torch.rsqrt(wide.square().mean(1, keepdim=True) + EPS) * s["w"].double()).float()
    order = torch.sort(n.abs(), dim=1, descending=True, stable=True).indices
    index = torch.sort(order[:, :OUTLIERS], dim=1).values
    bulk = n.abs().gather(1, order[:, OUTLIERS:OUTLIERS + 1])[:, 0]
    sa = torch.where(bulk > 0, (bulk.double() / 127.0).float(), torch.ones_like(bulk))
    q = (n.double() / sa.double()[:, None]).float().double()
    q = (torch.sign(q) * torch.floor(q.abs() + 0.5)).clamp(-127, 127)
    out = torch.zeros_like(n, dtype=torch.bool).scatter_(1, index, True)
    return {"sum": x, "values": torch.where(out, 0.0, q).float() * sa[:, None], "sa": sa,
            "index": index.to(torch.int32), "outlier": n.gather(1, index)}


# ---- one pass -----------------------------------------------------------------

def run(state):
    if state["kind"] == "cache":
        if not own:
            return _plain_cache(state)
        h, slot, rows = state["handle"], state["slot"].data_ptr(), state["slot"].shape[0]
        h.write_dev(state["new_k"].data_ptr(), state["new_v"].data_ptr(), slot, rows)
        h.read_dev(slot, rows, state["out_k"].data_ptr(), state["out_v"].data_ptr())
        return {"k": state["out_k"], "v": state["out_v"]}
    if state["kind"] == "attn":
        if not own:
            return _plain_attn(state)
        q, table, ws = state["q"], state["table"], state["ws"]
        state["handle"].attn_dev(q.data_ptr(), q.shape[0], q.shape[1], table.data_ptr(), table.shape[1],
                                 state["lens"].data_ptr(), table.shape[0], state["out"].data_ptr(),
                                 first_ptr=None if state["decode"] else state["first"].data_ptr(),
                                 cap=state["cap"], window=state["window"], ws_ptr=ws.data_ptr(), ws_bytes=ws.numel())
        return state["out"]
    if not own:
        return _plain_norm(state)
    ctx = _context()[0]
    x, y, a8, sa = state["x"], state["y"], state["a8"], state["sa"]
    total = x if y is None else state["sum"]
    ctx.norm_quant_dev(x.data_ptr(), None if y is None else y.data_ptr(), state["w"].data_ptr(), EPS, x.shape[0],
                       x.shape[1], None if y is None else total.data_ptr(), a8.data_ptr(), sa.data_ptr(),
                       state["index"].data_ptr(), state["outlier"].data_ptr())
    values = a8[:, :x.shape[1]] * sa[:, None]  # what the bytes stand for
    return {"sum": total, "values": values, "sa": sa, "index": state["index"], "outlier": state["outlier"]}


# ---- what a pass cannot do without ---------------------------------------------

def _size(case):
    return {"f32": 4, "f16": 2, "rowi8": 1}[case["dtype"]]


def work(case):
    if case["kind"] == "norm":
        m, k = case["rows"], case["k"]
        # x, y and w read, the sum, the int8 rows, their steps and outliers written
        return {"bytes": m * k * (4 + (8 if case["residual"] else 0) + 1) + 4 * k + m * (4 + 8 * OUTLIERS),
                "flops": 6 * m * k}
    kv, hd, size = case["kv"], case["hd"], _size(case)
    token = 2 * kv * (hd * size + (4 if size == 1 else 0))
    if case["kind"] == "cache":
        # read f32, write the cache; read the cache, write f32
        return {"bytes": case["rows"] * (2 * 2 * kv * hd * 4 + 2 * token + 16), "flops": 4 * case["rows"] * kv * hd}
    lens, rows = _lengths(case)
    read = pairs = 0
    for n, r in zip(lens, rows):
        r = min(n, r)
        w = case["window"] or n
        read += min(n, w + r - 1) if r else 0
        pairs += sum(min(w, n - r + i + 1) for i in range(r))
    heads = kv * case["rep"]
    return {"bytes": read * token + 8 * sum(rows) * heads * hd, "flops": 4 * pairs * heads * hd}


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


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "cache":
        if case["dtype"] == "rowi8":
            return {"k": _rounded(s["new_k"]), "v": _rounded(s["new_v"])}
        t = s["k"].dtype
        return {"k": s["new_k"].to(t).double(), "v": s["new_v"].to(t).double()}
    if s["kind"] == "norm":
        x = s["x"].double()
        if s["y"] is not None:
            x = (x + s["y"].double()).float().double()
        var = (x * x).sum(1) / x.shape[1]
        n = (x / torch.sqrt(var + EPS)[:, None] * s["w"].double()).float().double()
        big, where = torch.topk(n.abs(), OUTLIERS + 1, dim=1, sorted=True)
        step = torch.where(big[:, -1] > 0, (big[:, -1] / 127).float().double(), 1.0)
        q = (n / step[:, None]).float().double()
        q = torch.where(q < 0, -torch.floor(0.5 - q), torch.floor(q + 0.5)).clamp(-127.0, 127.0)
        index = where[:, :OUTLIERS].sort(1).values
        return {"sum": x, "values": (q * step[:, None]).scatter(1, index, 0.0), "sa": step, "index": None,
                "outlier": n.gather(1, index)}
    lens, rows = _lengths(case)
    page, hd, rep, kv = case["page"], case["hd"], case["rep"], case["kv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        held = s["table"][i, :(n + page - 1) // page].long()
        for h in range(kv if n else 0):
            k = s["k"][held, h].double()
            v = s["v"][held, h].double()
            if s["ks"] is not None:
                k = k * s["ks"][held, h].double()[:, :, None]
                v = v * s["vs"][held, h].double()[:, None, :]
            k = k.reshape(-1, hd)[:n]
            v = v.transpose(1, 2).reshape(-1, hd)[:n]
            pos = torch.arange(n - r, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = j > pos
            if case["window"]:
                hidden = hidden | (pos - j >= case["window"])
            for e in range(h * rep, (h + 1) * rep):
                z = s["q"][at:at + r, e].double() @ k.T.contiguous() / math.sqrt(hd)
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                out[at:at + r, e] = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ v
        at += r
    return out
