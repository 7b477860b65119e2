"""Timed cases of the paged serving operators: rotary positions, page planning, the paged cache's append, decode
attention over a paged cache, and token log probabilities.

A case is a dict of plain values whose "kind" names the entry point:
  rope      rotary positions of given rows: half or interleaved pairs, part of the head, scaled (soc_rope_apply)
  plan      pages, slots and positions of a step from the requests' lengths before and after it (soc_paged_plan)
  append    rotary positions of new queries and keys, keys and values into their slots (soc_paged_append)
  attn      one new token of each sequence over its pages (soc_paged_attention_decode)
  logprobs  log probability and rank of given tokens, entropy, top alternatives (soc_logprobs)
With `own` true a pass calls the library; otherwise it computes the same in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # the rotary step of a batch of 64 users deep in long conversations, queries as a view of the fused projection
        {"name": "rope 64 yarn f32", "kind": "rope", "rows": 64, "heads": 32, "head_dim": 128, "rotary_dim": 128,
         "layout": "half", "scaling": "yarn", "factor": 4.0, "dtype": "f32", "longest": 131072, "pad": 2048},
        # a long prompt's queries in 16 bits, half of each head rotated in interleaved pairs, an odd number of rows
        {"name": "rope 4093 part f16", "kind": "rope", "rows": 4093, "heads": 16, "head_dim": 128, "rotary_dim": 64,
         "layout": "interleaved", "scaling": "ntk", "factor": 2.0, "dtype": "f16", "longest": 40960, "pad": 0},
        # the plan of a plain decode step: every request one token longer
        {"name": "plan decode 64", "kind": "plan", "n": 64, "page": 16, "longest": 4096, "max_rows": 64,
         "mixed": False},
        # a busy server's step: decodes, prompts, chunks of prompts, finished and rolled back requests
        {"name": "plan mixed 1000", "kind": "plan", "n": 1000, "page": 16, "longest": 8192, "max_rows": 32768,
         "mixed": True},
        # the cache write of a decode batch out of its fused fp32 projection, one row a page
        {"name": "append decode 48", "kind": "append", "rows": 48, "nq": 32, "nkv": 8, "head_dim": 128, "page": 16,
         "rotary_dim": 128, "layout": "half", "dtype": "f32", "prompt": False, "longest": 40960},
        # a step of several prompts, odd in number, rows of padding at its end
        {"name": "append prompts 2531", "kind": "append", "rows": 2531, "nq": 16, "nkv": 8, "head_dim": 128,
         "page": 64, "rotary_dim": 128, "layout": "half", "dtype": "f32", "prompt": True, "longest": 40960},
        # one user late in a long conversation
        {"name": "attention 1 x 4071", "kind": "attn", "n": 1, "longest": 4071, "even": True, "nq": 32, "nkv": 8,
         "head_dim": 128, "page": 16, "dtype": "f32"},
        # a small model's batch of ragged lengths, one request still empty
        {"name": "attention 48 ragged", "kind": "attn", "n": 48, "longest": 1500, "even": False, "nq": 16, "nkv": 8,
         "head_dim": 128, "page": 32, "dtype": "f16"},
        # a full server: long ragged sequences that fill gigabytes of cache
        {"name": "attention 200 ragged", "kind": "attn", "n": 200, "longest": 8192, "even": False, "nq": 32, "nkv": 8,
         "head_dim": 128, "page": 64, "dtype": "f32"},
        # the log probability of each generated token with its alternatives, one user
        {"name": "logprobs 1 top 20", "kind": "logprobs", "rows": 1, "vocab": 151936, "dtype": "f32", "top": 20,
         "temperature": 1.0, "masked": False},
        # the same for a batch whose grammar allows half of the vocabulary, in 16 bits
        {"name": "logprobs 64 masked f16", "kind": "logprobs", "rows": 64, "vocab": 151936, "dtype": "f16", "top": 5,
         "temperature": 0.7, "masked": True},
        # scoring a document: every position's token
        {"name": "logprobs 777 top 8", "kind": "logprobs", "rows": 777, "vocab": 151936, "dtype": "f32", "top": 8,
         "temperature": 1.0, "masked": False},
    ]


def _spread(rng, lo, hi, step=1):
    """A size between lo and hi, even over its logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["rope", "plan", "append", "attn", "attn", "logprobs", "logprobs"])
    dtype = rng.choice(["f32", "f16"])
    if kind == "rope":
        head_dim = rng.choice([64, 80, 128, 128, 256])
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return {"kind": kind, "rows": _spread(rng, 1, 8000), "heads": rng.choice([1, 8, 16, 32, 40]),
                "head_dim": head_dim, "rotary_dim": rng.choice([head_dim, head_dim // 2, head_dim // 4]),
                "layout": rng.choice(["half", "interleaved"]), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]), "dtype": dtype,
                "longest": _spread(rng, 1000, 1000000), "pad": rng.choice([0, 8, 2048])}
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        n = _spread(rng, 1, 2000)
        mixed = rng.random() < 0.7
        return {"kind": kind, "n": n, "page": page, "longest": _spread(rng, 100, 8192),
                "max_rows": n + _spread(rng, 100, 32000) if mixed else n, "mixed": mixed}
    heads = rng.choice([(16, 8), (32, 8), (8, 8), (8, 2), (14, 2), (48, 4)])
    if kind == "append":
        prompt = rng.random() < 0.5
        head_dim = rng.choice([64, 128, 128])
        return {"kind": kind, "rows": _spread(rng, 1, 6000) if prompt else _spread(rng, 1, 512), "nq": heads[0],
                "nkv": heads[1], "head_dim": head_dim, "page": page,
                "rotary_dim": rng.choice([head_dim, head_dim, head_dim // 2]),
                "layout": rng.choice(["half", "interleaved"]), "dtype": dtype, "prompt": prompt,
                "longest": _spread(rng, 1000, 100000)}
    if kind == "attn":
        longest = _spread(rng, 1, 40000)
        return {"kind": kind, "n": _spread(rng, 1, max(1, min(512, 600000 // longest))), "longest": longest,
                "even": rng.random() < 0.3, "nq": heads[0], "nkv": heads[1], "head_dim": rng.choice([64, 128, 128]),
                "page": page, "dtype": dtype}
    vocab = _spread(rng, 1000, 151936)
    return {"kind": kind, "rows": _spread(rng, 1, min(2000, 100000000 // vocab)), "vocab": vocab, "dtype": dtype,
            "top": rng.choice([0, 1, 5, 8, 20, 33, 64]), "temperature": rng.choice([0.6, 0.7, 1.0]),
            "masked": rng.random() < 0.3}


# ---- inputs ----------------------------------------------------------------------------------------------------------
_ctx = None


def _library():
    """The library's Python package and the program's one device context."""
    global _ctx
    import soc_amd
    if _ctx is None:
        _ctx = soc_amd.Context(0)
    return soc_amd, _ctx


DTYPES = {"f32": torch.float32, "f16": torch.float16}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * sigma).to(dtype)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _lengths(case):
    """The sequences' lengths, by the case alone: all `longest`, or spread between a 64th of it and all of it, the last
    of them empty."""
    n, top = case["n"], case["longest"]
    if case["even"]:
        return np.full(n, top, np.int64)
    low = max(1, top // 64)
    r = (np.arange(n) * 0.6180339887498949 + 0.37) % 1.0
    lengths = low + np.floor(r * (top + 1 - low)).astype(np.int64)
    if n > 1:
        lengths[-1] = 0
    return lengths


def _table(r, lengths, page, spare=7):
    """Distinct pages in random order for sequences of these lengths: (table [n][widest], pages in the cache, those in
    nobody's hands)."""
    held = -(-lengths // page)
    pages = int(held.sum()) + spare
    order = r.permutation(pages).astype(np.int32)
    width = max(1, int(held.max()))
    table = np.full((lengths.size, width), -1, np.int32)
    table[np.arange(width)[None, :] < held[:, None]] = order[: pages - spare]
    return table, pages, order[pages - spare:]


def _plan_lengths(case, r):
    """Lengths before and after a step of `n` requests that adds at most max_rows tokens."""
    n, top = case["n"], case["longest"]
    old = r.randint(1, top, n)
    new = old + 1
    if case["mixed"]:
        what = r.permutation(n) % 10
        prompts = np.flatnonzero(what == 0)
        most = max(1, (case["max_rows"] - n) // max(1, prompts.size))
        old[prompts] = np.where(r.rand(prompts.size) < 0.7, 0, old[prompts])  # new, or the next chunk of a long one
        new[prompts] = np.minimum(top, old[prompts] + r.randint(1, most + 1, prompts.size))
        new[what == 1] = 0  # finished
        back = what == 2  # proposed tokens that were not taken
        new[back] = np.maximum(1, old[back] - r.randint(0, 9, int(back.sum())))
    return old.astype(np.int64), new.astype(np.int64)


def prepare(case, seed):
    kind, g, r = case["kind"], _generator(seed), np.random.RandomState(seed)
    s = {"case": case}
    if kind == "rope":
        rows, width, dtype = case["rows"], case["heads"] * case["head_dim"], DTYPES[case["dtype"]]
        s["x"] = _normal(g, (rows, width + case["pad"]), dtype)
        s["y"] = torch.zeros((rows, width), device="cuda", dtype=dtype)
        s["positions"] = _ints(r.randint(0, case["longest"], rows).astype(np.int32))
    elif kind == "plan":
        old, new = _plan_lengths(case, r)
        page, width = case["page"], -(-case["longest"] // case["page"]) + 1
        held = -(-old // page)
        pages = case["n"] * width  # a cache that holds every request at its longest
        order = r.permutation(pages).astype(np.int32)
        table = np.full((case["n"], width), -1, np.int32)
        table[np.arange(width)[None, :] < held[:, None]] = order[: int(held.sum())]
        free = order[int(held.sum()):]
        head = int(r.randint(0, 1 << 40))  # pages taken since the server began
        ring = np.full(pages, -1, np.int32)
        ring[(head + np.arange(free.size)) % pages] = free
        s.update(old=_ints(old.astype(np.int32)), new=_ints(new.astype(np.int32)), table=_ints(table),
                 ring=_ints(ring), cursors=_ints(np.array([head, head + free.size], np.int64)), pages=pages)
        s["cursors_out"] = torch.zeros_like(s["cursors"])
        s["starts"] = torch.zeros(case["n"] + 1, device="cuda", dtype=torch.int32)
        s["positions"] = torch.zeros(case["max_rows"], device="cuda", dtype=torch.int32)
        s["slots"] = torch.zeros(case["max_rows"], device="cuda", dtype=torch.int32)
        s["status"] = torch.zeros(1, device="cuda", dtype=torch.int32)
    elif kind == "append":
        rows, nq, nkv, hd, page = (case[k] for k in ("rows", "nq", "nkv", "head_dim", "page"))
        dtype = DTYPES[case["dtype"]]
        s["qkv"] = _normal(g, (rows, (nq + 2 * nkv) * hd), dtype)
        if case["prompt"]:  # consecutive slots of pages in any order
            pages = -(-rows // page) + 5
            at = np.arange(rows)
            slots = r.permutation(pages)[at // page] * page + at % page
            slots[rows - rows // 50:] = -1  # padding
        else:
            pages = rows + 5
            slots = r.permutation(pages)[:rows] * page + r.randint(0, page, rows)
        s["keys"] = _normal(g, (pages, nkv, page, hd), torch.float16)
        s["values"] = _normal(g, (pages, nkv, page, hd), torch.float16)
        s["q"] = torch.zeros((rows, nq * hd), device="cuda", dtype=dtype)
        s["slots"] = _ints(slots.astype(np.int32))
        s["positions"] = _ints(r.randint(0, case["longest"], rows).astype(np.int32))
    elif kind == "attn":
        n, nq, nkv, hd, page = (case[k] for k in ("n", "nq", "nkv", "head_dim", "page"))
        lengths = _lengths(case)
        table, pages, _ = _table(r, lengths, page)
        s["q"] = _normal(g, (n, nq * hd), DTYPES[case["dtype"]])
        s["keys"] = _normal(g, (pages, nkv, page, hd), torch.float16)
        s["values"] = _normal(g, (pages, nkv, page, hd), torch.float16)
        s["table"], s["lengths"] = _ints(table), _ints(lengths.astype(np.int32))
        s["out"] = torch.zeros((n, nq * hd), device="cuda", dtype=DTYPES[case["dtype"]])
        s["lse"] = torch.zeros((n, nq), device="cuda", dtype=torch.float32)
    else:
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        x = _normal(g, (rows, vocab), torch.float32, 2.5)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        x.scatter_add_(1, tokens[:, None], 8.0 * torch.rand((rows, 1), generator=g, device="cuda"))
        if case["masked"]:
            x[torch.rand((rows, vocab), generator=g, device="cuda") < 0.5] = -math.inf
        s["logits"] = x.to(DTYPES[case["dtype"]])
        s["tokens"] = tokens.to(torch.int32)
        for name, dtype in (("logprobs", torch.float32), ("entropy", torch.float32), ("ranks", torch.int32)):
            s[name] = torch.zeros(rows, device="cuda", dtype=dtype)
        s["top_ids"] = torch.zeros((rows, top), device="cuda", dtype=torch.int32)
        s["top_logprobs"] = torch.zeros((rows, top), device="cuda", dtype=torch.float32)
    if own:  # the handles that a program keeps
        lib, ctx = _library()
        if kind in ("rope", "append"):
            s["rope"] = lib.Rope(ctx, case["head_dim"], case["rotary_dim"], layout=case["layout"], theta=1e6,
                                 scaling=case.get("scaling", "none"), factor=case.get("factor", 1.0),
                                 original_max_position=32768)
        if kind in ("append", "attn"):
            s["cache"] = lib.PagedCache(s["keys"].data_ptr(), s["values"].data_ptr(), s["keys"].shape[0], case["page"],
                                        case["nkv"], case["head_dim"])
    return s


# ---- one pass: the library's calls -----------------------------------------------------------------------------------
def _run_own(s):
    case, kind = s["case"], s["case"]["kind"]
    lib, ctx = _library()
    if kind == "rope":
        width = case["heads"] * case["head_dim"]
        s["rope"].apply(s["x"].data_ptr(), s["y"].data_ptr(), case["dtype"], case["rows"], case["heads"],
                        positions=s["positions"].data_ptr(), x_stride=width + case["pad"], y_stride=width)
        return s["y"]
    if kind == "plan":
        lib.paged_plan(ctx, case["n"], s["old"].data_ptr(), s["new"].data_ptr(), case["page"], s["table"].data_ptr(),
                       s["table"].shape[1], s["table"].shape[1], s["ring"].data_ptr(), s["pages"],
                       s["cursors"].data_ptr(), s["cursors_out"].data_ptr(), s["starts"].data_ptr(),
                       s["positions"].data_ptr(), s["slots"].data_ptr(), case["max_rows"], s["status"].data_ptr())
        return {"table": s["table"], "ring": s["ring"], "cursors": s["cursors_out"], "starts": s["starts"],
                "positions": s["positions"], "slots": s["slots"], "status": s["status"]}
    if kind == "append":
        nq, nkv, hd = case["nq"], case["nkv"], case["head_dim"]
        base, size, row = s["qkv"].data_ptr(), s["qkv"].element_size(), (nq + 2 * nkv) * hd
        lib.paged_append(ctx, s["cache"], s["rope"], base, row, base + nq * hd * size, row,
                         base + (nq + nkv) * hd * size, row, case["dtype"], s["q"].data_ptr(), nq * hd, case["rows"],
                         nq, s["positions"].data_ptr(), s["slots"].data_ptr())
        return {"q": s["q"], "keys": s["keys"], "values": s["values"]}
    if kind == "attn":
        width = case["nq"] * case["head_dim"]
        lib.paged_attention_decode(ctx, s["cache"], s["q"].data_ptr(), width, case["dtype"], s["table"].data_ptr(),
                                   s["table"].shape[1], s["table"].shape[1], s["lengths"].data_ptr(), case["n"],
                                   case["nq"], 0.0, s["out"].data_ptr(), width, s["lse"].data_ptr())
        return {"out": s["out"], "lse": s["lse"]}
    lib.logprobs(ctx, s["logits"].data_ptr(), case["dtype"], case["vocab"], case["rows"], case["vocab"],
                 case["temperature"], s["tokens"].data_ptr(), s["logprobs"].data_ptr(), s["ranks"].data_ptr(),
                 s["entropy"].data_ptr(), case["top"], s["top_ids"].data_ptr() if case["top"] else None,
                 s["top_logprobs"].data_ptr() if case["top"] else None)
    return {k: s[k] for k in ("logprobs", "ranks", "entropy", "top_ids", "top_logprobs")}


# ---- one pass: the plain form ----------------------------------------------------------------------------------------
def _frequencies(case, device):
    """Radians a position of each pair, and what cosines and sines are multiplied by (64 bits)."""
    d, theta, factor, scaling = case["rotary_dim"], 1e6, case.get("factor", 1.0), case.get("scaling", "none")
    if scaling == "ntk":
        theta = theta * factor ** (d / (d - 2))
    i = torch.arange(d // 2, device=device, dtype=torch.float64)
    f = theta ** (-2.0 * i / d)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        def border(turns):
            return d * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(0, math.floor(border(32.0))), min(d - 1, math.ceil(border(1.0)))
        ramp = ((i - low) / (high - low if high > low else 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    return f, 1.0


def _rotate(x, positions, case):
    """x [rows][heads][head_dim] in 32 bits, rotated."""
    f, m = _frequencies(case, x.device)
    a = positions.to(torch.float64)[:, None, None] * f
    c, s = (torch.cos(a) * m).float(), (torch.sin(a) * m).float()
    d = case["rotary_dim"]
    if case["layout"] == "half":
        u, v = x[..., : d // 2], x[..., d // 2: d]
        turned = torch.cat([u * c - v * s, v * c + u * s], -1)
    else:
        u, v = x[..., 0:d:2], x[..., 1:d:2]
        turned = torch.stack([u * c - v * s, v * c + u * s], -1).flatten(-2)
    return torch.cat([turned, x[..., d:]], -1)


def _run_plan(s):
    case = s["case"]
    page, pages, most = case["page"], s["pages"], case["max_rows"]
    old, new, table, ring = s["old"].long(), s["new"].long(), s["table"].clone(), s["ring"].clone()
    head, tail = s["cursors"][0], s["cursors"][1]
    held, want = (old + page - 1) // page, (new + page - 1) // page
    take, give, add = (want - held).clamp(min=0), (held - want).clamp(min=0), (new - old).clamp(min=0)
    width = torch.arange(table.shape[1], device=table.device)[None, :]
    taken = (width >= held[:, None]) & (width < want[:, None])
    given = (width >= want[:, None]) & (width < held[:, None])
    table[taken] = ring[(head + torch.arange(int(take.sum()), device=table.device)) % pages]
    back = s["table"][given]
    ring[(tail + torch.arange(back.shape[0], device=table.device)) % pages] = back
    ends = torch.cumsum(add, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    row = torch.arange(most, device=table.device)
    who = torch.searchsorted(ends, row, right=True).clamp(max=case["n"] - 1)
    live = row < ends[-1]
    position = torch.where(live, old[who] + row - starts[who], 0)
    slot = table[who, position // page].long() * page + position % page
    return {"table": table, "ring": ring, "cursors": torch.stack([head + take.sum(), tail + give.sum()]),
            "starts": starts.int(), "positions": position.int(), "slots": torch.where(live, slot, -1).int(),
            "status": torch.zeros_like(s["status"])}


def _run_append(s):
    case = s["case"]
    nq, nkv, hd, page = case["nq"], case["nkv"], case["head_dim"], case["page"]
    rows = s["qkv"].float().view(case["rows"], nq + 2 * nkv, hd)
    turned = _rotate(rows[:, : nq + nkv], s["positions"], case)
    live = s["slots"] >= 0
    slots = s["slots"][live].long()
    s["q"][live] = turned[:, :nq].flatten(1).to(s["q"].dtype)[live]
    s["keys"][slots // page, :, slots % page] = turned[:, nq:].half()[live]
    s["values"][slots // page, :, slots % page] = rows[:, nq + nkv:].half()[live]
    return {"q": s["q"], "keys": s["keys"], "values": s["values"]}


def _run_attn(s):
    case = s["case"]
    n, nq, nkv, hd = case["n"], case["nq"], case["nkv"], case["head_dim"]
    at = s["table"].clamp(min=0).long()
    k = s["keys"][at].permute(0, 2, 4, 1, 3).reshape(n, nkv, hd, -1).float()
    v = s["values"][at].permute(0, 2, 1, 3, 4).reshape(n, nkv, -1, hd).float()
    q = s["q"].float().view(n, nkv, nq // nkv, hd)
    seen = (torch.arange(k.shape[-1], device=k.device)[None, :] < s["lengths"][:, None])[:, None, None, :]
    score = (torch.matmul(q, k) / math.sqrt(hd)).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.masked_fill(~seen[:, :, 0, :, None], 0.0)) / torch.where(total > 0, total, 1.0)
    return {"out": out.reshape(n, nq * hd).to(s["out"].dtype), "lse": (top + torch.log(total)).reshape(n, nq)}


def _run_logprobs(s):
    case = s["case"]
    raw = s["logits"].float()
    x = raw / case["temperature"]
    t = s["tokens"].long()[:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    norm = top + torch.log(total)
    mean = (e * torch.where(e > 0, x - top, 0.0)).sum(-1, keepdim=True) / total
    mine = raw.gather(1, t)
    before = torch.arange(case["vocab"], device=raw.device)[None, :] < t
    ranks = ((raw > mine) | ((raw == mine) & before)).sum(-1)
    best, ids = torch.sort(raw, dim=-1, descending=True, stable=True)
    k = case["top"]
    return {"logprobs": (x.gather(1, t) - norm)[:, 0], "ranks": ranks.int(),
            "entropy": (torch.log(total) - mean)[:, 0], "top_ids": ids[:, :k].int().contiguous(),
            "top_logprobs": best[:, :k] / case["temperature"] - norm}


def run(state):
    if own:
        return _run_own(state)
    case, kind = state["case"], state["case"]["kind"]
    if kind == "rope":
        x = state["x"][:, : case["heads"] * case["head_dim"]].float().view(case["rows"], case["heads"], -1)
        return _rotate(x, state["positions"], case).flatten(1).to(state["y"].dtype)
    return {"plan": _run_plan, "append": _run_append, "attn": _run_attn, "logprobs": _run_logprobs}[kind](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], 2 if case.get("dtype") == "f16" else 4
    if kind == "rope":
        values = case["rows"] * case["heads"] * case["head_dim"]
        return {"bytes": 2 * size * values + 4 * case["rows"], "flops": 3 * values}
    if kind == "plan":  # lengths in; starts, positions and slots out; about one table entry a page of new rows
        n, rows = case["n"], case["max_rows"]
        return {"bytes": 8 * n + 4 * (n + 1) + 8 * rows + 8 * (rows // case["page"] + 1), "flops": 0}
    if kind == "append":
        rows, q, kv = case["rows"], case["nq"] * case["head_dim"], case["nkv"] * case["head_dim"]
        return {"bytes": rows * (size * (2 * q + 2 * kv) + 4 * kv + 8), "flops": 3 * rows * (q + kv)}
    if kind == "attn":
        keys, q = int(_lengths(case).sum()), case["nq"] * case["head_dim"]
        return {"bytes": keys * (4 * case["nkv"] * case["head_dim"] + 4 / case["page"]) +
                case["n"] * (2 * size * q + 4 * case["nq"] + 4),
                "flops": 4 * keys * q}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (size * vocab + 16 + 8 * case["top"]), "flops": 4 * rows * vocab}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None

    def turned(x, positions):
        """x [rows][heads][head_dim] with every pair (a, b) as (a cos t - b sin t, b cos t + a sin t)."""
        d, y = case["rotary_dim"], x.clone()
        base, factor, scaling, gain = 1e6, case.get("factor", 1.0), case.get("scaling", "none"), 1.0
        wave = [base ** (2.0 * i / d) for i in range(d // 2)]  # positions a radian
        if scaling == "linear":
            wave = [w * factor for w in wave]
        elif scaling == "ntk":
            wave = [(base * factor ** (d / (d - 2.0))) ** (2.0 * i / d) for i in range(d // 2)]
        elif scaling == "yarn":
            gain = 1.0 + math.log(factor) / 10.0
            first = max(0, math.floor(d / 2 * math.log(32768 / (32.0 * 2 * math.pi), base)))
            last = min(d - 1, math.ceil(d / 2 * math.log(32768 / (2 * math.pi), base)))
            for i in range(d // 2):
                share = min(1.0, max(0.0, (i - first) / (last - first)))  # of the stretched wave
                wave[i] = 1.0 / (share / (factor * wave[i]) + (1.0 - share) / wave[i])
        for i in range(d // 2):
            a, b = (i, i + d // 2) if case["layout"] == "half" else (2 * i, 2 * i + 1)
            t = (positions.double() / wave[i])[:, None]
            y[..., a] = gain * (x[..., a] * torch.cos(t) - x[..., b] * torch.sin(t))
            y[..., b] = gain * (x[..., b] * torch.cos(t) + x[..., a] * torch.sin(t))
        return y

    s = prepare(case, seed)
    if kind == "rope":
        x = s["x"][:, : case["heads"] * case["head_dim"]].double().reshape(case["rows"], case["heads"], -1)
        return turned(x, s["positions"]).flatten(1)
    if kind == "append":
        nq, nkv, hd, page = case["nq"], case["nkv"], case["head_dim"], case["page"]
        x = s["qkv"].double().view(case["rows"], -1, hd)
        y = turned(x[:, : nq + nkv], s["positions"])
        q, keys, values = s["q"].double(), s["keys"].double(), s["values"].double()
        for r, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                q[r] = y[r, :nq].flatten()
                keys[slot // page, :, slot % page] = y[r, nq:]
                values[slot // page, :, slot % page] = x[r, nq + nkv:]
        return {"q": q, "keys": keys, "values": values}
    if kind == "attn":
        nq, nkv, hd, page = case["nq"], case["nkv"], case["head_dim"], case["page"]
        out = torch.zeros((case["n"], nq, hd), device="cuda", dtype=torch.float64)
        lse = torch.full((case["n"], nq), -math.inf, device="cuda", dtype=torch.float64)
        for b, length in enumerate(s["lengths"].tolist()):
            if length == 0:
                continue
            mine = s["table"][b, : -(-length // page)].long()
            k, v = (s[x][mine].double().transpose(0, 1).reshape(nkv, -1, hd)[:, :length].contiguous()
                    for x in ("keys", "values"))
            q = s["q"][b].double().view(nkv, nq // nkv, hd)
            score = torch.bmm(q, k.transpose(1, 2).contiguous()) * hd ** -0.5
            lse[b] = torch.logsumexp(score, -1).flatten()
            out[b] = torch.bmm(torch.softmax(score, -1), v).reshape(nq, hd)
        return {"out": out.flatten(1), "lse": lse}
    logprobs, entropy, best = [], [], []
    for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double() / case["temperature"]
        lp = torch.log_softmax(x, -1)
        logprobs.append(lp.gather(1, t.long()[:, None])[:, 0])
        entropy.append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(-1))
        best.append(torch.topk(lp, case["top"], dim=-1).values)
    return {"logprobs": torch.cat(logprobs), "ranks": None, "entropy": torch.cat(entropy), "top_ids": None,
            "top_logprobs": torch.cat(best)}
