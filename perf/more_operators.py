"""Timed cases of the operators for several continuations of one prompt over the paged cache: the choice of a beam
search's next beams, forked block tables, copies of pages, compaction of the pool, and decode attention that reads a common
prefix once.

A case is a dict of plain values whose "kind" names the entry point:
  beam     the best continuations of each request's beams over the vocabulary (soc_beam_select)
  fork     block table rows that go on from other rows: shared pages, copied pages, freed pages (soc_paged_fork)
  copy     pages copied in all layers of a cache (soc_paged_copy)
  compact  the pages in use brought to the front of the pool (soc_paged_compact)
  shared   one new token of each sequence, groups of sequences with a common prefix (soc_paged_attention_shared)
With `own` true a pass calls the library; otherwise it computes the same in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


def listed():
    return [
        # one user's beam search: a step of four beams
        {"name": "beam 1 x 4", "kind": "beam", "groups": 1, "beams": 4, "vocab": 151936, "dtype": "f32", "top": 8,
         "stops": 1, "temperature": 1.0, "first": False, "masked": False},
        # a small batch in 16 bits whose grammar allows half of the vocabulary, two stop tokens
        {"name": "beam 16 x 4 masked f16", "kind": "beam", "groups": 16, "beams": 4, "vocab": 151936, "dtype": "f16",
         "top": 12, "stops": 2, "temperature": 0.7, "first": False, "masked": True},
        # a full server, eight beams a request
        {"name": "beam 64 x 8", "kind": "beam", "groups": 64, "beams": 8, "vocab": 151936, "dtype": "f32", "top": 16,
         "stops": 1, "temperature": 1.0, "first": False, "masked": False},
        # one user's four beams follow their parents, a thousand tokens into the request
        {"name": "fork 1 x 4", "kind": "fork", "groups": 1, "beams": 4, "page": 16, "longest": 1000, "own_tail": 100,
         "mixed": False},
        # a full server: beams follow their parents, requests end, prompts that begin like another's take over its pages
        {"name": "fork 128 x 8 mixed", "kind": "fork", "groups": 128, "beams": 8, "page": 16, "longest": 4096,
         "own_tail": 600, "mixed": True},
        # the partly filled pages of one user's beams, all layers of a small model
        {"name": "copy 3 partial", "kind": "copy", "copies": 3, "room": 4, "layers": 28, "nkv": 8, "head_dim": 128,
         "page": 16, "partial": True},
        # whole pages moved out of a part of the pool that is to be given up
        {"name": "copy 90 whole", "kind": "copy", "copies": 90, "room": 128, "layers": 4, "nkv": 8, "head_dim": 128,
         "page": 64, "partial": False},
        # a small pool after some of its requests ended
        {"name": "compact 2000", "kind": "compact", "pages": 2000, "n": 32, "page": 64, "used": 0.5, "most": 2000},
        # a server's pool, two thirds in use
        {"name": "compact 131072", "kind": "compact", "pages": 131072, "n": 256, "page": 16, "used": 0.67,
         "most": 131072},
        # one user's four beams behind a prompt of a thousand tokens, a small model
        {"name": "shared 1 x 4", "kind": "shared", "groups": 1, "members": 4, "even": True, "prefix": 1000, "tail": 100,
         "nq": 16, "nkv": 8, "head_dim": 128, "page": 16, "dtype": "f32"},
        # requests with one to eight samples each behind prompts of their own, in 16 bits
        {"name": "shared 24 ragged f16", "kind": "shared", "groups": 24, "members": 8, "even": False, "prefix": 3001,
         "tail": 300, "nq": 32, "nkv": 8, "head_dim": 128, "page": 32, "dtype": "f16"},
        # many users behind one long system prompt
        {"name": "shared 1 x 256", "kind": "shared", "groups": 1, "members": 256, "even": True, "prefix": 4096,
         "tail": 512, "nq": 32, "nkv": 8, "head_dim": 128, "page": 64, "dtype": "f32"},
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v))))


def draw(rng):
    kind = rng.choice(["beam", "beam", "fork", "copy", "compact", "shared", "shared", "shared"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "beam":
        vocab = _spread(rng, 1000, 151936)
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        stops = rng.choice([0, 1, 1, 2])
        return {"kind": kind, "groups": _spread(rng, 1, max(1, min(256, 70000000 // (vocab * beams)))), "beams": beams,
                "vocab": vocab, "dtype": rng.choice(["f32", "f16"]),
                "top": rng.choice([0, beams, min(64, 2 * beams), beams * (1 + stops)]), "stops": stops,
                "temperature": rng.choice([0.7, 1.0, 1.3]), "first": rng.random() < 0.2, "masked": rng.random() < 0.3}
    if kind == "fork":
        longest = _spread(rng, 20, 8192)
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        return {"kind": kind, "groups": _spread(rng, 1, max(1, min(2000, 4000000 // longest) // beams)), "beams": beams,
                "page": page, "longest": longest, "own_tail": _spread(rng, 1, longest), "mixed": rng.random() < 0.6}
    if kind == "copy":
        copies = _spread(rng, 1, 90)
        layers = rng.choice([1, 2, 3, 4, 28]) if page <= 32 and copies <= 24 else rng.choice([1, 2, 3])
        return {"kind": kind, "copies": copies, "room": copies + rng.choice([0, 1, 40]), "layers": layers,
                "nkv": rng.choice([2, 4, 8]), "head_dim": rng.choice([64, 128]), "page": min(page, 64),
                "partial": rng.random() < 0.6}
    if kind == "compact":
        pages = _spread(rng, 40, 131072)
        return {"kind": kind, "pages": pages, "n": _spread(rng, 1, min(1000, pages // 4)), "page": page,
                "used": rng.choice([0.1, 0.5, 0.9]), "most": rng.choice([pages, _spread(rng, 1, pages)])}
    heads = rng.choice([(16, 8), (32, 8), (8, 8), (8, 2), (14, 2), (48, 4)])
    prefix = _spread(rng, 10, 12000)
    members = _spread(rng, 1, 256)
    tail = _spread(rng, 1, 1000)
    return {"kind": kind, "groups": _spread(rng, 1, max(1, min(64, 1000000 // (members * (prefix + tail))))),
            "members": members, "even": rng.random() < 0.4, "prefix": prefix, "tail": tail, "nq": heads[0],
            "nkv": heads[1], "head_dim": rng.choice([64, 128, 128]), "page": page, "dtype": rng.choice(["f32", "f16"])}


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


def _ints(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a).astype(dtype))).cuda()


def _fill(shape, value=-1, dtype=torch.int32):
    return torch.full(shape, value, device="cuda", dtype=dtype)


def _candidates(case):
    """How many of a group's best are looked at: enough that `beams` of them end with no stop token."""
    return max(case["top"], case["beams"] * (1 + case["stops"]))


def _group_sizes(case):
    """Rows of each group, by the case alone."""
    if case["even"]:
        return np.full(case["groups"], case["members"], np.int64)
    r = (np.arange(case["groups"]) * 0.6180339887498949 + 0.37) % 1.0
    return 1 + np.floor(r * case["members"]).astype(np.int64)


def _shared_lengths(case):
    """(prefix of each group, length of each row), by the case alone; ragged cases end with an empty row."""
    sizes = _group_sizes(case)
    n = int(sizes.sum())
    if case["even"]:
        prefix = np.full(sizes.size, case["prefix"], np.int64)
        tail = np.full(n, case["tail"], np.int64)
    else:
        r = (np.arange(sizes.size) * 0.7548776662466927 + 0.11) % 1.0
        prefix = (case["prefix"] // 8 + np.floor(r * (case["prefix"] - case["prefix"] // 8 + 1))).astype(np.int64)
        r = (np.arange(n) * 0.6180339887498949 + 0.73) % 1.0
        tail = 1 + np.floor(r * case["tail"]).astype(np.int64)
    lengths = np.repeat(prefix, sizes) + tail
    if not case["even"] and n > 1:
        lengths[-1] = 0
    return prefix, lengths


def _prepare_beam(case, s, g, r):
    rows, vocab, groups, beams = case["groups"] * case["beams"], case["vocab"], case["groups"], case["beams"]
    x = _normal(g, (rows, vocab), torch.float32, 2.5)
    stops = r.choice(vocab, case["stops"], replace=False).astype(np.int32)
    likely = torch.randint(0, vocab, (rows, 4), generator=g, device="cuda")
    x.scatter_add_(1, likely, 8.0 * torch.rand((rows, 4), generator=g, device="cuda"))
    for t in stops:  # a request that may well be at its end
        x[:, int(t)] += 12.0 * torch.rand(rows, generator=g, device="cuda")
    if case["masked"]:
        x[torch.rand((rows, vocab), generator=g, device="cuda") < 0.5] = -math.inf
    scores = -20.0 * torch.rand((groups, beams), generator=g, device="cuda")
    if case["first"]:  # every beam is the prompt itself: only the first may go on
        scores[:, 0], scores[:, 1:] = 0.0, -math.inf
    s.update(logits=x.to(DTYPES[case["dtype"]]), scores=scores.flatten().contiguous(), stops=[int(t) for t in stops])
    for name, shape in (("top", (groups, case["top"])), ("next", (groups, beams))):
        s[name + "_rows"], s[name + "_tokens"] = _fill(shape), _fill(shape)
        s[name + "_scores"] = _fill(shape, 0.0, torch.float32)


def _prepare_fork(case, s, r):
    """Requests whose beams share their prompt's full pages; a beam's own tail of the same length in all of a request's."""
    groups, beams, page, longest = case["groups"], case["beams"], case["page"], case["longest"]
    n = groups * beams
    width = -(-longest // page) + 1
    tail = min(case["own_tail"], longest)
    at = np.arange(groups)  # lengths by the case alone
    length = tail + np.floor((at * 0.6180339887498949 + 0.37) % 1.0 * (longest + 1 - tail)).astype(np.int64)
    prompt = length - 1 - np.floor((at * 0.7548776662466927 + 0.11) % 1.0 * tail).astype(np.int64)
    shared, held = prompt // page, -(-length // page)
    pages = int((shared + beams * (held - shared)).sum()) + 2 * n + 5
    order = r.permutation(pages).astype(np.int32)
    table, at = np.full((n, width), -1, np.int32), 0
    for g in range(groups):
        own_pages = beams * (held[g] - shared[g])
        rows = table[g * beams: (g + 1) * beams]
        rows[:, : shared[g]] = order[at: at + shared[g]]
        rows[:, shared[g]: held[g]] = order[at + shared[g]: at + shared[g] + own_pages].reshape(beams, -1)
        at += shared[g] + own_pages
    old = np.repeat(length, beams)
    parents = np.arange(n) // beams * beams + r.randint(0, beams, n)
    keep = old[parents]
    if case["mixed"]:
        what = np.repeat(r.permutation(groups) % 8, beams)
        parents[what == 0] = -1  # finished
        keep[what == 0] = 0
        begin = what == 1  # a new request in these rows, whose prompt begins as another's did
        parents[begin] = r.randint(0, n, int(begin.sum()))
        keep[begin] = (old[parents[begin]] * r.rand(int(begin.sum()))).astype(np.int64)
    head = int(r.randint(0, 1 << 40))
    ring = np.full(pages, -1, np.int32)
    ring[(head + np.arange(pages - at)) % pages] = order[at:]
    s.update(parents=_ints(parents), keep=_ints(keep), old=_ints(old), table=_ints(table), ring=_ints(ring),
             cursors=_ints([head, head + pages - at], np.int64), pages=pages)
    s.update(new_table=_fill((n, width)), cursors_out=torch.zeros_like(s["cursors"]), new_lens=_fill((n,)),
             next_lens=_fill((n,)), copies=_fill((n, 3)), count=_fill((1,)), status=_fill((1,)))


def _prepare_copy(case, s, g, r):
    copies, page = case["copies"], case["page"]
    pages = 2 * case["copies"] + 9
    order = r.permutation(pages)
    moves = np.full((case["room"], 3), -1, np.int64)
    moves[:copies, 0], moves[:copies, 1] = order[:copies], order[copies: 2 * copies]
    moves[:copies, 2] = r.randint(1, page, copies) if case["partial"] else page
    shape = (pages, case["nkv"], page, case["head_dim"])
    s["pools"] = [(_normal(g, shape, torch.float16), _normal(g, shape, torch.float16)) for _ in range(case["layers"])]
    s["moves"], s["count"] = _ints(moves), _ints([copies])


def _prepare_compact(case, s, r):
    pages, n, page = case["pages"], case["n"], case["page"]
    used = max(n, int(case["used"] * pages))
    share = 0.2 + (np.arange(n) * 0.6180339887498949 + 0.37) % 1.0  # by the case alone
    held = 1 + (share / share.sum() * (used - n)).astype(np.int64)
    lengths = held * page - r.randint(0, page, n)
    order = r.permutation(pages).astype(np.int32)
    width = int(held.max())
    table = np.full((n, width), -1, np.int32)
    table[np.arange(width)[None, :] < held[:, None]] = order[: held.sum()]
    free = order[held.sum():]
    head = int(r.randint(0, 1 << 40))
    ring = np.full(pages, -1, np.int32)
    ring[(head + np.arange(free.size)) % pages] = free
    most = case["most"]
    s.update(lens=_ints(lengths), table=_ints(table), ring=_ints(ring), held=int(held.sum()),
             cursors=_ints([head, head + free.size], np.int64), new_table=_fill((n, width)), new_ring=_fill((pages,)),
             moves=_fill((most, 3)), count=_fill((1,)), status=_fill((1,)))


def _prepare_shared(case, s, g, r):
    nq, nkv, hd, page = case["nq"], case["nkv"], case["head_dim"], case["page"]
    sizes, (prefix, lengths) = _group_sizes(case), _shared_lengths(case)
    starts = np.concatenate([[0], np.cumsum(sizes)])
    n, dtype = int(starts[-1]), DTYPES[case["dtype"]]
    held, common = -(-lengths // page), np.repeat(prefix // page, sizes)
    width = max(1, int(held.max()))
    # rows of a group name the same full pages of the prefix, then pages of their own
    first = np.concatenate([[0], np.cumsum(prefix // page)])
    mine = np.concatenate([[0], np.cumsum(np.maximum(0, held - common))]) + first[-1]
    pages = int(mine[-1]) + 7
    order = r.permutation(pages).astype(np.int32)
    group = np.repeat(np.arange(sizes.size), sizes)
    at = np.arange(width)[None, :]
    index = np.where(at < common[:, None], first[group][:, None] + at, mine[:-1][:, None] + at - common[:, None])
    table = np.where(at < np.maximum(held, 0)[:, None], order[index.clip(0, pages - 1)], -1)
    s["q"] = _normal(g, (n, nq * hd), dtype)
    s["keys"] = _normal(g, (pages, nkv, page, hd), torch.float16)
    s["values"] = _normal(g, (pages, nkv, page, hd), torch.float16)
    # the page that the prefix ends in: each row has its own copy of what it holds of the prefix
    rows = np.flatnonzero((np.repeat(prefix % page, sizes) > 0) & (lengths > 0))
    copy = _ints(table[rows, common[rows]], np.int64)
    source = _ints(table[starts[group[rows]], common[rows]].clip(0), np.int64)
    place = torch.arange(page, device="cuda")[None, :] < _ints(np.repeat(prefix % page, sizes)[rows])[:, None]
    for pool in (s["keys"], s["values"]):
        pool[copy] = torch.where(place[:, None, :, None], pool[source], pool[copy])
    s.update(table=_ints(table), lengths=_ints(lengths), starts=_ints(starts), prefix=_ints(prefix),
             out=torch.zeros((n, nq * hd), device="cuda", dtype=dtype),
             lse=torch.zeros((n, nq), device="cuda", dtype=torch.float32))


def prepare(case, seed):
    kind, g, r = case["kind"], _generator(seed), np.random.RandomState(seed)
    s = {"case": case}
    if kind == "beam":
        _prepare_beam(case, s, g, r)
    elif kind == "fork":
        _prepare_fork(case, s, r)
    elif kind == "copy":
        _prepare_copy(case, s, g, r)
    elif kind == "compact":
        _prepare_compact(case, s, r)
    else:
        _prepare_shared(case, s, g, r)
    if own:  # the handles that a program keeps
        lib, _ = _library()
        if kind == "copy":
            s["layers"] = lib.PagedLayers([
                lib.PagedCache(k.data_ptr(), v.data_ptr(), k.shape[0], case["page"], case["nkv"], case["head_dim"])
                for k, v in s["pools"]])
        if kind == "shared":
            s["cache"] = lib.PagedCache(s["keys"].data_ptr(), s["values"].data_ptr(), s["keys"].shape[0], case["page"],
                                        case["nkv"], case["head_dim"])
    return s


# ---- one pass: the library's calls -----------------------------------------------------------------------------------
def _beam_outputs(s):
    return {k: s[k] for k in ("top_rows", "top_tokens", "top_scores", "next_rows", "next_tokens", "next_scores")}


def _run_own(s):
    case, kind = s["case"], s["case"]["kind"]
    lib, ctx = _library()
    if kind == "beam":
        top = [s["top_" + k].data_ptr() if case["top"] else None for k in ("rows", "tokens", "scores")]
        lib.beam_select(ctx, s["logits"].data_ptr(), case["dtype"], case["vocab"], case["groups"], case["beams"],
                        case["vocab"], case["temperature"], s["scores"].data_ptr(), s["stops"], case["top"], *top,
                        s["next_rows"].data_ptr(), s["next_tokens"].data_ptr(), s["next_scores"].data_ptr())
        return _beam_outputs(s)
    if kind == "fork":
        n, width = s["table"].shape
        lib.paged_fork(ctx, n, s["parents"].data_ptr(), s["keep"].data_ptr(), s["old"].data_ptr(), case["page"],
                       s["table"].data_ptr(), s["new_table"].data_ptr(), width, width, s["ring"].data_ptr(), s["pages"],
                       s["cursors"].data_ptr(), s["cursors_out"].data_ptr(), s["new_lens"].data_ptr(),
                       s["next_lens"].data_ptr(), s["copies"].data_ptr(), s["count"].data_ptr(),
                       s["status"].data_ptr())
        return {"table": s["new_table"], "ring": s["ring"], "cursors": s["cursors_out"], "new_lens": s["new_lens"],
                "next_lens": s["next_lens"], "copies": s["copies"], "count": s["count"], "status": s["status"]}
    if kind == "copy":
        lib.paged_copy(ctx, s["layers"], s["moves"].data_ptr(), s["count"].data_ptr(), case["room"])
        return [p for pair in s["pools"] for p in pair]
    if kind == "compact":
        n, width = s["table"].shape
        lib.paged_compact(ctx, n, s["lens"].data_ptr(), case["page"], s["table"].data_ptr(), s["new_table"].data_ptr(),
                          width, width, s["ring"].data_ptr(), s["new_ring"].data_ptr(), case["pages"],
                          s["cursors"].data_ptr(), s["moves"].data_ptr(), case["most"], s["count"].data_ptr(),
                          s["status"].data_ptr())
        return {"table": s["new_table"], "ring": s["new_ring"], "moves": s["moves"], "count": s["count"],
                "status": s["status"]}
    width, (n, pages) = case["nq"] * case["head_dim"], s["table"].shape
    lib.paged_attention_shared(ctx, s["cache"], s["q"].data_ptr(), width, case["dtype"], s["table"].data_ptr(), pages,
                               pages, s["lengths"].data_ptr(), n, s["starts"].data_ptr(), s["prefix"].data_ptr(),
                               case["groups"], case["members"], case["prefix"], case["nq"], 0.0, s["out"].data_ptr(),
                               width, s["lse"].data_ptr())
    return {"out": s["out"], "lse": s["lse"]}


# ---- one pass: the plain form ----------------------------------------------------------------------------------------
def _run_beam(s):
    # in 64 bits: beams of nearly the same score stand in their order's borders
    case = s["case"]
    groups, beams, vocab, top = case["groups"], case["beams"], case["vocab"], case["top"]
    many = _candidates(case)
    out = {k: v.clone() for k, v in _beam_outputs(s).items()}
    for g in range(0, groups, 32):  # 32 requests at a time
        rows = slice(g * beams, min(groups, g + 32) * beams)
        x = s["logits"][rows].double()
        x = (x - x.amax(-1, keepdim=True)) / case["temperature"]
        score = x - torch.log(torch.exp(x).sum(-1, keepdim=True)) + s["scores"][rows].double()[:, None]
        score = score.view(-1, beams * vocab)
        best, at = torch.sort(score, dim=-1, descending=True, stable=True)
        best, at = best[:, :many], at[:, :many]
        there = best > -math.inf
        token = torch.where(there, at % vocab, -1)
        first = (torch.arange(g, g + score.shape[0], device=at.device) * beams)[:, None]
        row = torch.where(there, first + at // vocab, -1)
        mine = slice(g, g + score.shape[0])
        out["top_rows"][mine], out["top_tokens"][mine] = row[:, :top].int(), token[:, :top].int()
        out["top_scores"][mine] = best[:, :top].float()
        goes_on = there
        for stop in s["stops"]:
            goes_on = goes_on & (token != stop)
        # those that go on first, in order; what is left of the row stands for none
        place = torch.sort((~goes_on).int(), dim=-1, stable=True).indices[:, :beams]
        some = goes_on.gather(1, place)
        for name, v, none in (("rows", row, -1), ("tokens", token, -1), ("scores", best, -math.inf)):
            v = torch.where(some, v.gather(1, place), none)
            out["next_" + name][mine] = -1 if name != "scores" else -math.inf
            out["next_" + name][mine, : v.shape[1]] = v.to(out["next_" + name].dtype)
    return out


def _run_fork(s):
    case = s["case"]
    page, pages = case["page"], s["pages"]
    parents, keep, old, table = s["parents"].long(), s["keep"].long(), s["old"].long(), s["table"]
    new, ring, copies = s["new_table"].clone(), s["ring"].clone(), s["copies"].clone()
    head, tail = s["cursors"][0], s["cursors"][1]
    n = parents.shape[0]
    row = torch.arange(n, device=table.device)
    live, of = parents >= 0, parents.clamp(min=0)
    length = torch.where(live, keep, 0)
    want, held = (length + page - 1) // page, (old + page - 1) // page
    partial = length % page != 0
    # the parent's own partly filled page stays with the first child that needs it
    heir = partial & (want == held[of]) & (old[of] % page != 0)
    first = torch.full_like(row, n).scatter_reduce(0, of, torch.where(heir, row, n), "amin")
    copied = partial & ~(heir & (first[of] == row))
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    kept = col < want[:, None]
    new[kept] = table[of][kept]
    where = (want - 1).clamp(min=0)
    to = ring[(head + torch.cumsum(copied, 0) - 1) % pages]
    count = copied.sum()
    listed_copies = torch.stack([table[of, where], to, (length % page).int()], -1)[copied]
    copies[: listed_copies.shape[0]] = listed_copies
    new[row[copied], where[copied]] = to[copied]
    # pages that a row let go and no row names now, each where the last row let it go
    named = torch.zeros(pages, dtype=torch.bool, device=table.device)
    named[new[kept].long()] = True
    gone = (col < held[:, None]) & ~(kept & (new == table))
    page_of = table[gone].long()
    order = torch.arange(page_of.shape[0], device=table.device)
    last = torch.full((pages,), -1, dtype=torch.long, device=table.device)
    last.scatter_reduce_(0, page_of, order, "amax")
    back = page_of[~named[page_of] & (last[page_of] == order)]
    ring[(tail + torch.arange(back.shape[0], device=table.device)) % pages] = back.int()
    return {"table": new, "ring": ring, "cursors": torch.stack([head + count, tail + back.shape[0]]),
            "new_lens": length.int(), "next_lens": torch.where(live, length + 1, 0).int(), "copies": copies,
            "count": count.int().view(1), "status": torch.zeros_like(s["status"])}


def _run_copy(s):
    case = s["case"]
    moves = s["moves"][: case["copies"]].long()
    place = torch.arange(case["page"], device=moves.device)[None, :] < moves[:, 2:]
    for pair in s["pools"]:
        for pool in pair:
            moved = torch.where(place[:, None, :, None], pool[moves[:, 0]], pool[moves[:, 1]])
            pool[moves[:, 1]] = moved
    return [p for pair in s["pools"] for p in pair]


def _run_compact(s):
    case = s["case"]
    pages, page = case["pages"], case["page"]
    head, tail = s["cursors"][0], s["cursors"][1]
    ring, table, moves = s["new_ring"].clone(), s["new_table"].clone(), s["moves"].clone()
    many = pages - s["held"]
    spot = (head + torch.arange(many, device=table.device)) % pages
    free = torch.zeros(pages, dtype=torch.bool, device=table.device)
    free[s["ring"][spot].long()] = True
    keep = pages - many  # pages in use, which fill the front
    hole = torch.nonzero(free[:keep])[:, 0]
    high = (keep + torch.nonzero(~free[keep:])[:, 0]).flip(0)
    k = min(case["most"], high.shape[0])
    hole, high = hole[:k], high[:k]
    goes = torch.arange(pages, device=table.device)
    goes[high] = hole
    free[hole], free[high] = False, True
    ring[spot] = torch.nonzero(free)[:, 0].int()
    held = (s["lens"].long() + page - 1) // page
    kept = torch.arange(table.shape[1], device=table.device)[None, :] < held[:, None]
    table[kept] = goes[s["table"][kept].long()].int()
    moves[:k] = torch.stack([high, hole, torch.full_like(hole, page)], -1).int()
    return {"table": table, "ring": ring, "moves": moves, "count": _fill((1,), k), "status": _fill((1,), 0)}


def _run_shared(s):
    case = s["case"]
    nq, nkv, hd, page = case["nq"], case["nkv"], case["head_dim"], case["page"]
    outs, lses = [], []
    n = s["q"].shape[0]
    step = max(1, 600000 // (s["table"].shape[1] * page))  # rows at a time, by the memory they take
    for b in range(0, n, step):
        rows = slice(b, b + step)
        at = s["table"][rows].clamp(min=0).long()
        k = s["keys"][at].permute(0, 2, 4, 1, 3).reshape(at.shape[0], nkv, hd, -1).float()
        v = s["values"][at].permute(0, 2, 1, 3, 4).reshape(at.shape[0], nkv, -1, hd).float()
        q = s["q"][rows].float().view(-1, nkv, nq // nkv, hd)
        seen = (torch.arange(k.shape[-1], device=k.device)[None, :] < s["lengths"][rows][:, None])[:, None, None, :]
        score = (torch.matmul(q, k) / math.sqrt(hd)).masked_fill(~seen, -math.inf)
        top = score.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.exp(score - top)
        total = p.sum(-1, keepdim=True)
        out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
        outs.append(out.reshape(-1, nq * hd).to(s["out"].dtype))
        lses.append((top + torch.log(total)).reshape(-1, nq))
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def run(state):
    if own:
        return _run_own(state)
    return {"beam": _run_beam, "fork": _run_fork, "copy": _run_copy, "compact": _run_compact,
            "shared": _run_shared}[state["case"]["kind"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], 2 if case.get("dtype") == "f16" else 4
    if kind == "beam":
        logits = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": size * logits + case["groups"] * (16 * case["beams"] + 12 * case["top"]), "flops": 4 * logits}
    if kind == "fork":  # three words in, two out a row; about three quarters of the longest row's entries in and out
        n = case["groups"] * case["beams"]
        return {"bytes": n * (20 + 8 * (3 * case["longest"] // (4 * case["page"]) + 1)), "flops": 0}
    if kind == "copy":  # a partial page is half full on average
        page = case["nkv"] * case["page"] * case["head_dim"] * (1 if case["partial"] else 2)
        return {"bytes": 12 * case["copies"] + 4 * case["copies"] * case["layers"] * page, "flops": 0}
    if kind == "compact":  # free pages in and out, table entries in and out, moves
        used = max(case["n"], int(case["used"] * case["pages"]))
        free = case["pages"] - used
        moved = min(case["most"], used * free // case["pages"])
        return {"bytes": 8 * free + 8 * used + 4 * case["n"] + 12 * moved, "flops": 0}
    prefix, lengths = _shared_lengths(case)
    sizes = _group_sizes(case)
    q = case["nq"] * case["head_dim"]
    tails = np.maximum(0, lengths - np.repeat(prefix, sizes))
    keys = int(prefix.sum() + tails.sum())
    return {"bytes": keys * 4 * case["nkv"] * case["head_dim"] + lengths.size * (2 * size * q + 4 * case["nq"] + 4),
            "flops": 4 * int(lengths.sum()) * q}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    kind = case["kind"]
    if kind not in ("beam", "shared"):
        return None  # page ids, lengths, and values that are only moved
    s = prepare(case, seed)
    if kind == "beam":
        groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
        top, following = [], []
        for g in range(groups):
            rows = slice(g * beams, (g + 1) * beams)
            z = torch.log_softmax(s["logits"][rows].double() / case["temperature"], -1) + \
                s["scores"][rows].double()[:, None]
            top.append(torch.topk(z.flatten(), case["top"]).values)
            z[:, s["stops"]] = -math.inf
            following.append(torch.topk(z.flatten(), beams).values)
        return {"top_rows": None, "top_tokens": None, "top_scores": torch.stack(top), "next_rows": None,
                "next_tokens": None, "next_scores": torch.stack(following)}
    nq, nkv, hd = case["nq"], case["nkv"], case["head_dim"]
    lengths = s["lengths"].tolist()
    if sum(lengths) > 4000000:
        return None
    out = torch.zeros((len(lengths), nq, hd), device="cuda", dtype=torch.float64)
    lse = torch.full((len(lengths), nq), -math.inf, device="cuda", dtype=torch.float64)
    for b, length in enumerate(lengths):
        if length == 0:
            continue
        mine = s["table"][b, : -(-length // case["page"])].long()
        k, v = (s[x][mine].double().transpose(0, 1).reshape(nkv, -1, hd)[:, :length].contiguous()
                for x in ("keys", "values"))
        q = s["q"][b].double().view(nkv, nq // nkv, hd)
        z = torch.bmm(q, k.transpose(1, 2).contiguous()) * hd ** -0.5
        lse[b] = torch.logsumexp(z, -1).flatten()
        out[b] = torch.bmm(torch.softmax(z, -1), v).reshape(nq, hd)
    return {"out": out.flatten(1), "lse": lse}
