"""A beam search by the library's calls alone, several requests at a time, against one in Python: the model is a seeded one of
one layer over a paged cache, so that a page that went to the wrong beam, or was copied, freed or moved wrongly, changes what a
later step attends to. Steps are queued one behind the other without reading anything back; every eighth step the pool is
compacted. The host's search follows the beams' tokens by itself and computes each step from whole sequences in 64 bits.

Beams are compared by their scores (the attention of a step is off by about 1e-6 of the values, the logits by as much, a step's
score by 2e-5 at most, and errors add over the steps), and their sequences wherever the next candidate's score is further away
than that."""
import math

import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import check, lib
from tests.device import Arrays

pytestmark = pytest.mark.gpu


class Model:
    """Embedding -> q, k, v -> attention -> logits; keys are not rotated."""

    def __init__(self, vocab, nq, nkv, hd, seed):
        rng = np.random.default_rng(seed)
        self.vocab, self.nq, self.nkv, self.hd = vocab, nq, nkv, hd
        self.q, self.k, self.v = (rng.standard_normal((vocab, h * hd)).astype(np.float32) for h in (nq, nkv, nkv))
        self.head = (0.25 * rng.standard_normal((nq * hd, vocab)) / math.sqrt(hd)).astype(np.float32)

    def logits(self, tokens):
        k, v = (x[tokens].astype(np.float16).astype(np.float64).reshape(len(tokens), self.nkv, self.hd) for x in (self.k, self.v))
        q = self.q[tokens[-1]].astype(np.float64).reshape(self.nkv, -1, self.hd)
        z = np.einsum("ghd,tgd->ght", q, k) / math.sqrt(self.hd)
        p = np.exp(z - z.max(-1, keepdims=True))
        out = np.einsum("ght,tgd->ghd", p / p.sum(-1, keepdims=True), v)
        return 8.0 * (out.reshape(-1) @ self.head.astype(np.float64))


def host_search(model, prompt, beams, steps, stops):
    """The live beams after `steps` steps, and how far the nearest rival was from changing them."""
    live, gap = [(0.0, list(prompt))], np.inf
    for _ in range(steps):
        cands = []
        for b, (score, tokens) in enumerate(live):
            z = model.logits(tokens)
            lp = z - z.max() - np.log(np.exp(z - z.max()).sum())
            cands += [(score + lp[t], b, t) for t in range(model.vocab) if t not in stops]
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        best = cands[: beams + 1]
        gap = min([gap] + [best[i][0] - best[i + 1][0] for i in range(len(best) - 1)])
        live = [(s, live[b][1] + [t]) for s, b, t in best[:beams]]
    return live, gap


@pytest.mark.parametrize("page,hd,nq,nkv,always", [(16, 64, 4, 2, True), (32, 128, 8, 2, True), (16, 128, 2, 2, False)])
def test_beam_search_of_several_requests(gpu_ctx, page, hd, nq, nkv, always, monkeypatch):
    if always:
        monkeypatch.setenv("SOC_PAGED_SHARED", "always")
    ctx, rng = gpu_ctx, np.random.default_rng(17)
    model = Model(97, nq, nkv, hd, 5)
    groups, beams, steps, width, pages, stops = 3, 4, 20, 16, 130, [11, 60]
    prompts = [rng.integers(0, 97, n).tolist() for n in (150, 133, 40)]
    n, qw, kw, max_rows = groups * beams, nq * hd, nkv * hd, 400
    with Arrays(ctx) as mem:
        z = lambda *s, t=np.int32: mem.up(np.zeros(s, t))  # noqa: E731
        tables = [mem.up(np.full((n, width), -1, np.int32)) for _ in range(2)]
        ring, cursors = mem.up(rng.permutation(pages).astype(np.int32)), mem.up(np.array([0, pages], np.int64))
        pk, pv = (mem.up(np.full((pages, nkv, page, hd), np.nan, np.float16)) for _ in range(2))
        cache = S.PagedCache(pk, pv, pages, page, nkv, hd)
        layers, rope = S.PagedLayers([cache]), None
        eq, ek, ev, head = (mem.up(x) for x in (model.q, model.k, model.v, model.head))
        starts, positions, slots, lens, old, new = z(n + 1), z(max_rows), z(max_rows), z(n), z(n), z(n)
        status, copies, count, moves, moved = [z(1) for _ in range(60)], z(n, 3), z(1), z(pages, 3), z(1)
        q, out, logits = z(n, qw, t=np.float32), z(n, qw, t=np.float32), z(n, 97, t=np.float32)
        k, v = z(max_rows, kw, t=np.float32), z(max_rows, kw, t=np.float32)
        # the first step's beams are one row each: the others have no score
        first = np.where(np.arange(n) % beams == 0, 0.0, -np.inf).astype(np.float32)
        scores, parents, tokens = mem.up(first), z(n), z(n)
        log = [(z(n), z(n), z(n, t=np.float32)) for _ in range(steps)]
        groups_at = mem.up(np.arange(0, n + 1, beams, dtype=np.int32))
        prefix = mem.up(np.array([len(p) for p in prompts], np.int32))
        used = iter(status)

        def append(rows, ids):
            for e, p in ((ek, k), (ev, v)):
                check(lib().soc_op_embedding(ctx.h, ids, e, 0, p, rows, kw, 97))
            S.paged_append(ctx, cache, rope, None, 0, k, kw, v, kw, "f32", None, 0, rows, 0, None, slots)

        def attend_and_choose(step, ids, table, lengths):
            check(lib().soc_op_embedding(ctx.h, ids, eq, 0, q, n, qw, 97))
            S.paged_attention_shared(ctx, cache, q, qw, "f32", table, width, width, lengths, n, groups_at, prefix, groups, beams,
                                     160, nq, 0.0, out, qw)
            check(lib().soc_op_matmul(ctx.h, out, head, None, None, logits, n, qw, 97, 0, 0))
            rows, toks, vals = log[step]
            S.beam_select(ctx, logits, "f32", 97, groups, beams, 97, 0.125, scores, stops, 0, None, None, None, rows, toks, vals)

        # prompts: the first row of each request
        lengths = np.zeros(n, np.int32)
        lengths[::beams] = [len(p) for p in prompts]
        ctx.write(new, lengths)
        flat = np.zeros(max_rows, np.int32)
        flat[: sum(map(len, prompts))] = sum(prompts, [])
        S.paged_plan(ctx, n, old, new, page, tables[0], width, width, ring, pages, cursors, cursors, starts, positions, slots,
                     max_rows, next(used), step_lens=lens)
        append(max_rows, mem.up(flat))
        last = np.zeros(n, np.int32)
        last[::beams] = [p[-1] for p in prompts]
        attend_and_choose(0, mem.up(last), tables[0], lens)
        at = 0
        for step in range(1, steps):
            rows, toks, vals = log[step - 1]
            S.paged_fork(ctx, n, rows, None, lens, page, tables[at], tables[1 - at], width, width, ring, pages, cursors, cursors,
                         old, new, copies, count, next(used))
            S.paged_copy(ctx, layers, copies, count, n)
            at = 1 - at
            if step % 8 == 0:
                S.paged_compact(ctx, n, old, page, tables[at], tables[at], width, width, ring, ring, pages, cursors, moves, pages,
                                moved, next(used))
                S.paged_copy(ctx, layers, moves, moved, pages)
            S.paged_plan(ctx, n, old, new, page, tables[at], width, width, ring, pages, cursors, cursors, starts, positions, slots,
                         n, next(used), step_lens=lens)
            append(n, toks)  # a row of a plan is a row of the batch: all beams go on
            scores = vals
            attend_and_choose(step, toks, tables[at], lens)
        ctx.synchronize()
        assert all(int(mem.down(s)[0]) == 0 for s in status)
        # the beams, followed back through their parents
        history = [[mem.down(p) for p in entry] for entry in log]
        table, held, c = mem.down(tables[at]), mem.down(lens), mem.down(cursors)
        free = mem.down(ring)[np.arange(c[0], c[1]) % pages]
    named = {int(p) for i in range(n) for p in table[i, : -(-int(held[i]) // page)]}
    assert len(set(free.tolist())) == free.size and named.isdisjoint(free.tolist()) and len(named) + free.size == pages
    assert (held == np.repeat([len(p) for p in prompts], beams) + steps - 1).all()
    for g, prompt in enumerate(prompts):
        want, gap = host_search(model, prompt, beams, steps, stops)
        tol = 2e-5 * steps
        for b in range(beams):
            row, seq = g * beams + b, []
            score = float(history[-1][2][row])
            for rows, toks, _ in reversed(history):
                seq.append(int(toks[row]))
                row = int(rows[row])
            assert abs(score - want[b][0]) <= tol, (g, b, score, want[b][0])
            if gap > 2 * tol:
                assert list(prompt) + seq[::-1] == want[b][1], (g, b)


def test_two_contexts_in_turn(gpu_ctx):
    """Two contexts' calls in turn, each with words and workspaces of its own."""
    from tests.test_gpu_fork import check_fork, pool, some_parents

    rng, other = np.random.default_rng(2), S.Context(0)
    try:
        for i in range(6):
            old, table, ring, cursors = pool(rng, 8 + 90 * (i % 2), 60 + 200 * (i % 2), 16, 300)
            parents, keep = some_parents(rng, len(old), old)
            check_fork((gpu_ctx, other)[i % 2], parents, keep, old, 16, table, ring, cursors)
            check_fork((other, gpu_ctx)[i % 2], parents, keep, old, 16, table, ring, cursors)
    finally:
        other.close()


def test_copies_and_shared_pages_beyond_32_bit_offsets(gpu_ctx, monkeypatch):
    """A pool of more than 2^32 elements each of keys and values: pages at its end are copied to its front and back, and attended
    to by a group whose columns fill blocks and by one of a few columns."""
    monkeypatch.setenv("SOC_PAGED_SHARED", "always")
    from tests.test_gpu_paged_shared import formula

    ctx, rng = gpu_ctx, np.random.default_rng(6)
    page, nkv, nq, hd, sizes, prefix, tail = 256, 8, 16, 128, [12, 2], 512, 30
    per = nkv * page * hd
    pages, n = (1 << 32) // per + 40, sum(sizes)
    common = rng.standard_normal((2, 2, 2, nkv, page, hd)).astype(np.float16)  # [group][place][k, v]
    own = rng.standard_normal((n, 2, nkv, page, hd)).astype(np.float16)
    q = rng.standard_normal((n, nq * hd)).astype(np.float32)
    pk, pv = ctx.alloc(pages * per * 2), ctx.alloc(pages * per * 2)
    # written at the front or at the end, copied to the other: where they are read
    moves = np.array([[3, pages - 1, page], [pages - 2, 4, page], [5, pages - 3, page], [pages - 4, 6, 200]], np.int32)
    table = np.zeros((n, 3), np.int32)
    table[: sizes[0], :2] = [pages - 1, 4]
    table[sizes[0]:, :2] = [pages - 3, pages - 9]
    table[:, 2] = np.where(np.arange(n) % 2, np.arange(n) + 10, pages - 10 - np.arange(n))
    try:
        with Arrays(ctx) as mem:
            def write(p, kv):
                ctx.write(pk + int(p) * per * 2, kv[0])
                ctx.write(pv + int(p) * per * 2, kv[1])

            for p, kv in ((3, common[0, 0]), (pages - 2, common[0, 1]), (5, common[1, 0]), (pages - 9, common[1, 1])):
                write(p, kv)
            for r in range(n):
                write(table[r, 2], own[r])
            write(pages - 4, own[0])
            write(6, own[1])
            cache = S.PagedCache(pk, pv, pages, page, nkv, hd)
            S.paged_copy(ctx, S.PagedLayers([cache]), mem.up(moves), None, len(moves))
            out = mem.up(np.zeros_like(q))
            S.paged_attention_shared(ctx, cache, mem.up(q), nq * hd, "f32", mem.up(table), 3, 3,
                                     mem.up(np.full(n, prefix + tail, np.int32)), n, mem.up(np.array([0, 12, 14], np.int32)),
                                     mem.up(np.full(2, prefix, np.int32)), 2, 12, prefix, nq, 0.0, out, nq * hd)
            got = mem.down(out).reshape(n, nq, hd)
            part = ctx.download(pv + 6 * per * 2, (nkv, page, hd), np.float16)
    finally:
        ctx.synchronize()
        ctx.free(pk)
        ctx.free(pv)
    assert np.array_equal(part[:, :200], own[0, 1][:, :200]) and np.array_equal(part[:, 200:], own[1, 1][:, 200:])
    for r in range(n):
        g = int(r >= sizes[0])
        k, v = (np.concatenate([common[g, 0, i], common[g, 1, i], own[r, i][:, :tail]], 1) for i in range(2))
        want, _, tol, _ = formula(q[r].reshape(nq, hd), k, v, 1 / math.sqrt(hd))
        assert (np.abs(got[r] - want) <= tol).all(), r
