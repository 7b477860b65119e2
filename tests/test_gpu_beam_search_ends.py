"""A beam search whose prompts are long enough that attention reads them once for a request's beams (256 keys and more), in which
beams end, come back and end for good: a first step with fewer tokens to choose than beams, beams that a mask leaves without a
continuation, a request that ends before the others. The program reads each step's tokens and `row_starts` back, as one that
streams its tokens does, and puts the tokens of the rows that go on where the plan's rows are; the logits of rows that took no part
are NaN. Against the search in Python of tests/test_gpu_beam_search.py, with its tolerance."""
import math

import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import check, lib
from tests.device import Arrays
from tests.test_gpu_beam_search import Model

VOCAB, GROUPS, BEAMS, STEPS, STOPS = 97, 3, 4, 14, [11, 60]


def allowed(step, group, last):
    """Which tokens may follow `last` at a step of a request."""
    ok = np.ones(VOCAB, bool)
    if step == 0 and group != 1:  # two tokens, one of them a stop token; three
        ok[:] = False
        ok[[11, 20] if group == 0 else [5, 6, 7]] = True
    if step == 6 and group != 1:  # of some beams none, of the others one
        ok[:] = False
        ok[30] = last % 2 == 1
    if step == 9 and group == 2:  # of none: the request has ended
        ok[:] = False
    return ok


def host_search(model, prompt, group):
    """The live beams after each step, and how far the nearest rival was from changing them."""
    live, gap, history = [(0.0, list(prompt))], np.inf, []
    for step in range(STEPS):
        cands = []
        for b, (score, tokens) in enumerate(live):
            ok = allowed(step, group, tokens[-1])
            if not ok.any():
                continue
            z = np.where(ok, model.logits(tokens), -np.inf)
            lp = z - z.max() - np.log(np.exp(z - z.max()).sum())
            cands += [(score + lp[t], b, t) for t in range(VOCAB) if ok[t] and t not in STOPS]
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        best = cands[: BEAMS + 1]
        gap = min([gap] + [best[i][0] - best[i + 1][0] for i in range(len(best) - 1)])
        live = [(s, live[b][1] + [t]) for s, b, t in best[:BEAMS]]
        history.append(live)
    return history, gap


def setting(page, hd, nq, nkv, seed):
    model = Model(VOCAB, nq, nkv, hd, seed)
    rng = np.random.default_rng(seed)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (310, 40, 263)]
    return model, prompts, [host_search(model, p, g) for g, p in enumerate(prompts)]


TOL = 2e-5 * STEPS
CASES = [(16, 64, 4, 2, 10), (32, 128, 8, 2, 6), (16, 128, 20, 2, 13)]


@pytest.mark.parametrize("page,hd,nq,nkv,seed", CASES)
def test_the_search_in_python_has_clear_choices(page, hd, nq, nkv, seed):
    """What the comparison on the GPU needs: rivals further away than the tolerance, beams that end and come back."""
    _, _, searches = setting(page, hd, nq, nkv, seed)
    assert all(gap > 2 * TOL for _, gap in searches)
    live = [[len(step) for step in history] for history, _ in searches]
    assert live[0][0] == 1 and live[2][0] == 3 and all(n == BEAMS for n in live[1])
    assert 0 < live[0][6] < BEAMS and 0 < live[2][6] < BEAMS and live[0][-1] == live[2][8] == BEAMS and not any(live[2][9:])


@pytest.mark.gpu
@pytest.mark.parametrize("page,hd,nq,nkv,seed", CASES)
def test_beams_that_end(gpu_ctx, page, hd, nq, nkv, seed, monkeypatch):
    monkeypatch.setenv("SOC_PAGED_SHARED", "always")  # a small batch would be read row by row
    ctx = gpu_ctx
    model, prompts, searches = setting(page, hd, nq, nkv, seed)
    n, qw, kw, longest = GROUPS * BEAMS, nq * hd, nkv * hd, max(map(len, prompts))
    total = sum(map(len, prompts))
    width = -(-(longest + STEPS) // page)
    pages = -(-total // page) + n * (STEPS // page + 3)
    with Arrays(ctx) as mem:
        z = lambda *s, t=np.int32: mem.up(np.zeros(s, t))  # noqa: E731
        tables = [mem.up(np.full((n, width), -1, np.int32)) for _ in range(2)]
        order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
        ring, cursors = mem.up(order), mem.up(np.array([0, pages], np.int64))
        pk, pv = (mem.up(np.full((pages, nkv, page, hd), np.nan, np.float16)) for _ in range(2))
        cache = S.PagedCache(pk, pv, pages, page, nkv, hd)
        layers = S.PagedLayers([cache])
        eq, ek, ev, head = (mem.up(x) for x in (model.q, model.k, model.v, model.head))
        starts, positions, slots, lens, old, new = z(n + 1), z(total), z(total), z(n), z(n), z(n)
        copies, count, status, ids = z(n, 3), z(1), z(1), z(total)
        q, out, logits = z(n, qw, t=np.float32), z(n, qw, t=np.float32), z(n, VOCAB, t=np.float32)
        k, v = z(total, kw, t=np.float32), z(total, kw, t=np.float32)
        scores = mem.up(np.where(np.arange(n) % BEAMS == 0, 0.0, -np.inf).astype(np.float32))
        parents, tokens = z(n), z(n)
        groups_at = mem.up(np.arange(0, n + 1, BEAMS, dtype=np.int32))
        prefix = mem.up(np.array([len(p) for p in prompts], np.int32))

        def done():
            assert int(mem.down(status)[0]) == 0

        def append(rows, given):
            ctx.write(ids, given)
            for e, p in ((ek, k), (ev, v)):
                check(lib().soc_op_embedding(ctx.h, ids, e, 0, p, rows, kw, VOCAB))
            S.paged_append(ctx, cache, None, None, 0, k, kw, v, kw, "f32", None, 0, rows, 0, None, slots)

        def attend(last, table):
            ctx.write(ids, np.maximum(last, 0))
            check(lib().soc_op_embedding(ctx.h, ids, eq, 0, q, n, qw, VOCAB))
            S.paged_attention_shared(ctx, cache, q, qw, "f32", table, width, width, lens, n, groups_at, prefix, GROUPS, BEAMS,
                                     longest, nq, 0.0, out, qw)

        def choose(step, last):
            check(lib().soc_op_matmul(ctx.h, out, head, None, None, logits, n, qw, VOCAB, 0, 0))
            x = mem.down(logits)
            for r in range(n):
                if last[r] < 0:
                    x[r] = np.nan
                else:
                    x[r, ~allowed(step, r // BEAMS, int(last[r]))] = -np.inf
            ctx.write(logits, x)
            S.beam_select(ctx, logits, "f32", VOCAB, GROUPS, BEAMS, VOCAB, 0.125, scores, STOPS, 0, None, None, None, parents,
                          tokens, scores)
            return mem.down(parents), mem.down(tokens), mem.down(scores)

        # the prompts: the first row of each request
        lengths, last = np.zeros(n, np.int32), np.full(n, -1, np.int32)
        lengths[::BEAMS], last[::BEAMS] = [len(p) for p in prompts], [p[-1] for p in prompts]
        ctx.write(new, lengths)
        S.paged_plan(ctx, n, old, new, page, tables[0], width, width, ring, pages, cursors, cursors, starts, positions, slots, total,
                     status, step_lens=lens)
        done()
        append(total, np.array(sum(prompts, []), np.int32))
        attend(last, tables[0])
        seqs = [list(prompts[r // BEAMS]) for r in range(n)]
        at = 0
        for step in range(STEPS):
            par, tok, val = choose(step, last)
            seqs = [seqs[p] + [int(t)] if p >= 0 else [] for p, t in zip(par, tok)]
            for g, (history, _) in enumerate(searches):
                want = history[step]
                for b in range(BEAMS):
                    r = g * BEAMS + b
                    if b >= len(want):
                        assert (par[r], tok[r], val[r]) == (-1, -1, -np.inf), (step, r)
                    else:
                        assert par[r] // BEAMS == g and seqs[r] == want[b][1], (step, r)
                        assert abs(val[r] - want[b][0]) <= TOL
            if step == STEPS - 1:
                break
            S.paged_fork(ctx, n, parents, None, lens, page, tables[at], tables[1 - at], width, width, ring, pages, cursors, cursors,
                         old, new, copies, count, status)
            done()
            S.paged_copy(ctx, layers, copies, count, n)
            at = 1 - at
            S.paged_plan(ctx, n, old, new, page, tables[at], width, width, ring, pages, cursors, cursors, starts, positions, slots,
                         n, status, step_lens=lens)
            done()
            # a row that got no token has no row in the step
            where, given = mem.down(starts), np.zeros(n, np.int32)
            assert np.array_equal(np.diff(where), tok >= 0)
            given[where[:-1][tok >= 0]] = tok[tok >= 0]
            append(n, given)
            last = tok
            attend(last, tables[at])
            held, table, c = mem.down(lens), mem.down(tables[at]), mem.down(cursors)
            free = mem.down(ring)[np.arange(c[0], c[1]) % pages].tolist()
            named = {int(p) for i in range(n) for p in table[i, : -(-int(held[i]) // page)]}
            assert [int(h) for h in held] == [len(s) if s else 0 for s in seqs]
            assert len(set(free)) == len(free) and named.isdisjoint(free) and len(named) + len(free) == pages
        assert (held[2 * BEAMS:] == 0).all()
        # the prompts were read once, from the first row's pages: other pages in the later rows' tables change nothing (up to
        # what is whole tiles of 32 keys)
        got, other = mem.down(out), mem.down(tables[at])
        other[1:BEAMS, : 256 // page] = other[BEAMS, 0]
        S.paged_attention_shared(ctx, cache, q, qw, "f32", mem.up(other), width, width, lens, n, groups_at, prefix, GROUPS, BEAMS,
                                 longest, nq, 0.0, out, qw)
        assert np.array_equal(mem.down(out), got)
