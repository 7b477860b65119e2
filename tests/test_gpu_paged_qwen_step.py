"""A layer's step of a Qwen3-like model over pages, by the library's calls alone: the q and k heads normed
(soc_op_rmsnorm), rotated and stored (soc_paged_append), each request's last query row picked (soc_op_embedding), and
attention over its pages; and a prompt whose rows attend as sequences of their own. Against the formulas in 64 bits.

Tolerance of a normed value: 64 squares added as a tree (7 roundings of 2^-24 and the square's), mean and eps (2), half of
that from the root, which rounds once and its reciprocal twice, two products: below 16 2^-24. Rotation adds its own 8 2^-24;
a cached key is rounded to fp16. The attention is compared on the queries and keys that the calls before it left."""
import math

import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import check, lib
from tests.device import Arrays
from tests.test_gpu_paged import attend, plan_rules
from tests.test_gpu_rope import frequencies, rotate

pytestmark = pytest.mark.gpu


def test_steps_with_head_norms_and_mixed_rows(gpu_ctx):
    ctx, rng = gpu_ctx, np.random.default_rng(41)
    n, nq, nkv, hd, page, pages, width, max_rows, eps = 3, 8, 2, 64, 16, 20, 8, 64, 1e-6
    f = frequencies(hd, 1e6, "none", 1.0, 0)
    gains = [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    table, ring = np.full((n, width), -1, np.int32), rng.permutation(pages).astype(np.int32)
    cursors = np.array([0, pages], np.int64)
    with Arrays(ctx) as mem:
        z = lambda *s, t=np.int32: mem.up(np.zeros(s, t))  # noqa: E731
        po, pn, lens, pt, pr, pc = z(n), z(n), z(n), mem.up(table), mem.up(ring), mem.up(cursors)
        ps, pp, pl, st, last = z(n + 1), z(max_rows), z(max_rows), z(1), z(n)
        gq, gk = (mem.up(g) for g in gains)
        q_proj, q = z(max_rows, nq * hd, t=np.float32), z(max_rows, nq * hd, t=np.float32)
        k_proj, k = z(max_rows, nkv * hd, t=np.float32), z(max_rows, nkv * hd, t=np.float32)
        v, q_last, out = z(max_rows, nkv * hd, t=np.float32), z(n, nq * hd, t=np.float32), z(n, nq * hd, t=np.float32)
        pk, pv = (mem.up(np.full((pages, nkv, page, hd), np.nan, np.float16)) for _ in range(2))
        # a prompt's rows as sequences of their own
        rt, rl, ro = z(max_rows, width), z(max_rows), z(max_rows, nq * hd, t=np.float32)
        cache, rope = S.PagedCache(pk, pv, pages, page, nkv, hd), S.Rope(ctx, hd)
        for old, new in [([0, 0, 0], [37, 5, 0]), ([37, 5, 0], [38, 6, 20]), ([38, 6, 20], [39, 0, 50])]:
            rows = [rng.standard_normal((max_rows, h * hd)).astype(np.float32) * 3 for h in (nq, nkv, nkv)]
            for p, a in ((po, old), (pn, new)):
                ctx.write(p, np.array(a, np.int32))
            for p, a in zip((q_proj, k_proj, v), rows):
                ctx.write(p, a)
            S.paged_plan(ctx, n, po, pn, page, pt, width, width, pr, pages, pc, pc, ps, pp, pl, max_rows, st, step_lens=lens)
            check(lib().soc_op_rmsnorm(ctx.h, q_proj, gq, q, max_rows * nq, hd, eps))
            check(lib().soc_op_rmsnorm(ctx.h, k_proj, gk, k, max_rows * nkv, hd, eps))
            S.paged_append(ctx, cache, rope, q, nq * hd, k, nkv * hd, v, nkv * hd, "f32", q, nq * hd, max_rows, nq, pp, pl)
            # what the plan gives follows from the lengths: the host knows each request's last row
            want = plan_rules(old, new, page, table, ring, cursors, max_rows, pages)
            table, ring, cursors, starts, positions, slots, status = want
            ctx.write(last, (starts[1:] - 1).astype(np.int32))
            check(lib().soc_op_embedding(ctx.h, last, q, 0, q_last, n, nq * hd, max_rows))
            S.paged_attention_decode(ctx, cache, q_last, nq * hd, "f32", pt, width, width, lens, n, nq, 0.0, out, nq * hd)
            owner = np.repeat(np.arange(n), np.diff(starts))
            total = owner.size
            ctx.write(rt, np.ascontiguousarray(table[owner]))
            ctx.write(rl, positions[:total] + 1)
            S.paged_attention_decode(ctx, cache, q, nq * hd, "f32", rt, width, width, rl, total, nq, 0.0, ro, nq * hd)
            assert mem.down(st)[0] == status == 0
            got_q, got_out, got_rows = mem.down(q), mem.down(out), mem.down(ro)
            keys, values = mem.down(pk), mem.down(pv)
            for rows_in, gain, heads, got in ((rows[0], gains[0], nq, got_q), (rows[1], gains[1], nkv, None)):
                x = rows_in[:total].reshape(total, heads, hd).astype(np.float64)
                x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain
                y, tol = rotate(x, positions[:total], hd, "half", f, 1.0)
                tol = 3 * tol  # 8 for the rotation and 16 for what it takes
                if got is None:
                    got = keys[slots[:total] // page, :, slots[:total] % page].astype(np.float64)
                    tol = tol + np.abs(y) * 2.0 ** -11 + 2.0 ** -25
                assert (np.abs(got[:total].reshape(total, heads, hd) - y) <= tol).all()
            plain = []
            for i in range(n):
                mine = table[i, : -(-new[i] // page)]
                plain.append([t[mine].transpose(1, 0, 2, 3).reshape(nkv, -1, hd)[:, : new[i]] for t in (keys, values)])
                at = np.flatnonzero(owner == i)
                assert np.array_equal(plain[i][1][:, old[i]:], rows[2][at].reshape(-1, nkv, hd).transpose(1, 0, 2)
                                      .astype(np.float16)) or new[i] <= old[i]
                if at.size:
                    w, _, tol, _ = attend(got_q[at[-1]].reshape(nq, hd), *plain[i], 1 / math.sqrt(hd))
                    assert (np.abs(got_out[i].reshape(nq, hd) - w) <= tol).all(), (i, new)
            for r in range(total):
                kv = [t[:, : positions[r] + 1] for t in plain[owner[r]]]
                w, _, tol, _ = attend(got_q[r].reshape(nq, hd), *kv, 1 / math.sqrt(hd))
                assert (np.abs(got_rows[r].reshape(nq, hd) - w) <= tol).all(), (r, new)
        rope.close()
