"""What is queued behind a plan whose status nobody has read yet: soc_paged_plan_step's lengths keep the attention on the
pages that a request holds, also where the step was refused and the table's row still names pages that are another's."""
import math

import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import PLAN_CURSORS, PLAN_LENGTHS, PLAN_PAGES, PLAN_ROWS, SOC_ERR_INVALID
from tests.device import Arrays, guarded
from tests.test_gpu_paged import attend, make_pool, plan_rules

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 3, 255, 257, 1025, 4096])
@pytest.mark.parametrize("bits", [0, PLAN_LENGTHS, PLAN_CURSORS, PLAN_PAGES, PLAN_ROWS])
def test_step_lens(gpu_ctx, n, bits):
    """new_lens of a step that is done, old_lens of one that is not; everything else as soc_paged_plan gives it."""
    rng = np.random.default_rng(n + bits)
    page, width = 16, 5
    old, new = rng.integers(0, 65, n), rng.integers(0, 65, n)
    old[0], new[0] = 3, 40
    table, ring, cursors = make_pool(rng, old, page, width, n * width + 4, 77)
    max_rows = max(1, int(np.maximum(0, new - old).sum()))
    if bits == PLAN_LENGTHS:
        new[n - 1] = 16 * width + 1
    if bits == PLAN_CURSORS:
        cursors = np.array([9, 8])
    if bits == PLAN_PAGES:
        cursors = np.array([77, 77])
    if bits == PLAN_ROWS:
        max_rows -= 1
    want = plan_rules(old, new, page, table, ring, cursors, max_rows, ring.size)
    assert want[6] == bits
    for alias in (False, True):
        with Arrays(gpu_ctx) as mem:
            po, pn = mem.up(old.astype(np.int32)), mem.up(new.astype(np.int32))
            pt, pr, pc = mem.up(table), mem.up(ring), mem.up(np.asarray(cursors, np.int64))
            pc2 = pc if alias else mem.up(np.zeros(2, np.int64))
            ps, pp, pl, st = (mem.up(np.full(k, 99, np.int32)) for k in (n + 1, max_rows, max_rows, 1))
            lens = mem.up(guarded(np.full(n, 99, np.int32), 2, 3, 55))
            S.paged_plan(gpu_ctx, n, po, pn, page, pt, width, width, pr, ring.size, pc, pc2, ps, pp, pl, max_rows, st,
                         step_lens=lens + 8)
            got = mem.down(lens)
            assert (got[:2] == 55).all() and (got[-3:] == 55).all()
            assert np.array_equal(got[2:-3], old if bits else new)
            for p, w in zip((pt, pr, pc2, ps, pp, pl, st), want):
                assert np.array_equal(mem.down(p).reshape(-1).astype(np.int64), np.asarray(w, np.int64).reshape(-1))


def test_attention_behind_a_refused_plan(gpu_ctx):
    """A server's run of calls: request 0 rolled back, its page went to request 1, and the step in which it would need
    another is refused. What it attends to is its own, and request 1's as well; nothing is stored."""
    ctx, rng = gpu_ctx, np.random.default_rng(31)
    n, nq, nkv, hd, page, num_pages, width, max_rows = 2, 4, 2, 64, 16, 3, 3, 64
    row = (nq + 2 * nkv) * hd
    steps = [([0, 0], [32, 10], 0), ([32, 10], [15, 10], 0), ([15, 10], [15, 30], 0), ([15, 30], [16, 30], 0),
             ([16, 30], [17, 31], PLAN_PAGES)]
    with Arrays(ctx) as mem:
        z = lambda *s, t=np.int32: mem.up(np.zeros(s, t))  # noqa: E731
        po, pn, lens, pt = z(n), z(n), z(n), mem.up(np.full((n, width), -1, np.int32))
        pr, pc = mem.up(np.arange(num_pages, dtype=np.int32)), mem.up(np.array([0, num_pages], np.int64))
        ps, pp, pl, st = z(n + 1), z(max_rows), z(max_rows), z(1)
        pk, pv = (mem.up(np.full((num_pages, nkv, page, hd), np.nan, np.float16)) for _ in range(2))
        pqkv, pq = z(max_rows, row, t=np.float32), z(max_rows, nq * hd, t=np.float32)
        query = rng.standard_normal((n, nq * hd)).astype(np.float32)
        pd, pout = mem.up(query), z(n, nq * hd, t=np.float32)
        cache, rope = S.PagedCache(pk, pv, num_pages, page, nkv, hd), S.Rope(ctx, hd)
        # (the third step needs no page of request 0, so that the page it gave back goes to request 1)
        for old, new, bits in steps:
            ctx.write(po, np.array(old, np.int32))
            ctx.write(pn, np.array(new, np.int32))
            ctx.write(pqkv, rng.standard_normal((max_rows, row)).astype(np.float32))
            before = mem.down(pk).copy()
            S.paged_plan(ctx, n, po, pn, page, pt, width, width, pr, num_pages, pc, pc, ps, pp, pl, max_rows, st,
                         step_lens=lens)
            S.paged_append(ctx, cache, rope, pqkv, row, pqkv + 4 * nq * hd, row, pqkv + 4 * (nq + nkv) * hd, row, "f32", pq,
                           nq * hd, max_rows, nq, pp, pl)
            S.paged_attention_decode(ctx, cache, pd, nq * hd, "f32", pt, width, width, lens, n, nq, 0.0, pout, nq * hd)
            out, table, keys, values = mem.down(pout), mem.down(pt), mem.down(pk), mem.down(pv)
            assert mem.down(st)[0] == bits
            held = old if bits else new
            assert np.array_equal(mem.down(lens), held)
            if bits:
                assert np.array_equal(before.view(np.uint16), keys.view(np.uint16))
            pages = [set(table[i, : -(-held[i] // page)].tolist()) for i in range(n)]
            assert not pages[0] & pages[1]
            for i in range(n):
                k, v = (t[table[i, : -(-held[i] // page)]].transpose(1, 0, 2, 3).reshape(nkv, -1, hd)[:, : held[i]]
                        for t in (keys, values))
                want, _, tol, _ = attend(query[i].reshape(nq, hd), k, v, 1 / math.sqrt(hd))
                assert (np.abs(out[i].reshape(nq, hd) - want) <= tol).all(), (i, new)
        rope.close()


def test_stale_entries_are_not_attended_to(gpu_ctx):
    """Entries behind the pages held name the other request's page: its values (100) must not reach request 0 (ones)."""
    keys = np.zeros((2, 1, 16, 64), np.float16)
    values = np.ones((2, 1, 16, 64), np.float16)
    values[1] = 100
    with Arrays(gpu_ctx) as mem:
        po, pn = mem.up(np.array([16, 16], np.int32)), mem.up(np.array([17, 16], np.int32))
        pt, pr = mem.up(np.array([[0, 1], [1, -1]], np.int32)), mem.up(np.array([0, 1], np.int32))
        pc, lens, st = mem.up(np.array([2, 2], np.int64)), mem.up(np.zeros(2, np.int32)), mem.up(np.zeros(1, np.int32))
        ps, pp, pl = mem.up(np.zeros(3, np.int32)), mem.up(np.zeros(4, np.int32)), mem.up(np.zeros(4, np.int32))
        q, out = mem.up(np.ones((2, 64), np.float32)), mem.up(np.zeros((2, 64), np.float32))
        S.paged_plan(gpu_ctx, 2, po, pn, 16, pt, 2, 2, pr, 2, pc, pc, ps, pp, pl, 4, st, step_lens=lens)
        S.paged_attention_decode(gpu_ctx, S.PagedCache(mem.up(keys), mem.up(values), 2, 16, 1, 64), q, 64, "f32", pt, 2, 2,
                                 lens, 2, 1, 0.0, out, 64)
        assert mem.down(st)[0] == PLAN_PAGES
        got = mem.down(out)
    assert np.abs(got[0] - 1).max() < 1e-5 and np.abs(got[1] - 100).max() < 1e-3


def test_step_lens_operand_is_checked(gpu_ctx):
    with Arrays(gpu_ctx) as mem:
        z = lambda n, t=np.int32: mem.up(np.zeros(n, t))  # noqa: E731
        lens, new, table, ring, cur, starts, pos, slots, st, out = (z(8), z(4), z(8), z(9), z(2, np.int64), z(5), z(8), z(8),
                                                                    z(1), z(4))

        def call(step_lens):
            S.paged_plan(gpu_ctx, 4, lens, new, 16, table, 2, 2, ring, 9, cur, cur, starts, pos, slots, 8, st,
                         step_lens=step_lens)

        for p, text in [(lens, "overlap"), (new, "overlap"), (lens + 12, "overlap"), (out + 4, "past the end"),
                        (out + 2, "aligned"), (np.zeros(4, np.int32).ctypes.data, "not in device memory")]:
            with pytest.raises(S.SocError, match=text) as e:
                call(p)
            assert e.value.code == SOC_ERR_INVALID
        call(lens + 16)
        gpu_ctx.synchronize()
