"""Serving from a paged key-value cache: the plan of a step (soc_paged_plan) against the same rules in Python, the append
(soc_paged_append) and the decode attention (soc_paged_attention_decode) against their formulas in 64 bits, and all of
them together over several steps.

Tolerance of the attention. A score is a sum of head_dim products, queries exact to 2^-22, added in 32 bits in any order:
off by (head_dim + 8) 2^-24 sum |q_i k_i| scale = e. A weight is then off by 2 e + 8 2^-24 relative (its own score and
the common maximum's; the exponential), the weighted sum by that, by its weights' 2^-22 and by chains of at most 512
additions: |out - want| <= (2 e + 512 2^-24 + 8 2^-24 + 2^-21) max |v|. lse: e + 520 2^-24 + 2^-23 |lse|. fp16 results
add half a step, 2^-11 relative."""
import math

import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import (PLAN_CURSORS, PLAN_LENGTHS, PLAN_PAGES, PLAN_ROWS, SOC_ERR_INVALID)
from tests.device import NP, Arrays, guarded
from tests.test_gpu_rope import check as rope_check, frequencies, rotate

pytestmark = pytest.mark.gpu


# ---- plan ------------------------------------------------------------------------------------------------------------
def plan_rules(old, new, page, table, ring, cursors, max_rows, num_pages):
    """soc_paged_plan's contract, one request and page after the other."""
    table, ring = table.copy(), ring.copy()
    head, tail = (int(c) for c in cursors)
    max_pages = table.shape[1]

    def pages(n):
        return -(-int(n) // page)

    status = 0
    if any(n < 0 or pages(n) > max_pages for n in [*old, *new]):
        status |= PLAN_LENGTHS
    good = [(int(o), int(n)) if o >= 0 and n >= 0 and pages(o) <= max_pages and pages(n) <= max_pages else (0, 0)
            for o, n in zip(old, new)]
    take = sum(max(0, pages(n) - pages(o)) for o, n in good)
    give = sum(max(0, pages(o) - pages(n)) for o, n in good)
    rows = sum(max(0, n - o) for o, n in good)
    free = tail - head
    if head < 0 or tail < 0 or free < 0 or free > num_pages or free + give > num_pages:
        status |= PLAN_CURSORS
    elif take > free:
        status |= PLAN_PAGES
    if rows > max_rows:
        status |= PLAN_ROWS
    starts, positions, slots = [0], np.zeros(max_rows, np.int32), np.full(max_rows, -1, np.int32)
    if status:
        return table, ring, cursors, np.zeros(len(old) + 1, np.int32), positions, slots, status
    before = table.copy()
    for i, (o, n) in enumerate(good):
        for j in range(pages(o), pages(n)):
            table[i, j] = ring[head % num_pages]
            head += 1
        for j in range(pages(n), pages(o)):
            ring[tail % num_pages] = before[i, j]
            tail += 1
        at = np.arange(o, max(o, n))
        positions[starts[-1]: starts[-1] + at.size] = at
        ids = table[i, at // page].astype(np.int64)
        slots[starts[-1]: starts[-1] + at.size] = np.where((ids >= 0) & (ids < num_pages), ids * page + at % page, -1)
        starts.append(starts[-1] + at.size)
    return table, ring, np.array([head, tail]), np.array(starts, np.int32), positions, slots, 0


def run_plan(ctx, old, new, page, table, ring, cursors, max_rows, alias=False, extra=0):
    """The call between guard elements; (table, ring, cursors, starts, positions, slots, status)."""
    n, width = table.shape
    wide = np.full((n, width + extra), 77, np.int32)
    wide[:, :width] = table
    with Arrays(ctx) as mem:
        po, pn = mem.up(np.asarray(old, np.int32)), mem.up(np.asarray(new, np.int32))
        pt, pr, pc = mem.up(wide), mem.up(ring), mem.up(np.asarray(cursors, np.int64))
        pc2 = pc if alias else mem.up(np.full(2, 5, np.int64))
        outs = [mem.up(guarded(np.full(k, 99, np.int32), 2, 3, 55)) for k in (n + 1, max_rows, max_rows, 1)]
        S.paged_plan(ctx, n, po, pn, page, pt, width, width + extra, pr, ring.size, pc, pc2, outs[0] + 8, outs[1] + 8,
                     outs[2] + 8, max_rows, outs[3] + 8)
        starts, positions, slots, status = (mem.down(p) for p in outs)
        for g in (starts, positions, slots, status):
            assert (g[:2] == 55).all() and (g[-3:] == 55).all()
        t = mem.down(pt)
        assert (t[:, width:] == 77).all()
        assert np.array_equal(mem.down(po), np.asarray(old, np.int32))
        return (t[:, :width], mem.down(pr), mem.down(pc2), starts[2:-3], positions[2:-3], slots[2:-3], int(status[2]))


def same_plan(got, want):
    for name, g, w in zip(("table", "ring", "cursors", "starts", "positions", "slots"), got, want):
        assert np.array_equal(np.asarray(g).astype(np.int64), np.asarray(w).astype(np.int64)), name
    assert got[6] == want[6]


def make_pool(rng, old, page, width, num_pages, start=0):
    """(table, ring, cursors) of requests that hold `old` positions, the rest free."""
    held = -(-np.asarray(old) // page)
    order = rng.permutation(num_pages).astype(np.int32)
    table = np.full((len(old), width), -1, np.int32)
    table[np.arange(width)[None, :] < held[:, None]] = order[: held.sum()]
    free = order[held.sum():]
    ring = np.full(num_pages, -7, np.int32)
    ring[(start + np.arange(free.size)) % num_pages] = free
    return table, ring, np.array([start, start + free.size], np.int64)


def lengths(rng, n, longest):
    old = rng.integers(0, longest + 1, n)
    new = old.copy()
    kind = rng.integers(0, 6, n)
    new[kind == 0] = rng.integers(0, longest + 1, int((kind == 0).sum()))
    new[kind == 1] = 0
    new[kind >= 3] = np.minimum(longest, old[kind >= 3] + 1)
    old[kind == 2] = 0
    return old, new


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 257, 1000, 4096])
def test_plan_of_mixed_steps(gpu_ctx, n, page):
    rng = np.random.default_rng(n * 1000 + page)
    longest = 700
    old, new = lengths(rng, n, longest)
    width = -(-longest // page)
    rows = int(np.maximum(0, new - old).sum())
    table, ring, cursors = make_pool(rng, old, page, width, n * width + 3, int(rng.integers(0, 1 << 40)))
    for max_rows in (max(1, rows), rows + 1000):
        want = plan_rules(old, new, page, table, ring, cursors, max_rows, ring.size)
        assert want[6] == 0
        same_plan(run_plan(gpu_ctx, old, new, page, table, ring, cursors, max_rows), want)
        same_plan(run_plan(gpu_ctx, old, new, page, table, ring, cursors, max_rows, alias=True, extra=5), want)


@pytest.mark.parametrize("old,new", [([0], [1]), ([0], [0]), ([5], [0]), ([15], [16]), ([16], [17]), ([17], [16]),
                                     ([16], [15]), ([1], [700]), ([700], [1]), ([0, 0, 0], [0, 0, 0]),
                                     ([0] * 5, [1] * 5), ([32] * 3, [0, 33, 31])])
def test_plan_edges(gpu_ctx, old, new):
    rng = np.random.default_rng(3)
    table, ring, cursors = make_pool(rng, old, 16, 44, 300)
    want = plan_rules(old, new, 16, table, ring, cursors, 800, 300)
    assert want[6] == 0
    same_plan(run_plan(gpu_ctx, old, new, 16, table, ring, cursors, 800), want)


def test_plan_of_long_prompts(gpu_ctx):
    """A few requests with tens of thousands of rows, more than any block's share."""
    rng = np.random.default_rng(4)
    old, new = [0, 100, 40000, 7], [60001, 101, 0, 30000]
    table, ring, cursors = make_pool(rng, old, 64, 1000, 4000)
    want = plan_rules(old, new, 64, table, ring, cursors, 100000, 4000)
    assert want[6] == 0
    same_plan(run_plan(gpu_ctx, old, new, 64, table, ring, cursors, 100000), want)


def test_plan_exact_fits(gpu_ctx):
    """Every free page taken, every page given back, exactly max_rows rows."""
    rng = np.random.default_rng(5)
    old, new = [10, 0], [32, 48]
    table, ring, cursors = make_pool(rng, old, 16, 3, 5, 12345)
    want = plan_rules(old, new, 16, table, ring, cursors, 70, 5)
    assert want[6] == 0 and want[2][0] == want[2][1]
    same_plan(run_plan(gpu_ctx, old, new, 16, table, ring, cursors, 70), want)
    old, new = [32, 48], [0, 0]
    table, ring, cursors = make_pool(rng, old, 16, 3, 5, 99)
    want = plan_rules(old, new, 16, table, ring, cursors, 1, 5)
    assert want[6] == 0 and want[2][1] - want[2][0] == 5
    same_plan(run_plan(gpu_ctx, old, new, 16, table, ring, cursors, 1), want)


@pytest.mark.parametrize("what", ["negative", "negative after", "long", "long after", "largest", "head", "tail", "full",
                                  "backwards", "pages", "rows", "all"])
@pytest.mark.parametrize("n", [3, 600])
def test_plan_refused_on_the_device(gpu_ctx, what, n):
    """A step that cannot be done changes nothing: status bits, no rows, cursors as they were."""
    rng = np.random.default_rng(6)
    old, new = np.full(n, 20), np.full(n, 40)
    table, ring, cursors = make_pool(rng, old, 16, 4, 4 * n)
    max_rows, bits = 20 * n, 0
    if what in ("negative", "all"):
        old[n - 1], bits = -1, PLAN_LENGTHS
    if what == "negative after":
        new[0], bits = -2 ** 31, PLAN_LENGTHS
    if what == "long":
        old[1], bits = 65, PLAN_LENGTHS
    if what == "long after":
        new[n // 2], bits = 65, PLAN_LENGTHS
    if what == "largest":
        new[2], bits = 2 ** 31 - 1, PLAN_LENGTHS
    if what == "head":
        cursors, bits = np.array([-1, 5]), PLAN_CURSORS
    if what == "tail":
        cursors, bits = np.array([2 ** 62, -2 ** 62]), PLAN_CURSORS
    if what == "full":
        cursors, bits = np.array([7, 7 + 4 * n + 1]), PLAN_CURSORS
    if what == "backwards":
        cursors, bits = np.array([9, 8]), PLAN_CURSORS
    if what in ("pages", "all"):
        cursors, bits = np.array([9, 9 + n - (2 if what == "all" else 1)]), bits | PLAN_PAGES
    if what in ("rows", "all"):
        max_rows, bits = 20 * n - 21, bits | PLAN_ROWS
    if what == "rows":
        max_rows = 20 * n - 1
    want = plan_rules(old, new, 16, table, ring, cursors, max_rows, ring.size)
    assert want[6] == bits
    same_plan(run_plan(gpu_ctx, old, new, 16, table, ring, cursors, max_rows), want)
    same_plan(run_plan(gpu_ctx, old, new, 16, table, ring, cursors, max_rows, alias=True), want)


def test_plan_giving_back_more_than_the_ring_holds(gpu_ctx):
    """Cursors that count pages as free which requests still hold."""
    rng = np.random.default_rng(7)
    old, new = [64, 64], [0, 64]
    table, ring, _ = make_pool(rng, old, 16, 4, 10)
    want = plan_rules(old, new, 16, table, ring, [0, 8], 10, 10)
    assert want[6] == PLAN_CURSORS
    same_plan(run_plan(gpu_ctx, old, new, 16, table, ring, [0, 8], 10), want)


def test_plan_with_foreign_page_ids(gpu_ctx):
    """Page ids that are none of the cache's give no slot; nothing else changes."""
    rng = np.random.default_rng(8)
    old, new = [8, 16, 5, 40], [20, 17, 6, 41]
    table, ring, cursors = make_pool(rng, old, 16, 4, 20)
    ring[cursors[0] % 20] = -9
    ring[(cursors[0] + 1) % 20] = 2 ** 31 - 1
    table[2, 0], table[3, 2] = 20, -2 ** 31
    want = plan_rules(old, new, 16, table, ring, cursors, 30, 20)
    assert want[6] == 0 and (want[5][:17] == -1).sum() > 3
    same_plan(run_plan(gpu_ctx, old, new, 16, table, ring, cursors, 30), want)


def test_plan_over_many_steps_keeps_every_page(gpu_ctx):
    """A server's life in one set of buffers: after every step the pages held and the pages free are all pages once."""
    rng = np.random.default_rng(9)
    n, page, width, num_pages = 90, 32, 8, 400
    table = np.full((n, width), -1, np.int32)
    ring, cursors = rng.permutation(num_pages).astype(np.int32), np.array([0, num_pages], np.int64)
    old = np.zeros(n, np.int64)
    with Arrays(gpu_ctx) as mem:
        po, pn, pt, pr = mem.up(old.astype(np.int32)), mem.up(old.astype(np.int32)), mem.up(table), mem.up(ring)
        pc, ps = mem.up(cursors), mem.up(np.zeros(n + 1, np.int32))
        pp, pl, st = mem.up(np.zeros(6000, np.int32)), mem.up(np.zeros(6000, np.int32)), mem.up(np.zeros(1, np.int32))
        for step in range(25):
            _, new = lengths(rng, n, 120)
            new = np.where(rng.random(n) < 0.4, np.minimum(old + 1, 256), new)
            new = np.where(rng.random(n) < 0.1, 256, new)
            gpu_ctx.write(po, old.astype(np.int32))
            gpu_ctx.write(pn, new.astype(np.int32))
            S.paged_plan(gpu_ctx, n, po, pn, page, pt, width, width, pr, num_pages, pc, pc, ps, pp, pl, 6000, st)
            want = plan_rules(old, new, page, table, ring, cursors, 6000, num_pages)
            got = (mem.down(pt), mem.down(pr), mem.down(pc), mem.down(ps), mem.down(pp), mem.down(pl), int(mem.down(st)[0]))
            same_plan(got, want)
            table, ring, cursors = want[0], want[1], want[2]
            if want[6] == 0:
                old = new
            held = np.concatenate([table[i, : -(-int(old[i]) // page)] for i in range(n)])
            free = ring[np.arange(cursors[0], cursors[1]) % num_pages]
            assert np.array_equal(np.sort(np.concatenate([held, free])), np.arange(num_pages))


def test_plan_operands_are_checked(gpu_ctx):
    with Arrays(gpu_ctx) as mem:
        n, w = 4, 3
        p = dict(old=mem.up(np.zeros(n, np.int32)), new=mem.up(np.zeros(n, np.int32)),
                 table=mem.up(np.zeros((n, w), np.int32)), ring=mem.up(np.zeros(10, np.int32)),
                 cin=mem.up(np.zeros(2, np.int64)), cout=mem.up(np.zeros(2, np.int64)),
                 starts=mem.up(np.zeros(n + 1, np.int32)), pos=mem.up(np.zeros(8, np.int32)),
                 slots=mem.up(np.zeros(8, np.int32)), status=mem.up(np.zeros(1, np.int32)))

        def call(n=n, w=w, stride=w, pages=10, rows=8, **kw):
            a = {**p, **kw}
            S.paged_plan(gpu_ctx, n, a["old"], a["new"], 16, a["table"], w, stride, a["ring"], pages, a["cin"],
                         a["cout"], a["starts"], a["pos"], a["slots"], rows, a["status"])

        # device allocations are rounded up inside the runtime, not in what a range query answers
        for kw, text in [(dict(n=5), "past the end"), (dict(stride=4), "past the end"), (dict(stride=2), "stride"),
                         (dict(pages=11), "past the end"), (dict(rows=9), "past the end"), (dict(old=0), "null"),
                         (dict(cin=p["cin"] + 4), "aligned"), (dict(status=0), "null"),
                         (dict(slots=np.zeros(8, np.int32).ctypes.data), "not in device memory"),
                         (dict(table=p["table"] + 2), "aligned")]:
            with pytest.raises(S.SocError, match=text) as e:
                call(**kw)
            assert e.value.code == SOC_ERR_INVALID
        call()
        gpu_ctx.synchronize()


# ---- append ----------------------------------------------------------------------------------------------------------
def run_append(ctx, dtype, rows, nq, nkv, hd, page, d=None, layout="half", pages=None, slots=None, stride=0, shift=0,
               page_stride=0, fused=True, in_place=False, rope=True, seed=1):
    rng = np.random.default_rng(seed)
    d = hd if d is None else d
    pages = -(-rows // page) + 3 if pages is None else pages
    row = (nq + 2 * nkv) * hd + stride
    qkv = (rng.standard_normal(shift + rows * row) * 2).astype(NP[dtype])
    x = qkv[shift:].reshape(rows, row)[:, : (nq + 2 * nkv) * hd].reshape(rows, -1, hd)
    if slots is None:
        slots = rng.permutation(pages * page)[:rows]
    slots = np.asarray(slots, np.int32)
    positions = rng.integers(0, 30000, rows).astype(np.int32)
    size = page_stride or nkv * page * hd
    # an infinity in the first place of every page must stay where it is
    pool = rng.standard_normal((2, pages, size)).astype(np.float16)
    qw = nq * hd
    with Arrays(ctx) as mem:
        pqkv, pk, pv = mem.up(qkv), mem.up(pool[0]), mem.up(pool[1])
        pp, ps = mem.up(positions), mem.up(slots)
        before = np.full((rows, qw + 5), 3.0, NP[dtype])
        pq = mem.up(before)
        item = qkv.itemsize
        base = pqkv + shift * item
        cache = S.PagedCache(pk, pv, pages, page, nkv, hd, page_stride)
        r = S.Rope(ctx, hd, d, layout=layout) if rope else None
        out, out_stride = (base, row) if in_place else (pq, qw + 5)
        S.paged_append(ctx, cache, r, base if nq else None, row, base + nq * hd * item, row,
                       base + (nq + nkv) * hd * item, row, dtype, out if nq else None, out_stride, rows, nq,
                       pp if rope else None, ps)
        keys, values, q = mem.down(pk), mem.down(pv), mem.down(pq)
        after = mem.down(pqkv)
        if r is not None:
            r.close()
    if rope:
        want, tol = rotate(x[:, : nq + nkv], positions, d, layout, frequencies(d, 1e6, "none", 1.0, 0), 1.0)
    else:
        want, tol = x[:, : nq + nkv].astype(np.float64), np.zeros_like(x[:, : nq + nkv], np.float64)
    live = (slots >= 0) & (slots < pages * page)
    wk, wv = pool.copy()
    written = np.zeros((pages, size), bool)
    for i in np.flatnonzero(live):
        p, o = divmod(int(slots[i]), page)
        for h in range(nkv):
            at = slice((h * page + o) * hd, (h * page + o + 1) * hd)
            rope_check(keys[p, at], want[i, nq + h], tol[i, nq + h], "f16")
            wv[p, at] = x[i, nq + nkv + h].astype(np.float16)
            written[p, at] = True
    wk[written] = keys[written]
    assert np.array_equal(keys.view(np.uint16), wk.view(np.uint16))  # nothing else is touched
    assert np.array_equal(values.view(np.uint16), wv.view(np.uint16))
    if nq:
        got = (after[shift:].reshape(rows, row) if in_place else q)[:, :qw].reshape(rows, nq, hd)
        rope_check(got[live], want[live, :nq], tol[live, :nq], dtype)
        kept = x[:, :nq].reshape(rows, qw) if in_place else before[:, :qw]
        assert np.array_equal(got.reshape(rows, qw)[~live], kept[~live])
    assert (q[:, qw:] == 3.0).all()
    rest = after[shift:].reshape(rows, row)[:, qw:] if in_place else after
    assert np.array_equal(rest, qkv[shift:].reshape(rows, row)[:, qw:] if in_place else qkv)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("nq,nkv,hd,page,d", [(16, 8, 128, 16, 128), (32, 8, 128, 64, 128), (14, 2, 64, 32, 64),
                                              (3, 1, 64, 256, 32), (5, 5, 128, 128, 6), (1, 1, 128, 16, 2)])
def test_append_shapes(gpu_ctx, dtype, layout, nq, nkv, hd, page, d):
    run_append(gpu_ctx, dtype, 19, nq, nkv, hd, page, d, layout)


@pytest.mark.parametrize("rows", [1, 2, 255, 1000])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_append_rows(gpu_ctx, rows, dtype):
    run_append(gpu_ctx, dtype, rows, 4, 2, 128, 32)


@pytest.mark.parametrize("stride,shift", [(0, 4), (4, 0), (3, 0), (8, 1), (1, 3)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("in_place", [False, True])
def test_append_strides(gpu_ctx, stride, shift, dtype, in_place):
    run_append(gpu_ctx, dtype, 9, 4, 2, 128, 16, stride=stride, shift=shift, in_place=in_place)


def test_append_into_an_interleaved_pool(gpu_ctx):
    run_append(gpu_ctx, "f32", 40, 4, 2, 128, 16, page_stride=2 * 16 * 128 * 3 + 8)


def test_append_without_queries_and_without_rotation(gpu_ctx):
    run_append(gpu_ctx, "f32", 9, 0, 2, 128, 16)
    run_append(gpu_ctx, "f16", 9, 0, 3, 64, 32, rope=False)
    run_append(gpu_ctx, "f32", 9, 0, 3, 64, 32, rope=False, stride=3, shift=1)


def test_append_skips_rows_without_a_slot(gpu_ctx):
    """Padding (-1) and slots that are none of the cache's: nothing is stored and the query rows stay."""
    slots = [5, -1, 47, 48, -2 ** 31, 2 ** 31 - 1, 0, -1, -1]
    for in_place in (False, True):
        run_append(gpu_ctx, "f32", 9, 4, 2, 128, 16, pages=3, slots=slots, in_place=in_place)
    run_append(gpu_ctx, "f32", 4, 4, 2, 128, 16, pages=3, slots=[-1] * 4)


def test_append_rounds_to_fp16(gpu_ctx):
    """Values beyond fp16 become infinities, subnormals stay, ties go to even."""
    x = np.array([65519.0, 65520.0, -1e30, 2.0 ** -24, 2.0 ** -25, 3 * 2.0 ** -26, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11,
                  np.inf, np.nan, -0.0, 1e-30], np.float32)
    v = np.resize(x, (1, 128)).astype(np.float32)
    with Arrays(gpu_ctx) as mem:
        pv, pk, pv2 = mem.up(v), mem.up(np.zeros((1, 16, 128), np.float16)), mem.up(np.zeros((1, 16, 128), np.float16))
        S.paged_append(gpu_ctx, S.PagedCache(pk, pv2, 1, 16, 1, 128), None, None, 0, pv, 128, pv, 128, "f32", None, 0, 1,
                       0, None, mem.up(np.array([3], np.int32)))
        with np.errstate(over="ignore"):
            want = v[0].astype(np.float16)
        for p in (pk, pv2):
            got = mem.down(p)[0]
            assert np.array_equal(got[3], want, equal_nan=True)
            assert (np.delete(got, 3, 0) == 0).all()


# ---- decode attention --------------------------------------------------------------------------------------------------
def attend(q, k, v, scale):
    """q [nq][hd], k / v [nkv][len][hd] -> (out, lse, tolerances) in 64 bits."""
    nq, hd, nkv = q.shape[0], q.shape[1], k.shape[0]
    out, lse = np.zeros((nq, hd)), np.full(nq, -np.inf)
    tol, tol_lse = np.zeros((nq, hd)), np.zeros(nq)
    if k.shape[1] == 0:
        return out, lse, tol, tol_lse
    for h in range(nq):
        kh, vh = k[h // (nq // nkv)].astype(np.float64), v[h // (nq // nkv)].astype(np.float64)
        qh = q[h].astype(np.float64)
        s = kh @ qh * scale
        e = (hd + 8) * 2.0 ** -24 * (np.abs(kh) @ np.abs(qh)).max() * abs(scale)
        m = s.max()
        p = np.exp(s - m)
        out[h], lse[h] = p @ vh / p.sum(), m + np.log(p.sum())
        tol[h] = (2 * e + 520 * 2.0 ** -24 + 2.0 ** -21) * np.abs(vh).max()
        tol_lse[h] = e + 520 * 2.0 ** -24 + 2.0 ** -23 * abs(lse[h])
    return out, lse, tol, tol_lse


def run_attention(ctx, dtype, lens, nq, nkv, hd, page, scale=0.0, pages=None, width=None, page_stride=0, q_pad=0,
                  o_pad=0, extra=0, shift=0, in_place=False, lse=True, q_scale=1.0, kv=None, garbage=np.nan, table=None,
                  verify=True, seed=1):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int64)
    n, qw = lens.size, nq * hd
    held = -(-np.maximum(lens, 0) // page)
    width = max(1, int(held.max())) if width is None else width
    if table is None:
        pages = int(held.sum()) + 2 if pages is None else pages
        order = rng.permutation(pages)[: int(held.sum())].astype(np.int32)
        table = np.full((n, width), 2 ** 31 - 1, np.int32)  # entries behind a row's pages are not read as pages
        table[np.arange(width)[None, :] < held[:, None]] = order
    else:
        pages, width = pages or int(table.max()) + 1, table.shape[1]
    size = page_stride or nkv * page * hd
    pool = np.full((2, pages, size), garbage, np.float16)  # whatever is not a cached position holds `garbage`
    rows = []
    for b in range(n if verify is not False else 0):
        k = rng.standard_normal((nkv, max(0, lens[b]), hd)).astype(np.float16)
        v = rng.standard_normal((nkv, max(0, lens[b]), hd)).astype(np.float16)
        if kv is not None:
            k, v = kv(b, k, v)
        rows.append((k, v))
        for j in range(int(held[b])):
            m = min(page, int(lens[b]) - j * page)
            for which, src in enumerate((k, v)):
                dst = pool[which, table[b, j], : nkv * page * hd].reshape(nkv, page, hd)
                dst[:, :m] = src[:, j * page: j * page + m]
    q = np.full(shift + n * (qw + q_pad), 5.0, NP[dtype])
    qs = (rng.standard_normal((n, qw)) * q_scale).astype(NP[dtype])
    q[shift:].reshape(n, qw + q_pad)[:, :qw] = qs
    wide = np.full((n, width + extra), -5, np.int32)
    wide[:, :width] = table
    before = np.full((n, qw + o_pad), 7.0, NP[dtype])
    with Arrays(ctx) as mem:
        pk, pv, pq, pt = mem.up(pool[0]), mem.up(pool[1]), mem.up(q), mem.up(wide)
        po = mem.up(before)
        pl = mem.up(np.full(n * nq + 1, 7.0, np.float32))
        cache = S.PagedCache(pk, pv, pages, page, nkv, hd, page_stride)
        at = pq + shift * q.itemsize
        S.paged_attention_decode(ctx, cache, at, qw + q_pad, dtype, pt, width + extra, width,
                                 mem.up(lens.astype(np.int32)), n, nq, scale, at if in_place else po,
                                 qw + (q_pad if in_place else o_pad), pl if lse else None)
        out, gl = (mem.down(pq)[shift:] if in_place else mem.down(po)).reshape(n, -1), mem.down(pl)
        assert np.array_equal(mem.down(pk).view(np.uint16), pool[0].view(np.uint16))
    assert (out[:, qw:] == (5.0 if in_place else 7.0)).all() and gl[-1] == 7.0
    out, gl = out[:, :qw].reshape(n, nq, hd), gl[:-1].reshape(n, nq)
    if verify:
        for b in range(n):
            want, wl, tol, tol_l = attend(qs[b].reshape(nq, hd), *rows[b], scale or 1 / math.sqrt(hd))
            if dtype == "f16":
                tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
            worst = np.max(np.abs(out[b].astype(np.float64) - want) - tol)
            assert worst <= 0, (b, int(lens[b]), worst)
            if lse:
                same = (gl[b] == -np.inf) & (wl == -np.inf)
                with np.errstate(invalid="ignore"):
                    assert (same | (np.abs(gl[b] - wl) <= tol_l)).all(), (b, gl[b], wl)
    if not lse:
        assert (gl == 7.0).all()
    return out, gl


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_lengths(gpu_ctx, hd, page):
    """Every way a length can end in a tile and a page; what lies behind it is NaN."""
    lens = [0, 1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511,
            512, 513, 1023, 1025, 2049, 0]
    run_attention(gpu_ctx, "f32", lens, 4, 2, hd, page)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 8), (2, 1), (3, 1), (16, 8), (5, 1), (12, 2), (7, 1), (32, 8), (8, 1),
                                    (9, 1), (14, 2), (48, 4), (13, 1), (32, 2)])
def test_attention_head_groups(gpu_ctx, dtype, nq, nkv):
    run_attention(gpu_ctx, dtype, [70, 1, 33, 0, 600], nq, nkv, 128, 16)
    run_attention(gpu_ctx, dtype, [200], nq, nkv, 64, 64)


@pytest.mark.parametrize("lens", [[1], [4071], [10000], [20001, 3], [1] * 300, [600] * 70])
def test_attention_batches(gpu_ctx, lens):
    run_attention(gpu_ctx, "f32", lens, 8, 2, 128, 32)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_of_many_ragged_rows(gpu_ctx, dtype):
    """Rows enough that blocks take up to 2048 keys: lengths around one block and two, and short ones among them."""
    lens = np.random.default_rng(9).integers(0, 70, 1600)
    lens[::100] = [2047, 2048, 2049, 4096, 4097, 1024, 1025, 0, 1, 1500, 2100, 3000, 768, 769, 128, 129]
    run_attention(gpu_ctx, dtype, lens.tolist(), 5, 1, 64, 16, width=300)


def test_attention_of_a_wide_table(gpu_ctx):
    """A table far wider than any sequence: lengths on the device decide, not the width."""
    a, la = run_attention(gpu_ctx, "f32", [40, 3000, 0, 17], 8, 2, 128, 16)
    b, lb = run_attention(gpu_ctx, "f32", [40, 3000, 0, 17], 8, 2, 128, 16, width=20000)
    # another split of the keys: the two agree as each does with the formula
    assert np.max(np.abs(a - b)) < 1e-4 and a.shape == b.shape
    assert np.array_equal(np.isfinite(la), np.isfinite(lb))


@pytest.mark.parametrize("q_pad,o_pad,extra,shift", [(8, 0, 0, 0), (0, 3, 2, 0), (3, 0, 0, 1), (1, 1, 7, 2), (4, 4, 0, 4)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_strides(gpu_ctx, q_pad, o_pad, extra, shift, dtype):
    lens = [100, 7, 0, 1500]
    run_attention(gpu_ctx, dtype, lens, 6, 2, 128, 16, q_pad=q_pad, o_pad=o_pad, extra=extra, shift=shift)
    run_attention(gpu_ctx, dtype, lens, 6, 2, 64, 16, q_pad=q_pad, extra=extra, shift=shift, in_place=True)


def test_attention_of_an_interleaved_pool(gpu_ctx):
    run_attention(gpu_ctx, "f32", [100, 300], 8, 2, 128, 16, page_stride=2 * 16 * 128 * 2 + 64)


def test_attention_without_lse(gpu_ctx):
    a, _ = run_attention(gpu_ctx, "f32", [100, 0, 2000], 8, 2, 128, 16, lse=False)
    b, _ = run_attention(gpu_ctx, "f32", [100, 0, 2000], 8, 2, 128, 16)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("scale", [1.0, 0.02, -0.3, 3.0])
def test_attention_scales(gpu_ctx, scale):
    run_attention(gpu_ctx, "f32", [70, 900], 8, 2, 128, 16, scale=scale)


@pytest.mark.parametrize("q_scale", [1e-30, 1e-6, 100.0, 1e5, 1e7])
def test_attention_query_magnitudes(gpu_ctx, q_scale):
    """Queries far below and above what 16 bits hold: their scores keep 32-bit accuracy."""
    run_attention(gpu_ctx, "f32", [70, 900, 5], 8, 2, 128, 16, q_scale=q_scale)


def test_attention_large_and_small_cached_values(gpu_ctx):
    """The ends of fp16's range, subnormals among them; scores that leave one key."""
    def big(b, k, v):
        return k * np.float16(200), (v.astype(np.float32) * 20000).clip(-65504, 65504).astype(np.float16)

    def small(b, k, v):
        return k, (v.astype(np.float32) * 2.0 ** -22).astype(np.float16)

    run_attention(gpu_ctx, "f32", [70, 900, 5], 8, 2, 128, 16, kv=big)
    run_attention(gpu_ctx, "f32", [70, 900, 5], 8, 2, 128, 16, kv=small)


def test_attention_rising_and_falling_scores(gpu_ctx):
    """The running maximum moves at every key, or never."""
    def slope(b, k, v):
        t = np.linspace(0, 40, k.shape[1])[None, :, None] * (1 if b == 0 else -1)
        return (k * 0.1 + t).astype(np.float16), v

    run_attention(gpu_ctx, "f32", [3000, 3000], 4, 1, 128, 16, kv=slope)


@pytest.mark.parametrize("garbage", [np.inf, -np.inf, 65504.0])
def test_attention_ignores_what_lies_behind_the_length(gpu_ctx, garbage):
    run_attention(gpu_ctx, "f32", [1, 17, 35, 1000], 8, 2, 128, 32, garbage=garbage)


def test_attention_of_shared_pages(gpu_ctx):
    """Sequences with a common prefix name the same pages."""
    rng = np.random.default_rng(2)
    shared = rng.standard_normal((2, 2, 64, 128)).astype(np.float16)
    table = np.array([[3, 1, 0, 9], [3, 1, 5, 9], [3, 1, 9, 9]], np.int32)

    def kv(b, k, v):
        k, v = k.copy(), v.copy()
        k[:, :64], v[:, :64] = shared[0], shared[1]
        return k, v

    run_attention(gpu_ctx, "f32", [90, 70, 64], 8, 2, 128, 32, kv=kv, table=table, pages=10)


def test_attention_non_finite_values_it_attends_to(gpu_ctx):
    """A NaN or infinity that is attended to makes the heads of its KV head not finite; other heads and rows keep theirs."""
    for which in ("k", "v"):
        for bad in (np.nan, np.inf):
            def kv(b, k, v):
                if b == 1:
                    (k if which == "k" else v)[0, 150] = bad
                return k, v

            out, _ = run_attention(gpu_ctx, "f32", [200, 200, 200], 8, 2, 128, 16, kv=kv, verify=None)
            assert not np.isfinite(out[1, :4]).any()
            assert np.isfinite(out[1, 4:]).all() and np.isfinite(out[[0, 2]]).all()


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 40, 2 ** 31 - 1])
def test_attention_of_a_table_with_foreign_pages(gpu_ctx, bad):
    """A page that is none of the cache's within a row's length: that row is NaN, the others are not."""
    table = np.arange(40, dtype=np.int32).reshape(4, 10)
    table[1, 0] = table[2, 9] = bad
    table[3, 9] = bad  # behind the row's length: not looked at
    out, lse = run_attention(gpu_ctx, "f32", [160, 160, 150, 144], 8, 2, 128, 16, table=table, pages=40, verify=False,
                             garbage=0.5)
    assert np.isfinite(out[[0, 3]]).all() and np.isfinite(lse[[0, 3]]).all()
    assert np.isnan(out[[1, 2]]).all() and np.isnan(lse[[1, 2]]).all()
    assert np.max(np.abs(out[[0, 3]] - 0.5)) < 1e-4


def test_attention_of_foreign_lengths(gpu_ctx):
    """Lengths below zero are empty; beyond the table, NaN: no entry behind the row is looked at."""
    table = np.arange(40, dtype=np.int32).reshape(4, 10)
    out, lse = run_attention(gpu_ctx, "f32", [-1, 161, 2 ** 31 - 1, -2 ** 31], 8, 2, 128, 16, table=table, pages=40,
                             width=10, verify=False, garbage=0.5)
    assert (out[[0, 3]] == 0).all() and (lse[[0, 3]] == -np.inf).all()
    assert np.isnan(out[[1, 2]]).all() and np.isnan(lse[[1, 2]]).all()


def test_attention_joins_by_lse(gpu_ctx):
    """Attention over two parts of the keys, joined by their log sums, is the attention over all of them."""
    rng = np.random.default_rng(3)
    keys, values = (rng.standard_normal((12, 2, 16, 64)).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((1, 6 * 64)).astype(np.float32)
    parts = []
    with Arrays(gpu_ctx) as mem:
        cache = S.PagedCache(mem.up(keys), mem.up(values), 12, 16, 2, 64)
        pq = mem.up(q)
        for table, length in (([0, 1, 2, 3, 4, 5, 6], 100), ([0, 1, 2], 48), ([3, 4, 5, 6], 52)):
            po, pl = mem.up(np.zeros((1, 384), np.float32)), mem.up(np.zeros((1, 6), np.float32))
            S.paged_attention_decode(gpu_ctx, cache, pq, 384, "f32", mem.up(np.array(table, np.int32)), len(table),
                                     len(table), mem.up(np.array([length], np.int32)), 1, 6, 0.0, po, 384, pl)
            parts.append((mem.down(po).reshape(6, 64).astype(np.float64), mem.down(pl)[0].astype(np.float64)))
    (whole, l0), (a, la), (b, lb) = parts
    joined = (np.exp(la - l0)[:, None] * a + np.exp(lb - l0)[:, None] * b)
    assert np.max(np.abs(joined - whole)) < 1e-4
    assert np.max(np.abs(np.logaddexp(la, lb) - l0)) < 1e-4


def test_attention_bits_do_not_depend_on_timing_or_company(gpu_ctx):
    """Equal calls give equal bits, also after calls of other sizes used the workspace."""
    first = run_attention(gpu_ctx, "f32", [5000, 3, 700, 0, 4097], 32, 8, 128, 16)
    run_attention(gpu_ctx, "f32", [9000], 8, 1, 64, 64)
    run_attention(gpu_ctx, "f16", [300] * 100, 16, 8, 128, 32)
    again = run_attention(gpu_ctx, "f32", [5000, 3, 700, 0, 4097], 32, 8, 128, 16)
    assert np.array_equal(first[0].view(np.uint32), again[0].view(np.uint32))
    assert np.array_equal(first[1].view(np.uint32), again[1].view(np.uint32))


def test_attention_agrees_with_the_contiguous_one(gpu_ctx):
    """One sequence whose pages lie in order is soc_attention_decode over a plane of that capacity."""
    rng = np.random.default_rng(4)
    n, cap = 1000, 1024
    keys, values = (rng.standard_normal((2, cap, 128)).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((1, 8 * 128)).astype(np.float32)
    paged = [np.ascontiguousarray(t.reshape(2, cap // 64, 64, 128).transpose(1, 0, 2, 3)) for t in (keys, values)]
    with Arrays(gpu_ctx) as mem:
        pq, pa, pb = mem.up(q), mem.up(np.zeros_like(q)), mem.up(np.zeros_like(q))
        S.attention_decode(gpu_ctx, pq, mem.up(keys), mem.up(values), pa, n, 8, 2, cap)
        cache = S.PagedCache(mem.up(paged[0]), mem.up(paged[1]), 16, 64, 2, 128)
        S.paged_attention_decode(gpu_ctx, cache, pq, 1024, "f32", mem.up(np.arange(16, dtype=np.int32)), 16, 16,
                                 mem.up(np.array([n], np.int32)), 1, 8, 0.0, pb, 1024)
        a, b = mem.down(pa), mem.down(pb)
    _, _, tol, _ = attend(q.reshape(8, 128), keys[:, :n], values[:, :n], 1 / math.sqrt(128))
    assert (np.abs(a - b).reshape(8, 128) <= 2 * tol).all()


def test_attention_beyond_32_bit_offsets(gpu_ctx):
    """A pool of more than 2^32 bytes and elements behind 2^31: the last pages are reached, not their 32-bit wraps."""
    page, nkv, hd = 256, 8, 128
    per = nkv * page * hd
    pages = (1 << 32) // per + 9  # > 2^32 elements each of keys and values
    rng = np.random.default_rng(5)
    ctx = gpu_ctx
    k, v = (rng.standard_normal((3, nkv, page, hd)).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((1, 16 * hd)).astype(np.float32)
    pk, pv = ctx.alloc(pages * per * 2), ctx.alloc(pages * per * 2)
    ids = np.array([[pages - 1, 2, pages - 5]], np.int32)
    try:
        with Arrays(ctx) as mem:
            for i, p in enumerate(ids[0]):
                ctx.write(pk + int(p) * per * 2, k[i])
                ctx.write(pv + int(p) * per * 2, v[i])
            cache = S.PagedCache(pk, pv, pages, page, nkv, hd)
            po = mem.up(np.zeros_like(q))
            S.paged_attention_decode(ctx, cache, mem.up(q), 2048, "f32", mem.up(ids), 3, 3,
                                     mem.up(np.array([700], np.int32)), 1, 16, 0.0, po, 2048)
            got = mem.down(po).reshape(16, hd)
            # and a key and value appended to the last page
            row = rng.standard_normal((1, 2 * nkv * hd)).astype(np.float32)
            pr = mem.up(row)
            S.paged_append(ctx, cache, None, None, 0, pr, 2048, pr + 4096, 2048, "f32", None, 0, 1, 0, None,
                           mem.up(np.array([pages * page - 1], np.int32)))
            ctx.synchronize()
            last = ctx.download(pv + (pages - 1) * per * 2, (nkv, page, hd), np.float16)
            assert np.array_equal(last[:, -1].reshape(-1), row[0, 1024:].astype(np.float16))
    finally:
        ctx.synchronize()
        ctx.free(pk)
        ctx.free(pv)
    whole = [t.transpose(1, 0, 2, 3).reshape(nkv, 3 * page, hd)[:, :700] for t in (k, v)]
    want, _, tol, _ = attend(q.reshape(16, hd), *whole, 1 / math.sqrt(hd))
    assert (np.abs(got - want) <= tol).all()


def test_cache_operands_are_checked(gpu_ctx):
    with Arrays(gpu_ctx) as mem:
        pool = np.zeros((4, 2, 16, 64), np.float16)
        pk, pv, q, o = mem.up(pool), mem.up(pool), mem.up(np.zeros((3, 256), np.float32)), mem.up(np.zeros((3, 256), np.float32))
        t, n, l = mem.up(np.zeros((3, 2), np.int32)), mem.up(np.zeros(3, np.int32)), mem.up(np.zeros((3, 4), np.float32))

        def call(pages=4, stride=0, q=q, qs=256, t=t, ts=2, w=2, lens=n, rows=3, out=o, os=256, lse=l, k=pk, v=pv):
            S.paged_attention_decode(gpu_ctx, S.PagedCache(k, v, pages, 16, 2, 64, stride), q, qs, "f32", t, ts, w, lens,
                                     rows, 4, 0.0, out, os, lse)

        for kw, text in [(dict(pages=5), "past the end"), (dict(stride=2056), "past the end"), (dict(qs=257), "past the end"),
                         (dict(qs=255), "stride"), (dict(rows=4), "past the end"), (dict(ts=3), "past the end"),
                         (dict(ts=1), "stride"), (dict(lens=n + 4), "past the end"), (dict(os=300), "past the end"),
                         (dict(lse=l + 4), "past the end"), (dict(q=0), "null"), (dict(out=o + 1), "aligned"),
                         (dict(v=pool.ctypes.data // 16 * 16), "not in device memory"), (dict(t=0), "null")]:
            with pytest.raises(S.SocError, match=text) as e:
                call(**kw)
            assert e.value.code == SOC_ERR_INVALID
        call()
        gpu_ctx.synchronize()
        other = S.Context(0)
        rope = S.Rope(other, 64)
        try:
            x = mem.up(np.zeros((3, 256), np.float32))
            with pytest.raises(S.SocError, match="another context"):
                S.paged_append(gpu_ctx, S.PagedCache(pk, pv, 4, 16, 2, 64), rope, None, 0, x, 256, x + 512, 256, "f32", None,
                               0, 3, 0, n, n)
        finally:
            rope.close()
            other.close()


# ---- a serving step --------------------------------------------------------------------------------------------------
def test_steps_of_a_paged_server(gpu_ctx):
    """Prompts, decodes, a rollback and a finished request through plan, append, attention and logprobs in one set of
    buffers: what each decode row attends to is what a plain cache of its own would hold, in 64 bits."""
    ctx, rng = gpu_ctx, np.random.default_rng(10)
    n, nq, nkv, hd, page, num_pages, width, max_rows, vocab = 4, 8, 2, 64, 16, 24, 9, 128, 1003
    f = frequencies(hd, 1e6, "none", 1.0, 0)
    row = (nq + 2 * nkv) * hd
    steps = [([0, 0, 0, 0], [37, 0, 5, 60]), ([37, 0, 5, 60], [38, 70, 6, 61]), ([38, 70, 6, 61], [39, 71, 7, 0]),
             ([39, 71, 7, 0], [33, 72, 8, 16]), ([33, 72, 8, 16], [34, 73, 9, 17]), ([34, 73, 9, 17], [35, 0, 0, 18])]
    head = rng.standard_normal((nq * hd, vocab)).astype(np.float32) * 0.2
    plain = [[np.zeros((nkv, 0, hd)), np.zeros((nkv, 0, hd))] for _ in range(n)]
    with Arrays(ctx) as mem:
        z = lambda *s, t=np.int32: mem.up(np.zeros(s, t))  # noqa: E731
        po, pn, pt, pr = z(n), z(n), z(n, width), mem.up(rng.permutation(num_pages).astype(np.int32))
        pc, ps, pp, pl, st = mem.up(np.array([0, num_pages], np.int64)), z(n + 1), z(max_rows), z(max_rows), z(1)
        pk, pv = (mem.up(np.full((num_pages, nkv, page, hd), np.nan, np.float16)) for _ in range(2))
        pqkv, pq = z(max_rows, row, t=np.float32), z(max_rows, nq * hd, t=np.float32)
        pdq, pout, plse = z(n, nq * hd, t=np.float32), z(n, nq * hd, t=np.float32), z(n, nq, t=np.float32)
        plog, ptok, plp, pen = z(n, vocab, t=np.float32), z(n), z(n, t=np.float32), z(n, t=np.float32)
        pid, ptl = z(n, 5), z(n, 5, t=np.float32)
        cache, rope = S.PagedCache(pk, pv, num_pages, page, nkv, hd), S.Rope(ctx, hd)
        try:
            for old, new in steps:
                total = sum(max(0, b - a) for a, b in zip(old, new))
                x = rng.standard_normal((max_rows, row)).astype(np.float32)
                ctx.write(po, np.array(old, np.int32))
                ctx.write(pn, np.array(new, np.int32))
                ctx.write(pqkv, x)
                # queued one behind the other, padding rows among them
                S.paged_plan(ctx, n, po, pn, page, pt, width, width, pr, num_pages, pc, pc, ps, pp, pl, max_rows, st)
                S.paged_append(ctx, cache, rope, pqkv, row, pqkv + 4 * nq * hd, row, pqkv + 4 * (nq + nkv) * hd, row, "f32",
                               pq, nq * hd, max_rows, nq, pp, pl)
                assert mem.down(st)[0] == 0
                starts = mem.down(ps)
                assert starts[-1] == total
                q = mem.down(pq)
                last = np.zeros((n, nq * hd), np.float32)
                h = x.reshape(max_rows, -1, hd)
                for i in range(n):
                    k, v = (t[:, : new[i]] for t in plain[i])
                    at = np.arange(starts[i], starts[i + 1])
                    turned, _ = rotate(h[at, : nq + nkv], np.arange(old[i], old[i] + at.size), hd, "half", f, 1.0)
                    k = np.concatenate([k, turned[:, nq:].astype(np.float32).astype(np.float16).transpose(1, 0, 2)], 1)
                    v = np.concatenate([v, h[at, nq + nkv:].astype(np.float16).transpose(1, 0, 2)], 1)
                    plain[i] = [k, v]
                    assert k.shape[1] == new[i]
                    if at.size:
                        last[i] = q[at[-1]]
                ctx.write(pdq, last)
                S.paged_attention_decode(ctx, cache, pdq, nq * hd, "f32", pt, width, width, pn, n, nq, 0.0, pout, nq * hd,
                                         plse)
                out = mem.down(pout)
                logits = (out @ head).astype(np.float32)
                tokens = rng.integers(0, vocab, n).astype(np.int32)
                ctx.write(plog, logits)
                ctx.write(ptok, tokens)
                S.logprobs(ctx, plog, "f32", vocab, n, vocab, 1.0, ptok, plp, None, pen, 5, pid, ptl)
                lp, ids = mem.down(plp), mem.down(pid)
                table, keys = mem.down(pt), mem.down(pk)
                for i in range(n):
                    mine = keys[table[i, : -(-new[i] // page)]].transpose(1, 0, 2, 3).reshape(nkv, -1, hd)[:, : new[i]]
                    # a key may round to its other fp16 neighbour: one step, then the cached one is what counts
                    assert (np.abs(mine - plain[i][0]) <= 2.0 ** -10 * np.abs(plain[i][0]) + 2.0 ** -24).all()
                    plain[i][0] = mine
                    want, _, tol, _ = attend(last[i].reshape(nq, hd), mine, plain[i][1], 1 / math.sqrt(hd))
                    assert (np.abs(out[i].reshape(nq, hd) - want) <= tol).all(), (i, new)
                    e = np.exp(logits[i].astype(np.float64) - logits[i].max())
                    p = np.log(e / e.sum())
                    assert abs(lp[i] - p[tokens[i]]) < 1e-4
                    assert np.array_equal(ids[i], np.lexsort((np.arange(vocab), -logits[i].astype(np.float64)))[:5])
        finally:
            rope.close()
