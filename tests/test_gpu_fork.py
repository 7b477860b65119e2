"""Rows that go on from other rows: soc_paged_fork and soc_paged_compact against their rules in Python, one row and page after
the other, and soc_paged_copy against numpy. All of it is whole numbers and moved bits: equal or wrong."""
import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import PLAN_CURSORS, PLAN_LENGTHS, PLAN_PAGES, SOC_ERR_INVALID
from tests.device import Arrays, guarded

pytestmark = pytest.mark.gpu


def pages_of(n, page):
    return -(-int(n) // page)


def fork_rules(parents, keep, old, page, table, new_table, ring, cursors, num_pages):
    """soc_paged_fork's contract: (new_table, ring, cursors, new_lens, next_lens, copies, status)."""
    n, width = table.shape
    new_table, ring = new_table.copy(), ring.copy()
    head, tail = (int(c) for c in cursors)
    old = [int(x) for x in old]
    lost = [o < 0 or pages_of(o, page) > width for o in old]
    status, length = 0, [0] * n
    for i, p in enumerate(int(x) for x in parents):
        if lost[i]:
            status |= PLAN_LENGTHS
        if p == -1:
            continue
        k = None if not 0 <= p < n else old[p] if keep is None else int(keep[i])
        if k is None or lost[p] or not 0 <= k <= old[p]:
            status |= PLAN_LENGTHS
        else:
            length[i] = k
    heirs, copied = {}, []
    for i, p in enumerate(int(x) for x in parents):
        if length[i] % page:
            inherits = old[p] % page != 0 and pages_of(old[p], page) == pages_of(length[i], page)
            if not (inherits and heirs.setdefault(p, i) == i):
                copied.append(i)
    if head < 0 or tail < 0 or not 0 <= tail - head <= num_pages:
        status |= PLAN_CURSORS
    elif len(copied) > tail - head:
        status |= PLAN_PAGES
    if status:
        for i in range(n):
            if not lost[i]:
                new_table[i, : pages_of(old[i], page)] = table[i, : pages_of(old[i], page)]
        return new_table, ring, [head, tail], old, old, [], status
    copies = []
    for i in range(n):
        e = pages_of(length[i], page)
        new_table[i, :e] = table[parents[i], :e] if e else new_table[i, :e]
        if i in set(copied) if len(copied) < 50 else i in copied:
            to = int(ring[head % num_pages])
            head += 1
            copies.append([int(table[parents[i], e - 1]), to, length[i] % page])
            new_table[i, e - 1] = to
    named = {int(x) for i in range(n) for x in new_table[i, : pages_of(length[i], page)]}
    given, last = [], {}
    for i in range(n):
        e = pages_of(length[i], page)
        for j in range(pages_of(old[i], page)):
            a = int(table[i, j])
            if (j >= e or new_table[i, j] != a) and 0 <= a < num_pages and a not in named:
                last[a] = len(given)
                given.append(a)
    given = [a for t, a in enumerate(given) if last[a] == t]
    for a in given[: num_pages - (tail - head)]:
        ring[tail % num_pages] = a
        tail += 1
    nexts = [length[i] + 1 if parents[i] >= 0 else 0 for i in range(n)]
    return new_table, ring, [head, tail], length, nexts, copies, 0


def run_fork(ctx, parents, keep, old, page, table, ring, cursors, alias=False, extra=0, want_next=True):
    n, width = table.shape
    wide = np.full((n, width + extra), 77, np.int32)
    wide[:, :width] = table
    with Arrays(ctx) as mem:
        par, po = mem.up(np.asarray(parents, np.int32)), mem.up(np.asarray(old, np.int32))
        pk = None if keep is None else mem.up(np.asarray(keep, np.int32))
        pt, pr, pc = mem.up(wide), mem.up(ring), mem.up(np.asarray(cursors, np.int64))
        pn = mem.up(np.full((n, width + extra), 66, np.int32))
        pc2 = pc if alias else mem.up(np.full(2, 5, np.int64))
        outs = [mem.up(guarded(np.full(k, 99, np.int32), 2, 3, 55)) for k in (n, n, 3 * n, 1, 1)]
        S.paged_fork(ctx, n, par, pk, po, page, pt, pn, width, width + extra, pr, ring.size, pc, pc2, outs[0] + 8,
                     outs[1] + 8 if want_next else None, outs[2] + 8, outs[3] + 8, outs[4] + 8)
        lens, nexts, copies, count, status = (mem.down(p) for p in outs)
        for g in (lens, nexts, copies, count, status):
            assert (g[:2] == 55).all() and (g[-3:] == 55).all()
        if not want_next:
            assert (nexts[2:-3] == 99).all()
        t = mem.down(pn)
        assert (t[:, width:] == 66).all() and np.array_equal(mem.down(pt), wide)
        count = int(count[2])
        assert (copies[2 + 3 * count: -3] == 99).all()
        return (t[:, :width], mem.down(pr), mem.down(pc2), lens[2:-3], nexts[2:-3] if want_next else None,
                copies[2: 2 + 3 * count].reshape(-1, 3), int(status[2]))


def same_fork(got, want):
    for name, g, w in zip(("table", "ring", "cursors", "new_lens", "next_lens", "copies"), got, want):
        if g is not None:
            assert np.array_equal(np.asarray(g, np.int64).reshape(-1), np.asarray(w, np.int64).reshape(-1)), name
    assert got[6] == want[6]


def check_fork(ctx, parents, keep, old, page, table, ring, cursors, status=0, **kw):
    want = fork_rules(parents, keep, old, page, table, np.full(table.shape, 66, np.int32), ring, cursors, ring.size)
    assert want[6] == status
    same_fork(run_fork(ctx, parents, keep, old, page, table, ring, cursors, **kw), want)
    return want


def pool(rng, n, width, page, spare, longest=None, shared=True, start=0):
    """Rows that share pages from the front: row i begins as a row before it for part of its length."""
    old = rng.integers(0, (longest or width * page) + 1, n)
    table = np.full((n, width), -1, np.int32)
    free = list(rng.permutation(int(sum(-(-old // page))) + spare).astype(np.int32))
    num_pages = len(free)
    for i in range(n):
        e, k = pages_of(old[i], page), 0
        if shared and i and rng.random() < 0.6:
            j = int(rng.integers(0, i))
            k = int(rng.integers(0, min(old[i], old[j]) // page + 1))
            table[i, :k] = table[j, :k]
        for c in range(k, e):
            table[i, c] = free.pop()
    ring = np.full(num_pages, -7, np.int32)
    ring[(start + np.arange(len(free))) % num_pages] = free
    return old, table, ring, np.array([start, start + len(free)], np.int64)


def some_parents(rng, n, old):
    parents = rng.integers(-1, n, n)
    kind = rng.random(n)
    parents[kind < 0.3] = np.arange(n)[kind < 0.3]
    keep = np.where(parents >= 0, old[np.maximum(parents, 0)], rng.integers(-9, 9, n))
    less = (rng.random(n) < 0.3) & (parents >= 0)
    keep[less] = rng.integers(0, keep[less] + 1)
    return parents, keep


# rows x width: one block (up to 2048 entries) and three launches, chunks of 256 columns, 256 / 1024 / 4096 rows
@pytest.mark.parametrize("n,width,page", [
    (1, 1, 16), (1, 70, 16), (2, 3, 256), (4, 63, 16), (16, 100, 32), (1000, 2, 16), (8, 255, 32), (64, 256, 16), (1000, 16, 64), (1024, 16, 16),
    (65, 256, 16), (1025, 3, 16), (4096, 4, 16), (4096, 5, 128), (3, 9000, 16), (20, 1030, 32), (300, 70, 16), (700, 513, 16)])
def test_fork_mixed(gpu_ctx, n, width, page):
    rng = np.random.default_rng(n * 31 + width)
    longest = min(width * page, 40 * page) if n > 100 else None
    old, table, ring, cursors = pool(rng, n, width, page, 2 * n + 3, longest, start=int(rng.integers(0, 1 << 40)))
    parents, keep = some_parents(rng, n, old)
    check_fork(gpu_ctx, parents, keep, old, page, table, ring, cursors)
    check_fork(gpu_ctx, parents, keep, old, page, table, ring, cursors, alias=True, extra=5)
    check_fork(gpu_ctx, parents, None, old, page, table, ring, cursors, want_next=False)
    check_fork(gpu_ctx, np.arange(n), None, old, page, table, ring, cursors)  # nothing changes
    want = check_fork(gpu_ctx, np.full(n, -1), keep, old, page, table, ring, cursors)  # everything ends
    assert want[2][1] - want[2][0] == ring.size


@pytest.mark.parametrize("small", [True, False])
@pytest.mark.parametrize("parents,keep,old", [
    ([0], [0], [0]), ([0], [0], [20]), ([0], [5], [20]), ([0], [16], [20]), ([0], [17], [32]), ([-1], [3], [20]),
    ([0, 0], [20, 20], [20, 0]), ([1, 1], [20, 20], [7, 20]), ([1, 0], [20, 7], [7, 20]), ([0, 0, 0], [32, 20, 17], [32, 1, 1]),
    ([0, 0, 0], [20, 18, 16], [20, 0, 0]), ([2, 2, 2], [1, 2, 3], [48, 48, 3]), ([-1, -1, 0], [0, 0, 33], [33, 33, 33]),
    ([0, 0, 0, 0], [64, 64, 64, 64], [64, 64, 64, 64])])
def test_fork_edges(gpu_ctx, parents, keep, old, small):
    rng = np.random.default_rng(3)
    width = 4 if small else 16000  # beyond what one block takes
    n = len(old)
    if not small and n == 1:
        width = 17000
    table, free = np.full((n, width), -1, np.int32), list(rng.permutation(40).astype(np.int32))
    for i in range(n):
        for j in range(pages_of(old[i], 16)):
            table[i, j] = free.pop()
    ring = np.full(40, -7, np.int32)
    ring[(33 + np.arange(len(free))) % 40] = free
    check_fork(gpu_ctx, parents, keep, old, 16, table, ring, [33, 33 + len(free)])


def test_fork_steps_of_a_beam_search(gpu_ctx):
    """Steps of four beams: pages are neither lost nor held twice as theirs, and at the end all are free."""
    rng = np.random.default_rng(12)
    n, width, page, num_pages = 4, 20, 16, 60
    old, table = np.array([100, 0, 0, 0]), np.full((n, width), -1, np.int32)
    order = rng.permutation(num_pages).astype(np.int32)
    table[0, :7] = order[:7]
    ring, cursors = np.roll(order, -7), np.array([0, num_pages - 7], np.int64)
    parents = np.zeros(n, np.int64)
    for step in range(120):
        want = check_fork(gpu_ctx, parents, None, old, page, table, ring, cursors)
        table, ring, (head, tail), old = want[0], want[1], want[2], np.array(want[3])
        for i in range(n):  # the plan of a single token
            if parents[i] >= 0 and old[i] % page == 0:
                table[i, old[i] // page] = ring[head % num_pages]
                head += 1
            old[i] += parents[i] >= 0
        cursors = np.array([head, tail], np.int64)
        held = {int(p) for i in range(n) for p in table[i, : pages_of(old[i], page)]}
        free = {int(ring[k % num_pages]) for k in range(head, tail)}
        assert len(free) == tail - head and held.isdisjoint(free) and len(held) + len(free) == num_pages
        partial = [int(table[i, old[i] // page]) for i in range(n) if old[i] % page]
        assert len(set(partial)) == len(partial)
        parents = rng.integers(0, n, n)
    want = check_fork(gpu_ctx, np.full(n, -1), None, old, page, table, ring, cursors)
    assert want[2][1] - want[2][0] == num_pages


@pytest.mark.parametrize("n,width", [(3, 6), (600, 40)])
@pytest.mark.parametrize("what", ["parent", "parent low", "keep", "keep low", "length", "length low", "largest", "head", "tail",
                                  "full", "backwards", "pages", "all"])
def test_fork_refused_on_the_device(gpu_ctx, what, n, width):
    rng = np.random.default_rng(6)
    old, table, ring, cursors = pool(rng, n, width, 16, 3 * n, 90)
    old[0], table[0, :6] = 90, np.maximum(table[0, :6], 0)
    parents, keep = np.zeros(n, np.int64), np.full(n, 90)
    status = {"head": PLAN_CURSORS, "tail": PLAN_CURSORS, "full": PLAN_CURSORS, "backwards": PLAN_CURSORS,
              "pages": PLAN_PAGES, "all": PLAN_LENGTHS | PLAN_PAGES}.get(what, PLAN_LENGTHS)
    if what in ("parent", "all"):
        parents[n - 1] = n
    if what == "parent low":
        parents[1] = -2
    if what == "keep":
        keep[n // 2] = 91
    if what == "keep low":
        keep[2] = -1
    if what == "length":
        old[n - 1] = 16 * width + 1
    if what == "length low":
        old[1] = -5
    if what == "largest":
        old[0], keep[:] = 2 ** 31 - 1, 2 ** 31 - 1
    if what == "head":
        cursors = np.array([-1, 5])
    if what == "tail":
        cursors = np.array([2 ** 62, -2 ** 62])
    if what == "full":
        cursors = np.array([7, 8 + ring.size])
    if what == "backwards":
        cursors = np.array([9, 8])
    if what == "pages":
        cursors = np.array([9, 9 + n - 2])
    if what == "all":
        cursors = np.array([9, 9])
    for alias in (False, True):
        check_fork(gpu_ctx, parents, keep, old, 16, table, ring, cursors, status=status, alias=alias)


@pytest.mark.parametrize("n,width", [(3, 6), (600, 40)])
def test_fork_with_foreign_page_ids(gpu_ctx, n, width):
    """Page ids that are none of the cache's are passed on and never freed; nothing else changes."""
    rng = np.random.default_rng(8)
    old, table, ring, cursors = pool(rng, n, width, 16, 2 * n, 90)
    old[:3] = 90
    table[0, :6], table[1, :6], table[2, :6] = 2 ** 31 - 1, -2 ** 31, ring.size
    ring[cursors[0] % ring.size] = -9
    parents = np.arange(n)
    parents[0], parents[1], parents[2] = 1, 1, -1
    check_fork(gpu_ctx, parents, None, old, 16, table, ring, cursors)


@pytest.mark.parametrize("n,width", [(3, 12), (5, 400), (3, 9000), (1030, 70)])
def test_fork_frees_a_page_once_that_a_row_names_twice(gpu_ctx, n, width):
    """A table that no plan or fork makes: a row with the same page at several places. It goes to the ring once, in the place of
    the last of them, wherever they lie; and not at all where one of them goes on."""
    rng = np.random.default_rng(width)
    page, long = 16, min(width, 5000)
    old = np.minimum(rng.integers(1, 6 * page, n), width * page)
    old[:3] = long * page - 3
    used = -(-old // page)
    num_pages = int(used.sum()) + 3 * n
    order = rng.permutation(num_pages).astype(np.int32)
    table, at = np.full((n, width), -1, np.int32), 0
    for i in range(n):
        table[i, : used[i]] = order[at: at + used[i]]
        at += used[i]
    free = order[at:]
    ring = np.full(num_pages, -7, np.int32)
    ring[: free.size] = free
    table[0, long - 1] = table[0, 0]                                     # the ends of a row
    table[0, 1: long - 1: 3] = table[0, 2]                               # many times
    table[1, rng.integers(0, long, long // 2)] = table[1, long // 2]     # and in two rows
    table[2, rng.integers(0, long, 4)] = table[1, long // 2]
    cursors = [0, free.size]
    for parents in ([-1, -1, -1], [0, 0, -1], [-1, 2, 1], [1, -1, 2]):
        parents = np.concatenate([parents, np.where(rng.random(n - 3) < 0.5, np.arange(3, n), -1)]).astype(np.int64)
        keep = np.where(parents >= 0, old[np.maximum(parents, 0)], 0)
        want = check_fork(gpu_ctx, parents, keep, old, page, table, ring, cursors)
        entries = want[1][np.arange(want[2][0], want[2][1]) % num_pages]
        assert len(set(entries.tolist())) == entries.size
        check_fork(gpu_ctx, parents, np.minimum(keep, page * (long // 2)), old, page, table, ring, cursors)


def test_fork_of_two_pools_in_turn(gpu_ctx):
    """Calls of one context on pools of different sizes, the second growing what the context keeps for each page."""
    rng = np.random.default_rng(9)
    pools = [pool(rng, 8, 30, 16, 20), pool(rng, 8, 30, 16, 9000), pool(rng, 50, 400, 16, 200)]
    for _ in range(3):
        for old, table, ring, cursors in pools:
            parents, keep = some_parents(rng, len(old), old)
            check_fork(gpu_ctx, parents, keep, old, 16, table, ring, cursors)


def test_fork_refuses(gpu_ctx):
    rng = np.random.default_rng(10)
    old, table, ring, cursors = pool(rng, 4, 6, 16, 9)
    with Arrays(gpu_ctx) as mem:
        ints = [mem.up(np.zeros(64, np.int32)) for _ in range(9)]
        pt = mem.up(np.concatenate([table, table]))
        c = mem.up(cursors)

        def call(new_table=pt + 4 * 24, stride=6, new_lens=ints[3], next_lens=ints[4], ring_p=ints[5], pages=40):
            S.paged_fork(gpu_ctx, 4, ints[0], ints[1], ints[2], 16, pt, new_table, 6, stride, ring_p, pages, c, c, new_lens,
                         next_lens, ints[6], ints[7], ints[8])

        for kw, text in [({"new_table": pt}, "overlap"), ({"new_table": pt + 4 * 23}, "overlap"),
                         ({"new_lens": ints[2]}, "overlap"), ({"next_lens": ints[0] + 12}, "overlap"),
                         ({"next_lens": ints[1]}, "overlap"), ({"stride": 5}, "stride"), ({"stride": 600}, "allocation"),
                         ({"pages": 65}, "allocation"), ({"new_lens": None}, "null"), ({"ring_p": 4096}, "device memory")]:
            with pytest.raises(S.SocError, match=text) as e:
                call(**kw)
            assert e.value.code == SOC_ERR_INVALID
        call()
        gpu_ctx.synchronize()


# ---- copy ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("page", [16, 32, 256])
@pytest.mark.parametrize("layers,nkv,hd,stride", [(1, 1, 64, 0), (2, 8, 128, 0), (3, 2, 128, 40), (70, 1, 64, 0)])
def test_copy(gpu_ctx, page, layers, nkv, hd, stride):
    rng = np.random.default_rng(page + layers)
    num_pages, size = 23, nkv * page * hd
    step = size + stride
    moves = np.array([[0, 1, page], [22, 2, 1], [0, 3, page - 1], [4, 5, 0], [6, 7, -3], [8, 9, page + 1], [10, 10, page],
                      [-1, 11, 4], [23, 12, 4], [13, 23, 4], [13, -2 ** 31, 4], [2 ** 31 - 1, 14, 4], [8, 15, 7],
                      [16, 17, 2 ** 31 - 1], [16, 18, -2 ** 31], [19, 20, page]], np.int32)
    pools = rng.integers(0, 1 << 16, (layers, 2, num_pages * step), dtype=np.uint16)
    for count in (len(moves), len(moves) - 1, 0, -1, 1 << 20, None):
        want = pools.copy()
        shaped = want.reshape(layers, 2, num_pages, step)[..., :size].reshape(layers, 2, num_pages, nkv, page, hd)
        done = len(moves) if count is None else min(max(count, 0), len(moves))
        for a, b, k in moves[:done].tolist():
            k = min(max(k, 0), page)
            if 0 <= a < num_pages and 0 <= b < num_pages:
                shaped[:, :, b, :, :k] = shaped[:, :, a, :, :k]
        view = want.reshape(layers, 2, num_pages, step)
        view[..., :size] = shaped.reshape(layers, 2, num_pages, size)
        with Arrays(gpu_ctx) as mem:
            p = mem.up(pools)
            each = num_pages * step * 2
            caches = S.PagedLayers([S.PagedCache(p + 2 * l * each, p + (2 * l + 1) * each, num_pages, page, nkv, hd,
                                                 step if stride else 0) for l in range(layers)])
            pc = None if count is None else mem.up(np.array([count], np.int32))
            S.paged_copy(gpu_ctx, caches, mem.up(moves), pc, len(moves))
            assert np.array_equal(mem.down(p), want)


# ---- compact ---------------------------------------------------------------------------------------------------------
def compact_rules(lens, page, table, new_table, ring, new_ring, cursors, num_pages, max_moves):
    new_table, new_ring = new_table.copy(), new_ring.copy()
    n, width = table.shape
    head, tail = (int(c) for c in cursors)
    status = 0
    good = [0 <= x and pages_of(x, page) <= width for x in lens]
    if not all(good):
        status |= PLAN_LENGTHS
    sane = head >= 0 and tail >= 0 and 0 <= tail - head <= num_pages
    free = [int(ring[k % num_pages]) for k in range(head, tail)] if sane else []
    if not sane or len({x for x in free if 0 <= x < num_pages}) != tail - head:
        status |= PLAN_CURSORS
    moves, goes = [], {}
    if status == 0:
        holes = sorted(free)
        used = sorted(set(range(num_pages)) - set(free), reverse=True)
        for a, b in list(zip(used, holes))[:max_moves]:
            if a < b:
                break
            moves.append([a, b, page])
            goes[a] = b
        free = sorted(set(free) - set(goes.values()) | set(goes))
    if sane:
        for k, x in enumerate(free):
            new_ring[(head + k) % num_pages] = x
    for i in range(n):
        e = pages_of(lens[i], page) if lens[i] >= 0 else 0
        for j in range(min(e, width)):
            new_table[i, j] = goes.get(int(table[i, j]), int(table[i, j]))
    return new_table, new_ring, moves, status


def check_compact(ctx, lens, page, table, ring, cursors, max_moves, status=0, in_place=False, extra=0):
    n, width = table.shape
    wide = np.full((n, width + extra), 77, np.int32)
    wide[:, :width] = table
    table_out = wide if in_place else np.full((n, width + extra), 66, np.int32)
    ring_out = ring if in_place else np.full(ring.size, 44, np.int32)
    want = compact_rules(lens, page, table, table_out[:, :width], ring, ring_out, cursors, ring.size, max_moves)
    assert want[3] == status
    with Arrays(ctx) as mem:
        pl, pt, pr = mem.up(np.asarray(lens, np.int32)), mem.up(wide), mem.up(ring)
        pt2, pr2 = (pt, pr) if in_place else (mem.up(table_out), mem.up(ring_out))
        outs = [mem.up(guarded(np.full(k, 99, np.int32), 2, 3, 55)) for k in (3 * max_moves, 1, 1)]
        S.paged_compact(ctx, n, pl, page, pt, pt2, width, width + extra, pr, pr2, ring.size,
                        mem.up(np.asarray(cursors, np.int64)), outs[0] + 8, max_moves, outs[1] + 8, outs[2] + 8)
        moves, count, got = (mem.down(p) for p in outs)
        for g in (moves, count, got):
            assert (g[:2] == 55).all() and (g[-3:] == 55).all()
        assert int(got[2]) == status and int(count[2]) == len(want[2])
        k = len(want[2])
        assert moves[2: 2 + 3 * k].reshape(-1, 3).tolist() == want[2] and (moves[2 + 3 * k: -3] == 99).all()
        t = mem.down(pt2)
        assert np.array_equal(t[:, :width], want[0]) and (t[:, width:] == table_out[:, width:]).all()
        assert np.array_equal(mem.down(pr2), want[1])
    return want


@pytest.mark.parametrize("n,width,spare", [(1, 1, 0), (1, 1, 1), (1, 5, 300), (7, 9, 3), (30, 40, 400), (200, 64, 70000), (9, 9, 300000),
                                           (1000, 20, 5)])
def test_compact(gpu_ctx, n, width, spare):
    rng = np.random.default_rng(n + spare)
    old, table, ring, cursors = pool(rng, n, width, 16, spare, start=int(rng.integers(0, 1 << 40)))
    if cursors[0] == cursors[1] and ring.size == 0:
        old, table, ring, cursors = np.array([3]), np.zeros((1, 1), np.int32), np.full(1, -7, np.int32), np.zeros(2, np.int64)
    for in_place in (False, True):
        want = check_compact(gpu_ctx, old, 16, table, ring, cursors, ring.size, in_place=in_place, extra=3)
        check_compact(gpu_ctx, old, 16, table, ring, cursors, max(1, len(want[2]) // 3), in_place=in_place)
        check_compact(gpu_ctx, old, 16, table, ring, cursors, 1, in_place=in_place)
    used = ring.size - int(cursors[1] - cursors[0])
    held = {int(p) for i in range(n) for p in want[0][i, : pages_of(old[i], 16)]}
    assert all(p < used for p in held)


def test_compact_of_the_largest_pool(gpu_ctx):
    """2^20 pages: the bitmap takes 128 KiB of LDS."""
    rng = np.random.default_rng(4)
    old, table, ring, cursors = pool(rng, 40, 500, 16, 0, start=5)
    big = 1 << 20
    spread = rng.permutation(big).astype(np.int32)
    held = ring.size - int(cursors[1] - cursors[0])
    used = np.unique(table[table >= 0])
    name = np.full(ring.size + 1, -1, np.int32)
    name[used] = spread[: used.size]
    table = np.where(table >= 0, name[table], -1).astype(np.int32)
    free = spread[used.size:]
    ring = np.full(big, -7, np.int32)
    ring[(5 + np.arange(free.size)) % big] = free
    assert held <= used.size + 5
    check_compact(gpu_ctx, old, 16, table, ring, [5, 5 + free.size], 1 << 20)
    check_compact(gpu_ctx, old, 16, table, ring, [5, 5 + free.size], 777)


@pytest.mark.parametrize("what", ["length", "length low", "head", "backwards", "full", "foreign", "negative", "twice", "both"])
def test_compact_refused_on_the_device(gpu_ctx, what):
    rng = np.random.default_rng(5)
    old, table, ring, cursors = pool(rng, 9, 12, 16, 30)
    status = PLAN_LENGTHS if what.startswith("length") else PLAN_CURSORS
    if what in ("length", "both"):
        old[3], status = 16 * 12 + 1, status | PLAN_LENGTHS
    if what == "length low":
        old[8] = -1
    if what == "head":
        cursors = np.array([-3, 2])
    if what == "backwards":
        cursors = np.array([8, 7])
    if what == "full":
        cursors = np.array([0, ring.size + 1])
    at = int(cursors[0]) % ring.size
    if what == "foreign":
        ring[at] = ring.size
    if what in ("negative", "both"):
        ring[at] = -1
    if what == "twice":
        ring[at] = ring[at + 1]
    for in_place in (False, True):
        check_compact(gpu_ctx, old, 16, table, ring, cursors, 50, status=status, in_place=in_place)
    # and the next call finds the bitmap clear
    old, table, ring, cursors = pool(rng, 9, 12, 16, 30)
    check_compact(gpu_ctx, old, 16, table, ring, cursors, 50)


def test_compact_then_copy_then_read(gpu_ctx):
    """What rows hold is the same before and after a compaction whose moves are copied."""
    rng = np.random.default_rng(6)
    n, width, page, nkv, hd = 12, 10, 16, 2, 64
    old, table, ring, cursors = pool(rng, n, width, page, 60)
    planes = rng.integers(0, 1 << 16, (2, ring.size, nkv, page, hd), dtype=np.uint16)
    with Arrays(gpu_ctx) as mem:
        p, pt, pr = mem.up(planes), mem.up(table), mem.up(ring)
        moves, count, status = mem.up(np.zeros((100, 3), np.int32)), mem.up(np.zeros(1, np.int32)), mem.up(np.zeros(1, np.int32))
        S.paged_compact(gpu_ctx, n, mem.up(old.astype(np.int32)), page, pt, pt, width, width, pr, pr, ring.size,
                        mem.up(cursors), moves, 100, count, status)
        layers = S.PagedLayers([S.PagedCache(p, p + planes[0].nbytes, ring.size, page, nkv, hd)])
        S.paged_copy(gpu_ctx, layers, moves, count, 100)
        after, t = mem.down(p), mem.down(pt)
        assert int(mem.down(count)[0]) > 0 and int(mem.down(status)[0]) == 0
    used = ring.size - int(cursors[1] - cursors[0])
    for i in range(n):
        e = pages_of(old[i], page)
        assert (t[i, :e] < used).all() and np.array_equal(after[:, t[i, :e]], planes[:, table[i, :e]])
