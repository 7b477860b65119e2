"""Attention of one token of each sequence where groups of sequences share a prefix (soc_paged_attention_shared) against the
formula in 64 bits. That a group's rows share its prefix is the caller's word; the rest of the groups is a hint, so that
malformed ones, and prefixes longer than rows, change nothing but the time. (Prefixes of less than 256 keys are each row's own
keys, whatever the groups.)

Tolerance. A score is a sum of 2 head_dim products (queries as two fp16 parts, exact to 2^-22), added in 32 bits in any order:
off by (2 head_dim + 8) 2^-24 sum |q_i k_i| scale = e. A weight is then off by 2 e + 8 2^-24 relative, the weighted sum by
that, by its weights' 2^-22 and by its chain of additions: two a key of a wave, which has a quarter of a block's keys (2048 at
most, or an eighth of the sequence's if that is more) and a tile, and 264 parts and waves. So |out - want| <= (2 e + (c + 8)
2^-24 + 2^-21) max |v| with c that chain; lse: e + (c + 8) 2^-24 + 2^-23 |lse|. fp16 results add half a step, 2^-11."""
import math

import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import SOC_ERR_INVALID
from tests.device import NP, Arrays, guarded

pytestmark = pytest.mark.gpu
INF = np.inf


@pytest.fixture(autouse=True)
def shared(monkeypatch):
    """Small batches would be read row by row."""
    monkeypatch.setenv("SOC_PAGED_SHARED", "always")


def formula(q, k, v, scale):
    """q [nq][hd], k / v [nkv][len][hd] -> (out, lse, tolerances) in 64 bits."""
    nq, hd = q.shape
    nkv, length = k.shape[:2]
    if length == 0:
        return np.zeros((nq, hd)), np.full(nq, -INF), np.zeros((nq, hd)), np.zeros(nq)
    k, v, q = k.astype(np.float64), v.astype(np.float64), q.astype(np.float64).reshape(nkv, nq // nkv, hd)
    s = q @ k.transpose(0, 2, 1) * scale
    e = (2 * hd + 8) * 2.0 ** -24 * (np.abs(q) @ np.abs(k).transpose(0, 2, 1)).max(-1, keepdims=True) * abs(scale)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    total = p.sum(-1, keepdims=True)
    out, lse = p @ v / total, m + np.log(total)
    c = 2 * (max(2048, length // 8 + 128) // 4 + 32) + 264
    tol = (2 * e + (c + 8) * 2.0 ** -24 + 2.0 ** -21) * np.abs(v).max((1, 2))[:, None, None]
    tol_lse = e + (c + 8) * 2.0 ** -24 + 2.0 ** -23 * np.abs(lse)
    return (out.reshape(nq, hd), lse.reshape(nq), np.broadcast_to(tol, out.shape).reshape(nq, hd), tol_lse.reshape(nq))


class Batch:
    """Rows of groups that share `prefix` positions and go on with `tails` of their own (negative: a row that ends that far
    before the prefix does; None: an empty row). Shared full pages are named by all, the page that the prefix ends in is each
    row's own copy."""

    def __init__(self, sizes, prefix, tails, nq, nkv, hd, page, seed=1, garbage=np.nan, kv=None, share=True):
        rng = np.random.default_rng(seed)
        self.sizes, self.prefix, self.nq, self.nkv, self.hd, self.page = sizes, prefix, nq, nkv, hd, page
        n = self.n = sum(sizes)
        group = np.repeat(np.arange(len(sizes)), sizes)
        lens = [0 if t is None else max(0, prefix[g] + t) for g, t in zip(group, tails)]
        self.lens = np.array(lens, np.int64)
        held = -(-self.lens // page)
        self.width = max(1, int(held.max()))
        common = [prefix[g] // page if share else 0 for g in group]
        total = sum(prefix[g] // page for g in range(len(sizes))) * share + int(np.maximum(0, held - common).sum())
        self.pages = total + 2
        free = list(rng.permutation(self.pages).astype(np.int32))
        self.table = np.full((n, self.width), 2 ** 31 - 1, np.int32)
        self.pool = np.full((2, self.pages, nkv, page, hd), garbage, np.float16)
        self.rows = []
        row = 0
        for g, size in enumerate(sizes):
            first = rng.standard_normal((2, nkv, prefix[g], hd)).astype(np.float16)
            mine = [free.pop() for _ in range(prefix[g] // page)] if share else []
            for i in range(size):
                L = int(self.lens[row])
                own = rng.standard_normal((2, nkv, L, hd)).astype(np.float16)
                own[:, :, : prefix[g]] = first[:, :, : L]
                if kv is not None:
                    own = kv(row, own)
                self.rows.append(own)
                for j in range(int(held[row])):
                    p = mine[j] if j < len(mine) else free.pop()
                    self.table[row, j] = p
                    m = min(page, L - j * page)
                    self.pool[:, p, :, :m] = own[:, :, j * page: j * page + m]
                row += 1
        self.starts = np.concatenate([[0], np.cumsum(sizes)])
        self.q = rng.standard_normal((n, nq * hd)).astype(np.float32)

    def run(self, ctx, dtype="f32", *, starts=None, prefix=None, max_group=None, max_prefix=None, scale=0.0, q_pad=0, o_pad=0,
            extra=0, shift=0, in_place=False, lse=True, lens=None, table=None, q=None, page_stride=0):
        n, qw, dt = self.n, self.nq * self.hd, NP[dtype]
        starts = self.starts if starts is None else starts
        prefix = self.prefix if prefix is None else prefix
        groups = len(starts) - 1
        q = (self.q if q is None else q).astype(dt)
        wide = np.full((n, qw + q_pad), 3, dt)
        wide[:, :qw] = q
        flat = np.concatenate([np.full(shift, 3, dt), wide.reshape(-1)])
        t = np.full((n, self.width + extra), 2 ** 31 - 1, np.int32)
        t[:, : self.width] = self.table if table is None else table
        size = self.nkv * self.page * self.hd
        pool = self.pool.reshape(2, self.pages, size)
        if page_stride:
            spread = np.full((2, self.pages, page_stride), np.nan, np.float16)
            spread[:, :, :size] = pool
            pool = spread
        with Arrays(ctx) as mem:
            pq, pk, pv = mem.up(flat), mem.up(pool[0]), mem.up(pool[1])
            out = pq + shift * flat.itemsize if in_place else None
            po = None if in_place else mem.up(guarded(np.full((n, qw + o_pad), 9, dt), 8, 8, 7))
            pl = mem.up(guarded(np.full((n, self.nq), 9, np.float32), 2, 3, 7)) if lse else None
            cache = S.PagedCache(pk, pv, self.pages, self.page, self.nkv, self.hd, page_stride)
            S.paged_attention_shared(
                ctx, cache, pq + shift * flat.itemsize, qw + q_pad, dtype, mem.up(t), self.width + extra, self.width,
                mem.up(np.asarray(self.lens if lens is None else lens, np.int32)), n, mem.up(np.asarray(starts, np.int32)),
                mem.up(np.asarray(prefix, np.int32)), groups,
                min(n, max(1, int(max(self.sizes)))) if max_group is None else max_group,
                min(int(max(self.prefix)), self.width * self.page) if max_prefix is None else max_prefix, self.nq, scale,
                out if in_place else po + 8 * flat.itemsize, qw + (q_pad if in_place else o_pad), pl + 8 if lse else None)
            if in_place:
                got = mem.down(pq)[shift:].reshape(n, -1)
                assert (got[:, qw:] == 3).all()
            else:
                g = mem.down(po)
                assert (g[:8] == 7).all() and (g[-8:] == 7).all()
                got = g[8:-8].reshape(n, -1)
                assert (got[:, qw:] == 9).all()
            got_lse = None
            if lse:
                g = mem.down(pl)
                assert (g[:2] == 7).all() and (g[-3:] == 7).all()
                got_lse = g[2:-3].reshape(n, self.nq)
            return got[:, :qw].reshape(n, self.nq, self.hd), got_lse, q.reshape(n, self.nq, self.hd)

    def check(self, ctx, dtype="f32", skip=(), **kw):
        out, lse, q = self.run(ctx, dtype, **kw)
        scale = kw.get("scale") or 1 / math.sqrt(self.hd)
        for b in range(self.n):
            if b in skip:
                continue
            w, wl, tol, tol_lse = formula(q[b], *self.rows[b], scale)
            if dtype == "f16":
                tol = tol + np.abs(w) * 2.0 ** -11 + 2.0 ** -25
            bad = ~(np.abs(out[b] - w) <= tol)
            assert not bad.any(), (b, float(np.abs(out[b] - w).max()), float(tol.min()))
            if lse is not None:
                with np.errstate(invalid="ignore"):
                    same = (lse[b] == wl) | (np.abs(lse[b] - wl) <= tol_lse)
                assert same.all(), (b, lse[b], wl)
        return out, lse


def ragged(rng, sizes, longest):
    return [int(t) for t in rng.integers(0, longest + 1, sum(sizes))]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,page", [(128, 16), (64, 32), (128, 64), (64, 256), (128, 128)])
@pytest.mark.parametrize("sizes,prefix", [([4], [1000]), ([2, 3, 1], [128, 400, 300]), ([1, 1], [200, 150]), ([8], [127]),
                                          ([9, 2], [1025, 31]), ([3, 5], [0, 2311]), ([8, 3], [255, 256]), ([3, 7], [288, 257])])
def test_groups(gpu_ctx, dtype, hd, page, sizes, prefix):
    rng = np.random.default_rng(page + hd)
    b = Batch(sizes, prefix, ragged(rng, sizes, 150), 8, 2, hd, page)
    b.check(gpu_ctx, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (8, 8), (3, 1), (16, 8), (12, 2), (7, 1), (32, 8), (14, 2), (15, 1), (16, 1), (48, 4)])
@pytest.mark.parametrize("size", [2, 5, 16, 33])
def test_head_groups(gpu_ctx, dtype, nq, nkv, size):
    rng = np.random.default_rng(nq + size)
    Batch([size, 3], [300, 170], ragged(rng, [size, 3], 60), nq, nkv, 128, 16).check(gpu_ctx, dtype)
    Batch([size], [260], ragged(rng, [size], 5), nq, nkv, 64, 32).check(gpu_ctx, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("size,prefix,tail,nq,nkv", [(130, 600, 40, 8, 2), (300, 150, 10, 4, 4), (64, 4000, 3, 16, 8),
                                                     (257, 300, 0, 4, 1), (20, 9000, 700, 4, 2), (2, 20000, 100, 2, 1)])
def test_large_groups(gpu_ctx, dtype, size, prefix, tail, nq, nkv):
    rng = np.random.default_rng(size)
    Batch([size], [prefix], ragged(rng, [size], tail), nq, nkv, 128, 16).check(gpu_ctx, dtype)
    if size < 100:
        Batch([size], [prefix], ragged(rng, [size], tail), nq, nkv, 64, 64).check(gpu_ctx, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_many_groups(gpu_ctx, dtype):
    rng = np.random.default_rng(3)
    sizes = [int(s) for s in rng.integers(1, 6, 300)]
    prefix = [int(p) for p in rng.integers(0, 400, 300)]
    Batch(sizes, prefix, ragged(rng, sizes, 40), 4, 2, 64, 16).check(gpu_ctx, dtype)


@pytest.mark.parametrize("hd", [64, 128])
def test_rows_that_do_not_hold_the_prefix(gpu_ctx, hd):
    """Empty rows, first or last of their group, rows shorter than the prefix, rows that end with it."""
    b = Batch([4, 3, 2, 3], [500, 200, 300, 260], [None, 3, -100, 0, 10, None, 0, None, None, -259, -1, 40], 8, 2, hd, 16)
    out, lse = b.check(gpu_ctx)
    assert (out[0] == 0).all() and (lse[0] == -INF).all() and (out[8] == 0).all()
    b.check(gpu_ctx, "f16")


@pytest.mark.parametrize("page", [16, 64])
def test_wrong_hints_change_no_result(gpu_ctx, page):
    sizes, prefix = [5, 1, 6], [400, 130, 333]
    b = Batch(sizes, prefix, [3, 0, 10, 70, 31, 5, 1, 2, 3, 4, 5, 0], 8, 2, 128, page)
    for kw in [{"starts": [0, 7, 3, 12]}, {"starts": [0, 5, 6, 13]}, {"starts": [-1, 5, 6, 12]}, {"starts": [12, 6, 5, 0]},
               {"starts": [0, 2 ** 31 - 1, -2 ** 31, 12]}, {"starts": [0, 5, 6, 6]}, {"starts": [1, 4, 6, 9], "prefix": [400, 0, 333]},
               {"starts": [0, 0, 0, 5, 5, 6, 12, 12], "prefix": [9, 999, 400, 5, 130, 333, -4]},
               {"starts": [0, 5], "prefix": [400]}, {"starts": [6, 12], "prefix": [333]},
               {"prefix": [-1, -2 ** 31, 0]}, {"prefix": [400, 130, 100]}, {"prefix": [399, 129, 128]},
               {"max_prefix": 0}, {"max_prefix": 128}, {"max_prefix": 177}, {"max_prefix": 336},
               {"max_group": 1}, {"max_group": 2}, {"max_group": 4}, {"max_group": 12}, {"max_group": 5, "max_prefix": 200},
               {"max_group": 2 ** 31 - 1, "max_prefix": 2 ** 31 - 1}]:
        b.check(gpu_ctx, **kw)
    # prefixes as long as a number can be, cut to max_prefix; rows that end before it read their own keys; the last row in no group
    b.check(gpu_ctx, prefix=[2 ** 31 - 1, 130, 2 ** 31 - 1], max_prefix=333, starts=[0, 0, 5, 11])


@pytest.mark.parametrize("q_pad,o_pad,extra,shift", [(8, 0, 0, 0), (0, 3, 2, 0), (3, 0, 0, 1), (1, 1, 7, 2), (4, 4, 0, 4)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strides(gpu_ctx, q_pad, o_pad, extra, shift, dtype):
    b = Batch([5, 2], [300, 160], [4, 0, 20, 33, 1, 0, 90], 8, 2, 128, 32)
    kw = dict(q_pad=q_pad, extra=extra, shift=shift)
    one = b.check(gpu_ctx, dtype, o_pad=o_pad, **kw)
    two = b.check(gpu_ctx, dtype, in_place=True, **kw)
    three = b.check(gpu_ctx, dtype, lse=False, page_stride=2 * 32 * 128 + 8, **kw)
    assert np.array_equal(one[0], two[0]) and np.array_equal(one[1], two[1]) and np.array_equal(one[0], three[0])


@pytest.mark.parametrize("scale", [1.0, 0.02, -0.3, 3.0])
def test_scales(gpu_ctx, scale):
    Batch([6], [700], [4, 0, 20, 33, 1, 100], 8, 2, 64, 16).check(gpu_ctx, scale=scale)


@pytest.mark.parametrize("q_scale", [1e-38, 1e-30, 1e-6, 100.0, 1e5])
def test_query_magnitudes(gpu_ctx, q_scale):
    b = Batch([6], [700], [4, 0, 20, 33, 1, 100], 8, 2, 64, 16)
    b.check(gpu_ctx, q=b.q * np.float32(q_scale), scale=0.125 / q_scale if q_scale > 1e-38 else 0.0)


def test_rising_and_falling_scores(gpu_ctx):
    """The running maximum moves at every tile, or never after the first."""
    for sign in (1, -1):
        def kv(row, own):
            own = own.copy()
            length = own.shape[2]
            own[0] = np.float16(0.01) * own[0]
            own[0, :, :, 0] = sign * np.linspace(-60, 60, max(1, length))[None, :length]
            return own
        b = Batch([4], [900], [0, 0, 0, 0], 4, 2, 64, 16, kv=kv)
        b.q[:] = 0.01 * b.q
        b.q[:, ::64] = 1.0
        b.check(gpu_ctx)


@pytest.mark.parametrize("garbage", [INF, -INF, 65504.0])
def test_what_lies_behind_the_length_is_not_used(gpu_ctx, garbage):
    Batch([3, 2], [333, 150], [0, 1, 5, 0, 14], 8, 2, 128, 64, garbage=garbage).check(gpu_ctx)


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1])
def test_foreign_pages_and_lengths(gpu_ctx, bad):
    b = Batch([4, 3], [320, 200], [40, 40, 40, -300, 0, 9, 40], 8, 2, 64, 16)
    # in a row's own keys: that row; in the prefix: the rows that read it (here the first names it)
    table = b.table.copy()
    table[1, 21] = bad
    out, lse = b.check(gpu_ctx, table=table, skip=(1,))
    assert np.isnan(out[1]).all() and np.isnan(lse[1]).all()
    table = b.table.copy()
    table[:4, 3] = bad
    out, lse = b.check(gpu_ctx, table=table, skip=(0, 1, 2))
    assert np.isnan(out[:3]).all() and np.isnan(lse[:3]).all()
    lens = b.lens.copy()
    lens[0], lens[4] = 2 ** 31 - 1, -2 ** 31
    out, lse = b.check(gpu_ctx, lens=lens, skip=(0, 4))
    assert np.isnan(out[0]).all() and np.isnan(lse[0]).all() and (out[4] == 0).all() and (lse[4] == -INF).all()


def test_non_finite_queries_stay_in_their_row(gpu_ctx):
    b = Batch([5], [300], [4, 0, 20, 33, 1], 8, 2, 64, 16)
    q = b.q.copy()
    q[1, 5], q[3, 70] = np.nan, np.inf
    out, _ = b.check(gpu_ctx, q=q, skip=(1, 3))
    assert np.isnan(out[1, 0]).all() and np.isnan(out[3, 1]).all()


def test_bits_follow_from_the_row(gpu_ctx):
    """Not from the other rows' contents and lengths, nor from what else is queued."""
    b = Batch([6, 2], [700, 200], [4, 0, 20, 33, 1, 100, 3, 50], 8, 2, 128, 16)
    one = b.run(gpu_ctx)
    q, lens = b.q.copy(), b.lens.copy()
    q[1:] = 7.0
    lens[1], lens[2] = 0, 705
    two = b.run(gpu_ctx, q=q, lens=lens)
    assert np.array_equal(one[0][0], two[0][0]) and np.array_equal(one[1][0], two[1][0])
    for _ in range(3):
        assert np.array_equal(one[0], b.run(gpu_ctx)[0])


def test_agrees_with_the_unshared_one(gpu_ctx):
    b = Batch([7, 3], [900, 333], [4, 0, 20, 33, 1, 100, 3, 50, 0, None], 16, 4, 128, 32)
    out, lse, q = b.run(gpu_ctx)
    with Arrays(gpu_ctx) as mem:
        pk, pv, po = mem.up(b.pool[0]), mem.up(b.pool[1]), mem.up(np.zeros((b.n, 16 * 128), np.float32))
        S.paged_attention_decode(gpu_ctx, S.PagedCache(pk, pv, b.pages, 32, 4, 128), mem.up(b.q), 16 * 128, "f32", mem.up(b.table),
                                 b.width, b.width, mem.up(b.lens.astype(np.int32)), b.n, 16, 0.0, po, 16 * 128)
        other = mem.down(po).reshape(out.shape)
    for i in range(b.n):
        _, _, tol, _ = formula(q[i], *b.rows[i], 1 / math.sqrt(128))
        assert (np.abs(out[i] - other[i]) <= 2 * tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_little_to_read(gpu_ctx, dtype, monkeypatch):
    """A small batch is answered as soc_paged_attention_decode answers it; a prefix as long as the rows, and one row."""
    monkeypatch.delenv("SOC_PAGED_SHARED")
    b = Batch([7, 3], [900, 333], [4, 0, 20, 33, 1, 100, 3, 50, 0, None], 16, 4, 128, 32)
    out, _ = b.check(gpu_ctx, dtype)
    with Arrays(gpu_ctx) as mem:
        q = b.q.astype(NP[dtype])
        pk, pv, po = mem.up(b.pool[0]), mem.up(b.pool[1]), mem.up(np.zeros_like(q))
        S.paged_attention_decode(gpu_ctx, S.PagedCache(pk, pv, b.pages, 32, 4, 128), mem.up(q), 16 * 128, dtype, mem.up(b.table),
                                 b.width, b.width, mem.up(b.lens.astype(np.int32)), b.n, 16, 0.0, po, 16 * 128)
        assert np.array_equal(mem.down(po).reshape(out.shape), out)
    Batch([1], [300], [5], 4, 2, 64, 16).check(gpu_ctx, dtype)


def test_more_than_little_to_read(gpu_ctx, monkeypatch):
    """The same rule from the other side."""
    monkeypatch.delenv("SOC_PAGED_SHARED")
    b = Batch([20, 4], [1100, 500], [7] * 24, 16, 8, 128, 64)
    b.check(gpu_ctx)


def test_refusals(gpu_ctx):
    b = Batch([2], [130], [3, 4], 4, 2, 64, 16)
    with Arrays(gpu_ctx) as mem:
        pk, pv = mem.up(b.pool[0]), mem.up(b.pool[1])
        q, out, lse = mem.up(b.q), mem.up(b.q), mem.up(np.zeros(8, np.float32))
        t, lens, starts, prefix = (mem.up(x.astype(np.int32)) for x in (b.table, b.lens, np.array([0, 2]), np.array([130])))

        def call(cache=S.PagedCache(pk, pv, b.pages, 16, 2, 64), q=q, stride=256, out=out, out_stride=256, t=t, lens=lens,
                 starts=starts, prefix=prefix, lse=lse, pages=b.width, groups=1):
            S.paged_attention_shared(gpu_ctx, cache, q, stride, "f32", t, b.width, pages, lens, 2, starts, prefix, groups, 2,
                                     130, 4, 0.0, out, out_stride, lse)

        for kw, text in [({"cache": S.PagedCache(pk, pv, b.pages + 1, 16, 2, 64)}, "allocation"), ({"q": None}, "null"),
                         ({"stride": 255}, "stride"), ({"stride": 300}, "allocation"), ({"out_stride": 257}, "allocation"),
                         ({"t": 4096}, "device memory"), ({"lens": None}, "null"), ({"starts": starts + 4}, "allocation"),
                         ({"prefix": None}, "null"), ({"lse": lse + 4}, "allocation"), ({"out": q, "out_stride": 300}, "in place"),
                         ({"pages": b.width + 1}, "stride"), ({"groups": 2}, "allocation")]:
            with pytest.raises(S.SocError, match=text) as e:
                call(**kw)
            assert e.value.code == SOC_ERR_INVALID, kw
        call()
        gpu_ctx.synchronize()


def test_refuses_bounds_beyond_a_launch(gpu_ctx):
    n, nkv, nq, hd, page = 4096, 2, 32, 64, 16
    with Arrays(gpu_ctx) as mem:
        pool = np.zeros((20, nkv, page, hd), np.float16)
        cache = S.PagedCache(mem.up(pool), mem.up(pool), 20, page, nkv, hd)
        q, out = (mem.up(np.zeros((n, nq * hd), np.float32)) for _ in range(2))
        t, lens, prefix = mem.up(np.zeros((n, 256), np.int32)), mem.up(np.zeros(n, np.int32)), mem.up(np.zeros(n, np.int32))
        starts = mem.up(np.arange(n + 1, dtype=np.int32))

        def call(max_group):
            S.paged_attention_shared(gpu_ctx, cache, q, nq * hd, "f32", t, 256, 256, lens, n, starts, prefix, n, max_group, 4096,
                                     nq, 0.0, out, nq * hd)

        with pytest.raises(S.SocError, match="too many groups") as e:
            call(n)
        assert e.value.code == SOC_ERR_INVALID
        call(2)
        assert not mem.down(out).any()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bits", [10, 24, 28, 33, 40, 64, 100, -28, -64])
def test_scores_that_fp32_holds_but_not_to_a_unit(gpu_ctx, bits, hd, dtype):
    """Whole products, times +- 2^|bits|: what a score is off by in 32 bits passes the range of an exponential, but the largest
    scores are equal ones, and the others' weights are 0 from 2^10 on (e^-1024). So the result is the mean of the values at the
    largest product, off by their weights' 2^-22 and the chains of additions; lse is that score but for eight roundings (log2(e),
    ln 2 and the scale's product with it, the score, the reference, its logarithm's sum, the product with ln 2), 2^-21, and the
    logarithm of their count."""
    b = Batch([5, 2], [300, 290], [4, 0, 20, 33, 1, 100, 3], 16, 2, hd, 16,
              kv=lambda row, own: np.stack([np.clip(np.rint(own[0]), -3, 3), own[1]]))
    b.q[:] = np.clip(np.rint(b.q), -3, 3)
    scale = math.copysign(2.0 ** abs(bits), bits)
    out, lse, q = b.run(gpu_ctx, dtype, scale=scale)
    for r in range(b.n):
        k, v = b.rows[r].astype(np.float64)
        s = q[r].astype(np.float64).reshape(2, 8, hd) @ k.transpose(0, 2, 1) * scale
        top = s.max(-1, keepdims=True)
        w = (s == top) / (s == top).sum(-1, keepdims=True)
        want = (w @ v).reshape(16, hd)
        c = 2 * (2048 // 4 + 32) + 264
        tol = ((c + 8) * 2.0 ** -24 + 2.0 ** -21) * np.abs(v).max()
        if dtype == "f16":
            tol = tol + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
        assert (np.abs(out[r] - want) <= tol).all(), (r, float(np.abs(out[r] - want).max()))
        want_lse = (top[..., 0] + np.log((s == top).sum(-1))).reshape(16)
        assert (np.abs(lse[r] - want_lse) <= 2.0 ** -21 * np.abs(want_lse) + (c + 8) * 2.0 ** -24).all(), (r, lse[r], want_lse)


def unit_scale():
    """A scale whose fp32 product with log2(e) is 1: scores in base 2 are the products themselves."""
    log2e, s = np.float32(1.4426950408889634), np.float32(math.log(2))
    for c in [s, *(np.nextafter(s, np.float32(d), dtype=np.float32) for d in (0, 1))]:
        if np.float32(c * log2e) == 1:
            return float(c)
    raise AssertionError("no such scale")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,nkv,prefix,second", [(3, 1, 256, 32), (2, 256, 1024, 128)])
def test_a_row_s_bits_at_the_edge_of_a_rescale(gpu_ctx, rows, nkv, prefix, second, dtype):
    """Row 0's second score lies half a unit in the last place of 14 above its reference and 14: no weight passes 2^14, but the
    score less 14, rounded, passes the reference. Whether row 1, whose columns the same wave holds, is rescaled at that tile must not
    show in row 0. Blocks of 64 columns (24 of them, a wave's next tile 32 keys on) and of 16 (128 keys on)."""
    hd, G = 64, 8

    def kv(row, own):
        own = own.copy()
        own[0] = 0
        own[0, :, 0, :2] = 0.5, 2.0 ** -10            # row 0: 0.5 + 2^-20, reference 2^-20 - 9.5
        own[0, :, second, :3] = 4.5, 3 * 2.0 ** -11, 100  # row 0: 4.5 + 3 2^-21 = reference + 14 + 2^-21
        return own

    b = Batch([rows], [prefix], [0] * rows, G * nkv, nkv, hd, 16, kv=kv)
    q = np.zeros((rows, nkv * G, hd), np.float32)
    q[0, :, :2] = 1, 2.0 ** -10
    one = b.run(gpu_ctx, dtype, q=q.reshape(rows, -1), scale=unit_scale())
    q[1:, :, 2] = 1
    two = b.run(gpu_ctx, dtype, q=q.reshape(rows, -1), scale=unit_scale())
    assert np.array_equal(one[0][0], two[0][0]) and np.array_equal(one[1][0], two[1][0])


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("nq", [8, 24])
def test_wrong_hints_about_prefixes_that_are_read_once(gpu_ctx, page, nq):
    """Prefixes of 256 keys and more, which are read once (shorter ones are each row's own keys): starts out of order or out of
    range, prefixes that are cut, negative or longer than the rows, bounds that are too low."""
    sizes, prefix = [5, 1, 6], [400, 290, 333]
    b = Batch(sizes, prefix, [3, 0, 10, 70, 31, 5, 1, 2, 3, 4, 5, 0], nq, 2, 128, page)
    for kw in [{"starts": [0, 7, 3, 12]}, {"starts": [0, 5, 6, 13]}, {"starts": [1, 4, 6, 9], "prefix": [400, 0, 333]},
               {"starts": [0, 0, 0, 5, 5, 6, 12, 12], "prefix": [9, 999, 400, 5, 290, 333, -4]}, {"starts": [6, 12], "prefix": [333]},
               {"starts": [2, 5], "prefix": [300]}, {"prefix": [-1, -2 ** 31, 333]}, {"prefix": [399, 289, 256]},
               {"prefix": [2 ** 31 - 1, 290, 333], "max_prefix": 400}, {"max_prefix": 255}, {"max_prefix": 256}, {"max_prefix": 287},
               {"max_prefix": 300}, {"max_group": 2}, {"max_group": 5}, {"max_group": 4, "max_prefix": 320}]:
        b.check(gpu_ctx, **kw)


@pytest.mark.parametrize("nq", [8, 24])
def test_a_prefix_longer_than_what_the_rows_share(gpu_ctx, nq):
    """The caller's word, broken for the second group's rows, which share 290 positions and are said to share 384: one of them that
    holds them all lends its pages to the others. The other groups' rows are as they were, and so are rows too short for it."""
    b = Batch([3, 4, 2], [400, 290, 300], [3, 0, 10, 200, 150, 93, 120, 5, 6], nq, 2, 64, 16)
    out, lse, q = b.run(gpu_ctx, prefix=[400, 384, 300], max_prefix=400)
    for r in range(b.n):
        k, v = b.rows[r]
        if r in (4, 6):  # the first 384 positions are those of row 3, the first that holds them
            k, v = (np.concatenate([lent[:, :384], own[:, 384:]], 1) for lent, own in zip(b.rows[3], b.rows[r]))
        want, want_lse, tol, tol_lse = formula(q[r], k, v, 0.125)
        assert (np.abs(out[r] - want) <= tol).all() and (np.abs(lse[r] - want_lse) <= tol_lse).all(), r
