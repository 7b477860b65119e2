"""Log probabilities, ranks, entropy and top alternatives (soc_logprobs) against the formulas in 64 bits: vocabularies
from one token to more than Qwen3's, odd sizes, ties, masked rows, NaN and infinities, fp32 and fp16, strides.

Tolerances. A log probability is (x - M) / T - log S: the difference and its product with 1/T (itself rounded) are three
roundings of |x - M| / T, log S is off by S's relative error plus its own two steps. S is a sum of positive terms, each
off by |d| 2^-23 (its scaled argument) + 2 steps where it counts (|d| < 20), added in chains of at most 700 terms:
(700 + 44) 2^-24 = 4.5e-5 relative, in the worst case. The entropy log S - D / S has the same relative error in D, whose
terms are all negative: 4.5e-5 (|D / S| + 1) + the error of log S."""
import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import SOC_ERR_INVALID
from tests.device import NP, Arrays

pytestmark = pytest.mark.gpu

EPS_SUM = 4.5e-5


def order(row, k):
    """The first k token ids: NaNs, then by value, ties by id."""
    v = np.where(np.isnan(row), np.inf, row.astype(np.float64)) + 0.0
    return np.lexsort((np.arange(row.size), -v, ~np.isnan(row)))[:k]


def reference(row, t):
    """(log probabilities, entropy) in 64 bits; None where the row holds a NaN or +inf."""
    x = row.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any():
        return None, np.nan
    m = x.max()
    if m == -np.inf:
        return np.full(x.size, -np.inf), 0.0
    d = (x - m) / t
    e = np.exp(d)
    s = e.sum()
    return d - np.log(s), np.log(s) - np.where(e > 0, d, 0.0) @ e / s


def run(ctx, x, dtype="f32", t=1.0, tokens=None, top=0, pad=0, shift=0, entropy=True):
    rows, vocab = x.shape
    flat = np.full(shift + rows * (vocab + pad), np.nan, NP[dtype])
    flat[shift:].reshape(rows, vocab + pad)[:, :vocab] = x
    x = x.astype(NP[dtype])
    with Arrays(ctx) as mem:
        px = mem.up(flat)
        pt = mem.up(tokens) if tokens is not None else None
        lp, en = mem.up(np.full(rows, 9.0, np.float32)), mem.up(np.full(rows, 9.0, np.float32))
        rk = mem.up(np.full(rows, 9, np.int32))
        ids, tl = mem.up(np.full((rows, top), 9, np.int32)), mem.up(np.full((rows, top), 9.0, np.float32))
        S.logprobs(ctx, px + shift * flat.itemsize, dtype, vocab + pad, rows, vocab, t, pt,
                   lp if pt else None, rk if pt else None, en if entropy else None, top, ids if top else None,
                   tl if top else None)
        return x, mem.down(lp), mem.down(rk), mem.down(en), mem.down(ids), mem.down(tl)


def verify(x, t, tokens, top, lp, rk, en, ids, tl):
    t = 1.0 if t <= 0 else t
    for r, row in enumerate(x):
        want, h = reference(row, t)
        first = order(row, row.size)
        if top:
            assert np.array_equal(ids[r], first[:top]), (r, ids[r], first[:top])
        if want is None:
            assert np.isnan(en[r]) and np.isnan(tl[r]).all()
        else:
            assert abs(en[r] - h) <= EPS_SUM * (abs(h) + 3) + 1e-6, (r, en[r], h)

            def close(got, at):
                with np.errstate(over="ignore"):
                    w = want[at].astype(np.float32).astype(np.float64)  # -inf beyond 32 bits' range
                same = (got == -np.inf) & (w == -np.inf)
                off = np.abs(np.where(same, 0, got) - np.where(same, 0, w))
                scale = np.where(same, 0, np.abs(np.where(same, 0, w)))
                return (off <= EPS_SUM + 4 * 2.0 ** -24 * (scale + 12 / t)).all()

            if top:
                assert close(tl[r], ids[r]), (r, tl[r], want[ids[r]])
        if tokens is None:
            continue
        k = int(tokens[r])
        if 0 <= k < row.size:
            assert rk[r] == int(np.flatnonzero(first == k)[0])
            if want is None:
                assert np.isnan(lp[r])
            else:
                assert close(lp[r:r + 1], np.array([k])), (r, lp[r], want[k])
        else:
            assert rk[r] == -1 and (lp[r] == 0.0 if k == -1 else np.isnan(lp[r]))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 257, 1000, 1023, 4097, 16384, 50001])
def test_vocabularies(gpu_ctx, vocab, dtype):
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((5, vocab)) * 3
    tokens = rng.integers(0, vocab, 5).astype(np.int32)
    for top in sorted({0, 1, min(5, vocab), min(64, vocab)}):
        got = run(gpu_ctx, x, dtype, 1.0, tokens, top)
        verify(got[0], 1.0, tokens, top, *got[1:])


@pytest.mark.parametrize("rows", [1, 2, 17, 300])
@pytest.mark.parametrize("top", [0, 1, 20, 33, 64])
def test_rows_of_the_full_vocabulary(gpu_ctx, rows, top):
    rng = np.random.default_rng(rows * 100 + top)
    x = rng.standard_normal((rows, 151936), dtype=np.float32) * 2.5
    tokens = rng.integers(0, 151936, rows).astype(np.int32)
    got = run(gpu_ctx, x, "f32", 0.7, tokens, top)
    keep = slice(0, min(rows, 12))  # every row's reference takes a while
    verify(got[0][keep], 0.7, tokens[keep], top, *(g[keep] for g in got[1:]))


@pytest.mark.parametrize("vocab", [8192, 8193, 16384, 16385, 2 ** 18, 2 ** 18 + 1, 2 ** 20 - 1, 2 ** 20])
@pytest.mark.parametrize("pad", [0, 1])
def test_vocabularies_at_the_chunks_borders(gpu_ctx, vocab, pad):
    rng = np.random.default_rng(vocab)
    x = rng.integers(-40, 41, (3, vocab)).astype(np.float32) / 4
    tokens = np.array([0, vocab - 1, vocab // 2], np.int32)
    for dtype in ("f32", "f16"):
        got = run(gpu_ctx, x, dtype, 1.0, tokens, 64, pad)
        verify(got[0], 1.0, tokens, 64, *got[1:])


@pytest.mark.parametrize("t", [0.0, -2.0, 0.05, 0.6, 5.0, 1000.0])
def test_temperatures(gpu_ctx, t):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 3001)) * 2
    tokens = rng.integers(0, 3001, 4).astype(np.int32)
    got = run(gpu_ctx, x, "f32", t, tokens, 7)
    verify(got[0], t, tokens, 7, *got[1:])


def test_ties_go_to_the_lowest_id(gpu_ctx):
    rng = np.random.default_rng(6)
    rows = [np.zeros(70000), rng.integers(-3, 4, 70000), np.where(rng.random(70000) < 0.5, 0.0, -0.0),
            np.arange(70000) % 300, np.arange(70000), -np.arange(70000), np.arange(70000) // 1000]
    x = np.array(rows, np.float32)
    tokens = np.array([69999, 12345, 5, 299, 3, 0, 69999], np.int32)
    for top in (1, 5, 64):
        got = run(gpu_ctx, x, "f32", 1.0, tokens, top)
        verify(got[0], 1.0, tokens, top, *got[1:])


def test_masks_and_non_finite_rows(gpu_ctx):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((12, 5003)).astype(np.float32)
    x[0, rng.random(5003) < 0.9] = -np.inf
    x[1] = -np.inf                                     # nothing left
    x[2] = -np.inf
    x[2, 4000] = 1.5                                   # one token left
    x[3, 17] = np.nan
    x[4, 4999] = np.inf
    x[5, rng.random(5003) < 0.5] = np.finfo(np.float32).min  # masked by the type's lowest value
    x[6] = np.finfo(np.float32).min                    # all of them
    x[7] = np.nan
    x[8, [3, 900, 4000]] = [np.inf, np.nan, np.inf]
    x[9, :] = -np.inf
    x[9, [5, 9]] = [3.0, np.inf]
    x[10, :] = 3.0e38                                  # sums of logits would overflow
    x[10, 7] = -3.0e38
    x[11, 100] = -np.nan
    tokens = np.array([3, 3, 4000, 5, 4999, 11, 100, 0, 900, 9, 7, 100], np.int32)
    for dtype in ("f32", "f16"):
        y = x
        if dtype == "f16":
            with np.errstate(over="ignore", invalid="ignore"):
                y = x.astype(np.float16)
        for top in (0, 8, 64):
            got = run(gpu_ctx, y, dtype, 0.8, tokens, top)
            verify(got[0], 0.8, tokens, top, *got[1:])


def test_token_ids_outside_the_vocabulary(gpu_ctx):
    x = np.random.default_rng(8).standard_normal((6, 100)).astype(np.float32)
    tokens = np.array([-1, 100, -2, 2 ** 31 - 1, -2 ** 31, 99], np.int32)
    got = run(gpu_ctx, x, "f32", 1.0, tokens, 3)
    verify(got[0], 1.0, tokens, 3, *got[1:])


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 2), (4, 4), (8, 0), (5, 3), (13, 7)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strides_and_alignment(gpu_ctx, pad, shift, dtype):
    """What lies behind a row (NaN here) is not read as part of it."""
    rng = np.random.default_rng(9)
    for vocab in (1001, 40003):
        x = rng.standard_normal((5, vocab)) * 2
        tokens = rng.integers(0, vocab, 5).astype(np.int32)
        got = run(gpu_ctx, x, dtype, 1.0, tokens, 9, pad, shift)
        verify(got[0], 1.0, tokens, 9, *got[1:])


def test_parts_asked_for_alone(gpu_ctx):
    x = np.random.default_rng(10).standard_normal((3, 9000)).astype(np.float32)
    tokens = np.array([1, 2, 3], np.int32)
    full = run(gpu_ctx, x, "f32", 1.0, tokens, 6)
    alone = run(gpu_ctx, x, "f32", 1.0, None, 6, entropy=False)
    assert np.array_equal(alone[4], full[4]) and np.array_equal(alone[5], full[5])
    assert (alone[1] == 9).all() and (alone[2] == 9).all() and (alone[3] == 9).all()  # left as they were
    only = run(gpu_ctx, x, "f32", 1.0, tokens, 0, entropy=False)
    assert np.array_equal(only[1], full[1]) and np.array_equal(only[2], full[2]) and (only[3] == 9).all()


def test_calls_one_after_the_other_and_twice(gpu_ctx):
    """The workspace of one call serves the next, larger and smaller; equal inputs give equal bits."""
    rng = np.random.default_rng(11)
    shapes = [(1, 151936), (200, 4000), (3, 100), (64, 60000), (1, 151936), (1000, 2000)]
    data = [rng.standard_normal(s, dtype=np.float32) for s in shapes]
    tokens = [rng.integers(0, s[1], s[0]).astype(np.int32) for s in shapes]
    first = [run(gpu_ctx, x, "f32", 1.0, t, 20) for x, t in zip(data, tokens)]
    again = [run(gpu_ctx, x, "f32", 1.0, t, 20) for x, t in zip(data[::-1], tokens[::-1])][::-1]
    for a, b, t in zip(first, again, tokens):
        for u, v in zip(a[1:], b[1:]):
            assert np.array_equal(u.view(np.uint32), v.view(np.uint32))
        verify(a[0][:3], 1.0, t[:3], 20, *(g[:3] for g in a[1:]))


def test_agrees_with_the_sampler(gpu_ctx):
    """The alternatives of a row without ties are the sampler's candidates."""
    row = np.random.default_rng(12).permutation(151936).astype(np.float32) / 10000
    p = gpu_ctx.upload(row)
    try:
        _, ids, _ = S.sample_topk(gpu_ctx, p, row.size, 50, 0.7)
    finally:
        gpu_ctx.free(p)
    got = run(gpu_ctx, row[None], "f32", 0.7, None, 50)
    assert np.array_equal(got[4][0], ids)


def test_operands_are_checked(gpu_ctx):
    x = np.zeros((4, 100), np.float32)
    with Arrays(gpu_ctx) as mem:
        px, t, f, i = mem.up(x), mem.up(np.zeros(4, np.int32)), mem.up(np.zeros(4, np.float32)), mem.up(np.zeros(4, np.int32))

        def refused(text, *args):
            with pytest.raises(S.SocError, match=text) as e:
                S.logprobs(gpu_ctx, *args)
            assert e.value.code == SOC_ERR_INVALID

        refused("past the end", px, "f32", 100, 5, 100, 1.0, t, f, i, None, 0, None, None)
        refused("past the end", px, "f32", 101, 4, 100, 1.0, t, f, i, None, 0, None, None)
        refused("stride", px, "f32", 99, 4, 100, 1.0, t, f, i, None, 0, None, None)
        refused("not in device memory", x.ctypes.data, "f32", 100, 4, 100, 1.0, t, f, i, None, 0, None, None)
        refused("null", px, "f32", 100, 4, 100, 1.0, t, None, i, None, 0, None, None)
        refused("null", px, "f32", 100, 4, 100, 1.0, t, f, i, None, 1, None, f)
        refused("past the end", px, "f32", 100, 4, 100, 1.0, t, f, i, None, 2, i, f)
        refused("aligned", px, "f32", 100, 3, 100, 1.0, t, f, i, f + 2, 0, None, None)
