"""The best continuations of a request's beams (soc_beam_select) against the formula in 64 bits.

Tolerance. Within log S the terms 2^u have u off by 3 2^-24 |u| and the exponential by 2^-23, and they are added in chains of
at most 32 and a tree of 8: the relative error of S is at most (3 ln 2 H + 2 + 40) 2^-24, where H, the mean of |u| under the
row's own probabilities, is at most log2(vocab) <= 20. So a score is off by 84 2^-24, and by 2^-24 of itself from its
rounding. Rows and tokens are exact wherever the scores around theirs are further apart than that; equal rows are exact."""
import numpy as np
import pytest

import soc_amd as S
from soc_amd.capi import SOC_ERR_INVALID
from tests.device import NP, Arrays, guarded

pytestmark = pytest.mark.gpu
INF = np.inf


def all_scores(x, cum, t):
    """Scores of [rows][vocab] in 64 bits; -inf where a row or token offers nothing."""
    x = x.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        z = (x - x.max(-1, keepdims=True)) / (t if t > 0 else 1.0)
        s = z - np.log(np.exp(z).sum(-1, keepdims=True)) + cum.astype(np.float64)[:, None]
        good = np.isfinite(s.max(-1)) & np.isfinite(cum) & ~np.isnan(x).any(-1) & ~(x == INF).any(-1)
    return np.where(good[:, None] & ~np.isnan(s), s, -INF)


def want_of(x, cum, groups, beams, t, many):
    """A request's first `many`: (rows, tokens, scores), -1 and -inf where there are fewer."""
    vocab = x.shape[1]
    s = all_scores(x, cum, t).reshape(groups, beams * vocab)
    # by score, then row, then logit, then id: a stable sort by logit within the row comes first
    by_logit = np.argsort(-x.astype(np.float64), axis=-1, kind="stable") + (np.arange(groups * beams) % beams * vocab)[:, None]
    by_logit = by_logit.reshape(groups, beams * vocab)
    order = np.argsort(-np.take_along_axis(s, by_logit, 1), axis=-1, kind="stable")[:, : many + 1]
    at = np.take_along_axis(by_logit, order, 1)
    score = np.take_along_axis(s, at, 1)
    row = np.where(score > -INF, np.arange(groups)[:, None] * beams + at // vocab, -1)
    token = np.where(score > -INF, at % vocab, -1)
    return row, token, score


def run_beam(ctx, x, dtype, cum, groups, beams, t, stops, top, *, stride=None, offset=0, next_=True, alias=False):
    rows, vocab = x.shape
    stride = vocab if stride is None else stride
    flat = np.full(offset + rows * stride, np.nan, NP[dtype])
    flat[offset:].reshape(rows, stride)[:, :vocab] = x
    with Arrays(ctx) as mem:
        px, pc = mem.up(flat), mem.up(guarded(cum.astype(np.float32), 2, 3, 5.0))
        ptop = [mem.up(guarded(np.full(groups * top, 99, d), 2, 3, 55)) for d in (np.int32, np.int32, np.float32)]
        pnext = [mem.up(guarded(np.full(rows, 99, d), 2, 3, 55)) for d in (np.int32, np.int32, np.float32)]
        out = pc if alias else pnext[2]
        S.beam_select(ctx, px + offset * flat.itemsize, dtype, stride, groups, beams, vocab, t, pc + 8, stops, top,
                      *([p + 8 for p in ptop] if top else [None] * 3),
                      *([pnext[0] + 8, pnext[1] + 8, out + 8] if next_ else [None] * 3))
        got = [mem.down(p) for p in ptop] + [mem.down(p) for p in pnext[:2]] + [mem.down(out)]
        for g in got:
            assert (g[:2] == (5.0 if alias and g is got[5] else 55)).all()
            assert (g[-3:] == (5.0 if alias and g is got[5] else 55)).all()
        if not alias:
            assert np.array_equal(mem.down(pc)[2:-3], cum.astype(np.float32), equal_nan=True)
        if not next_:
            assert all((g[2:-3] == 99).all() for g in got[3:])
        return [g[2:-3].reshape(groups, -1) for g in got]


def check_list(got, want, scores, exact):
    """got (rows, tokens, scores) of one list against want's; `scores`: [rows][vocab] of all, 64 bits."""
    for g in range(got[0].shape[0]):
        wr, wt, ws = (w[g] for w in want)
        seen = set()
        for k in range(got[0].shape[1]):
            r, tok, s = int(got[0][g, k]), int(got[1][g, k]), float(got[2][g, k])
            if ws[k] == -INF:
                assert (r, tok, s) == (-1, -1, -INF)
                continue
            tol = 84 * 2.0 ** -24
            if not exact:
                near = [ws[i] for i in (k - 1, k + 1) if 0 <= i < ws.size and np.isfinite(ws[i])]
                clear = all(abs(v - ws[k]) > 2 * tol for v in near)
            if exact or clear:
                assert (r, tok) == (wr[k], wt[k]), (g, k)
            assert (r, tok) not in seen
            seen.add((r, tok))
            assert abs(scores[r, tok] - ws[k]) <= 2 * tol
            assert abs(s - scores[r, tok]) <= tol + 2.0 ** -24 * abs(s), (g, k, s, scores[r, tok])


def check(ctx, x, dtype, cum, groups, beams, t=1.0, stops=(), top=0, exact=False, **kw):
    x, cum = x.astype(NP[dtype]), cum.astype(np.float32)
    got = run_beam(ctx, x, dtype, cum, groups, beams, t, list(stops), top, **kw)
    scores = all_scores(x, cum.astype(np.float32), t)
    check_list(got[:3], [w[:, :top + 1] for w in want_of(x, cum, groups, beams, t, top)], scores, exact)
    if kw.get("next_", True):
        allowed = x.copy()
        allowed[:, list(stops)] = -INF  # not offered, but in the sums
        masked = scores.copy()
        masked[:, list(stops)] = -INF
        order = want_of(x, cum, groups, beams, t, beams * (1 + len(stops)) + 1)
        rows, tokens, vals = [], [], []
        for g in range(groups):
            on = [k for k in range(order[0].shape[1]) if order[0][g, k] >= 0 and order[1][g, k] not in stops][: beams + 1]
            pad = beams + 1 - len(on)
            rows.append([order[0][g, k] for k in on] + [-1] * pad)
            tokens.append([order[1][g, k] for k in on] + [-1] * pad)
            vals.append([order[2][g, k] for k in on] + [-INF] * pad)
        check_list(got[3:], [np.array(rows), np.array(tokens), np.array(vals)], masked, exact)
    return got


def logits(rng, rows, vocab, spread=2.5):
    x = rng.normal(0, spread, (rows, vocab))
    x[np.arange(rows)[:, None], rng.integers(0, vocab, (rows, 3))] += rng.random((rows, 3)) * 8
    return x


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("groups,beams,vocab,stops,top,t", [
    (1, 1, 1, 0, 1, 1.0), (1, 1, 5, 0, 3, 1.0), (2, 3, 7, 1, 6, 0.7), (1, 4, 1000, 1, 8, 1.0), (3, 2, 8191, 2, 5, 1.3),
    (2, 4, 8192, 0, 4, 1.0), (2, 4, 8193, 1, 0, 0.5), (1, 3, 16384, 1, 6, 1.0), (1, 3, 16385, 1, 64, 1.0),
    (5, 8, 30000, 1, 16, 1.0), (1, 4, 151936, 1, 8, 1.0), (2, 32, 9000, 1, 64, 1.0), (2, 64, 300, 0, 64, 1.0),
    (1, 21, 20000, 2, 64, 2.0), (3, 16, 2, 1, 30, 1.0), (1, 2, 262145, 1, 4, 1.0), (1, 2, 1 << 20, 3, 9, 1.0),
    (300, 1, 700, 1, 2, 1.0), (2, 7, 40000, 8, 1, 0.0), (2, 5, 600, 1, 10, -3.0)])
def test_beam(gpu_ctx, dtype, groups, beams, vocab, stops, top, t):
    rng = np.random.default_rng(vocab + beams)
    x, cum = logits(rng, groups * beams, vocab), -20 * rng.random(groups * beams)
    stop = rng.choice(vocab, min(stops, vocab), replace=False).tolist()
    for s in stop:
        x[:, s] += 10 * rng.random(groups * beams)
    check(gpu_ctx, x, dtype, cum, groups, beams, t, stop, top)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab,stride,offset", [(1001, 1001, 0), (1001, 1003, 1), (8200, 8201, 3), (20001, 20005, 2), (64, 67, 5)])
def test_beam_strides(gpu_ctx, dtype, vocab, stride, offset):
    rng = np.random.default_rng(vocab)
    x, cum = logits(rng, 12, vocab), -5 * rng.random(12)
    a = check(gpu_ctx, x, dtype, cum, 3, 4, 1.0, [7], 8, stride=stride, offset=offset)
    b = check(gpu_ctx, x, dtype, cum, 3, 4, 1.0, [7], 8, alias=True)
    for u, v in zip(a, b):  # the alignment of a row changes no bit
        assert np.array_equal(u, v)
    check(gpu_ctx, x, dtype, cum, 3, 4, 1.0, [7], 8, next_=False)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [9, 700, 30001])
def test_beam_ties(gpu_ctx, dtype, vocab):
    """Equal beams, equal logits: by row, then logit, then id; wherever the rows lie."""
    rng = np.random.default_rng(vocab)
    one = np.round(rng.normal(0, 1, (1, vocab)) * 2) / 2  # many equal logits
    x = np.repeat(one, 8, 0)
    check(gpu_ctx, x, dtype, np.full(8, -3.0), 2, 4, 1.0, [1], 8, exact=True, stride=vocab + 1, offset=1)
    check(gpu_ctx, np.zeros((64, vocab)), dtype, np.zeros(64), 1, 64, 1.0, [], 64, exact=True)
    check(gpu_ctx, np.zeros((32, vocab)), dtype, np.zeros(32), 1, 32, 1.0, [0], 64, exact=True)
    check(gpu_ctx, np.full((6, vocab), 7.5), dtype, np.full(6, -1e30), 2, 3, 1.0, [], 5, exact=True)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [5, 600, 25000])
def test_beam_masks(gpu_ctx, dtype, vocab):
    """Masked tokens, rows of nothing else, beams that are none, NaN and +inf: what is left offers, the rest does not."""
    rng = np.random.default_rng(vocab)
    x, cum = logits(rng, 24, vocab), -9 * rng.random(24)
    x[rng.random(x.shape) < 0.5] = -INF
    x[1] = -INF
    x[4:8] = -INF  # a request without any continuation
    x[8, vocab // 2], x[9, vocab - 1], x[10, 0] = INF, np.nan, np.nan
    x[13] = -INF
    x[13, 3] = -2.0  # one token
    cum[16:20] = [0, -INF, -INF, -INF]  # the first step
    cum[20:24] = [np.nan, INF, -INF, -1.0]
    got = check(gpu_ctx, x, dtype, cum, 6, 4, 1.0, [2], 12)
    assert (got[0][1] == -1).all() and (got[3][1] == -1).all() and (got[2][1] == -INF).all()
    assert set(got[0][2].tolist()) <= {11, -1} and set(got[0][4].tolist()) <= {16, -1}
    x[11] = np.nan
    check(gpu_ctx, x, dtype, cum, 6, 4, 1.0, [2], 12)
    check(gpu_ctx, np.full((4, vocab), np.nan), dtype, np.zeros(4), 1, 4, 1.0, [], 4)
    check(gpu_ctx, np.full((4, vocab), INF), dtype, np.zeros(4), 1, 4, 1.0, [], 4)


@pytest.mark.parametrize("t", [1e-30, 1e-3, 1.0, 1e6, 2.0 ** 100])
def test_beam_extreme_logits(gpu_ctx, t):
    """Logits further apart than fp32 reaches, scores far from zero."""
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (4, 3000))
    x[0, :5] = [3.4e38, -3.4e38, 3.3e38, -3.3e38, 0]
    x[1] *= 1e-40
    x[2] += 1e6
    x = x.astype(np.float32)
    cum = np.array([-1e6, -3.0, -4.0, -1e-3])
    got = run_beam(gpu_ctx, x, "f32", cum, 2, 2, t, [], 6)
    scores = all_scores(x, cum.astype(np.float32), t)
    with np.errstate(over="ignore"):
        for g in range(2):
            for k in range(6):
                r, tok, s = int(got[0][g, k]), int(got[1][g, k]), got[2][g, k]
                w = scores[r, tok]
                assert s == np.float32(w) or abs(s - w) <= 84 * 2.0 ** -24 + 2.0 ** -23 * abs(w)


def test_beam_more_rows_than_a_launch(gpu_ctx):
    """520 requests of 32 beams with 64 continuations each: the workspace holds some of them at a time."""
    rng = np.random.default_rng(8)
    vocab, beams, tile, times = 16400, 32, 4, 130
    x = logits(rng, tile * beams, vocab).astype(np.float16)
    cum = -5 * rng.random(tile * beams)
    groups = tile * times
    got = run_beam(gpu_ctx, np.tile(x, (times, 1)), "f16", np.tile(cum, times), groups, beams, 1.0, [4], 64)
    one = check(gpu_ctx, x, "f16", cum, tile, beams, 1.0, [4], 64)
    for k in range(6):
        g = got[k].reshape(times, tile, -1)
        shift = (np.arange(times) * tile * beams)[:, None, None] if k in (0, 3) else 0
        assert np.array_equal(g - shift, np.broadcast_to(one[k], g.shape))


def test_beam_calls_in_a_row(gpu_ctx):
    """Queued calls of different sizes, the workspace growing between them: each leaves the counters clear for the next."""
    rng = np.random.default_rng(9)
    for groups, beams, vocab in [(1, 2, 100), (3, 4, 20000), (1, 1, 70000), (40, 8, 9000), (3, 4, 20000), (2, 2, 8)]:
        x, cum = logits(rng, groups * beams, vocab), -5 * rng.random(groups * beams)
        check(gpu_ctx, x, "f32", cum, groups, beams, 1.0, [3], min(64, 2 * beams))


def test_beam_refuses(gpu_ctx):
    with Arrays(gpu_ctx) as mem:
        x, f, i = mem.up(np.zeros(4000, np.float32)), mem.up(np.zeros(64, np.float32)), mem.up(np.zeros(64, np.int32))

        def call(stride=1000, groups=2, scores=f, top=2, top_scores=f + 64, next_rows=i + 128, next_tokens=i + 160, next_scores=f + 160):
            S.beam_select(gpu_ctx, x, "f32", stride, groups, 2, 1000, 1.0, scores, [], top, i, i + 64, top_scores, next_rows,
                          next_tokens, next_scores)

        for kw, text in [({"stride": 999}, "stride"), ({"stride": 1001}, "allocation"), ({"groups": 3}, "allocation"),
                         ({"scores": None}, "null"), ({"scores": 4096}, "device memory"), ({"top_scores": f + 66}, "aligned"),
                         ({"next_tokens": None}, "null"), ({"next_scores": f + 244}, "allocation"),
                         ({"top": 30}, "allocation")]:
            with pytest.raises(S.SocError, match=text) as e:
                call(**kw)
            assert e.value.code == SOC_ERR_INVALID
        call()
        gpu_ctx.synchronize()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("beams,top", [(2, 6), (4, 8), (4, 40), (9, 18)])
def test_beam_of_equal_scores(gpu_ctx, dtype, beams, top):
    """A temperature at which all tokens are equally likely: a beam's come by logit, whichever part of the row they lie in."""
    rng = np.random.default_rng(top)
    x = rng.normal(0, 1, (2 * beams, 30001))
    check(gpu_ctx, x, dtype, np.full(2 * beams, -1.5), 2, beams, 2.0 ** 100, [], top, exact=True)


@pytest.mark.parametrize("beams,top", [(1, 64), (2, 6), (4, 64), (64, 64)])
def test_beam_of_the_largest_vocabulary(gpu_ctx, beams, top):
    rng = np.random.default_rng(beams)
    x = rng.standard_normal((beams, 1 << 20), np.float32) * np.float32(2.5)
    check(gpu_ctx, x, "f16", -5 * rng.random(beams), 1, beams, 1.0, [], top)
