"""The ends of what the paged serving operators take: logits further apart than 32 bits reach, scales and queries at the
ends of their range, infinities and NaN among the queries, ropes of every scaling in the append, and what a row's bits may
depend on. Tolerances are those of the operators' own tests."""
import math

import numpy as np
import pytest

import soc_amd as S
from tests.device import Arrays
from tests.test_gpu_logprobs import run as run_logprobs, verify as verify_logprobs
from tests.test_gpu_paged import attend, run_attention
from tests.test_gpu_rope import check as rope_check, frequencies, rotate

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [1.0, 1.5, 2.5, 1000.0, 1e30, 1e38, 3e38])
@pytest.mark.parametrize("vocab", [300, 20000])
def test_logprobs_of_logits_further_apart_than_fp32_reaches(gpu_ctx, vocab, t):
    """x - M beyond the largest fp32 number, divided by a temperature that brings it back: the quotient counts, in the log
    probabilities and, where the temperature is that high, in the sums."""
    rng = np.random.default_rng(int(vocab))
    x = (rng.uniform(-1, 1, (4, vocab)) * 3.4e38).astype(np.float32)
    x[1, :: 2] = np.finfo(np.float32).min
    x[2] = np.where(rng.random(vocab) < 0.5, np.finfo(np.float32).max, np.finfo(np.float32).min)
    x[3, : vocab - 5] = -np.inf
    tokens = np.array([0, 2, vocab // 2, vocab - 1], np.int32)
    tokens[2] = int(np.argmin(x[2]))
    got = run_logprobs(gpu_ctx, x, "f32", t, tokens, 64)
    verify_logprobs(got[0], t, tokens, 64, *got[1:])
    got = run_logprobs(gpu_ctx, x, "f32", t, tokens, 0)
    verify_logprobs(got[0], t, tokens, 0, *got[1:])


@pytest.mark.parametrize("scale", [3e38, -3e38, 1e-38])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_scales_at_the_ends_of_fp32(gpu_ctx, scale, hd):
    """A scale times log2(e) may pass fp32 where the scores do not."""
    run_attention(gpu_ctx, "f32", [70, 900, 5], 8, 2, hd, 16, scale=scale, q_scale=1e-38 if abs(scale) > 1 else 1e37)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("nq,nkv", [(8, 2), (10, 1)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_attention_of_non_finite_queries(gpu_ctx, bad, nq, nkv, dtype):
    """Heads whose query holds a NaN or infinity are NaN, as the formula's are (some score is NaN, or the largest infinite);
    every other head of the same group and row has the bits it has without them."""
    rng = np.random.default_rng(21)
    n, hd, page, length = 3, 128, 16, 600
    pages = n * -(-length // page)
    table = rng.permutation(pages).astype(np.int32).reshape(n, -1)
    keys, values = (rng.standard_normal((pages, nkv, page, hd)).astype(np.float16) for _ in range(2))
    clean = rng.standard_normal((n, nq, hd)).astype(np.float32 if dtype == "f32" else np.float16)
    dirty = clean.copy()
    dirty[1, 1, 77] = bad
    dirty[2, nq - 1, [0, 127]] = bad
    hit = np.zeros((n, nq), bool)
    hit[1, 1] = hit[2, nq - 1] = True
    lens = np.array([length, length - 3, 1], np.int32)
    found = []
    with Arrays(gpu_ctx) as mem:
        cache = S.PagedCache(mem.up(keys), mem.up(values), pages, page, nkv, hd)
        pt, pl = mem.up(table), mem.up(lens)
        for q in (clean, dirty):
            po, ps = mem.up(np.zeros_like(q)), mem.up(np.zeros((n, nq), np.float32))
            S.paged_attention_decode(gpu_ctx, cache, mem.up(q), nq * hd, dtype, pt, table.shape[1], table.shape[1], pl, n, nq,
                                     0.0, po, nq * hd, ps)
            found.append((mem.down(po), mem.down(ps)))
    (a, la), (b, lb) = found
    assert np.isfinite(a).all() and np.isfinite(la).all()
    assert np.isnan(b[hit]).all() and np.isnan(lb[hit]).all()
    assert np.array_equal(a[~hit], b[~hit]) and np.array_equal(la[~hit], lb[~hit])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("scaling,factor,d,layout", [("linear", 4.0, 128, "half"), ("ntk", 2.0, 64, "interleaved"),
                                                     ("yarn", 4.0, 128, "half"), ("yarn", 32.0, 72, "interleaved")])
def test_append_with_scaled_ropes(gpu_ctx, scaling, factor, d, layout, dtype):
    """Queries and cached keys of a scaled rope, YaRN's gain on both; values are not scaled."""
    rng = np.random.default_rng(22)
    rows, nq, nkv, hd, page = 37, 4, 2, 128, 16
    x = (rng.standard_normal((rows, nq + 2 * nkv, hd)) * 2).astype(np.float32 if dtype == "f32" else np.float16)
    positions = rng.integers(0, 200000, rows).astype(np.int32)
    slots = rng.permutation(5 * page)[:rows].astype(np.int32)
    row, size = (nq + 2 * nkv) * hd, x.itemsize
    with Arrays(gpu_ctx) as mem:
        p, pp, ps = mem.up(x), mem.up(positions), mem.up(slots)
        pk, pv = (mem.up(np.zeros((5, nkv, page, hd), np.float16)) for _ in range(2))
        pq = mem.up(np.zeros((rows, nq * hd), x.dtype))
        rope = S.Rope(gpu_ctx, hd, d, layout=layout, scaling=scaling, factor=factor, original_max_position=32768)
        S.paged_append(gpu_ctx, S.PagedCache(pk, pv, 5, page, nkv, hd), rope, p, row, p + nq * hd * size, row,
                       p + (nq + nkv) * hd * size, row, dtype, pq, nq * hd, rows, nq, pp, ps)
        q, keys, values = mem.down(pq).reshape(rows, nq, hd), mem.down(pk), mem.down(pv)
        rope.close()
    gain = 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0
    want, tol = rotate(x[:, : nq + nkv], positions, d, layout, frequencies(d, 1e6, scaling, factor, 32768), gain)
    rope_check(q, want[:, :nq], tol[:, :nq], dtype)
    rope_check(keys[slots // page, :, slots % page], want[:, nq:], tol[:, nq:], "f16")
    assert np.array_equal(values[slots // page, :, slots % page], x[:, nq + nkv:].astype(np.float16))


def test_attention_bits_do_not_depend_on_the_other_sequences(gpu_ctx):
    """With the number of sequences and the table's width given, a sequence's bits follow from its own query, keys, values
    and length: the others may have any length, or none, and any contents."""
    rng = np.random.default_rng(23)
    n, nq, nkv, hd, page, width, length = 6, 8, 2, 64, 16, 200, 2000
    pages = n * width
    held = []
    for other in (0, 7, 3200):
        keys, values = (rng.standard_normal((pages, nkv, page, hd)).astype(np.float16) for _ in range(2))
        q = rng.standard_normal((n, nq * hd)).astype(np.float32)
        own = np.random.default_rng(24)
        table = rng.permutation(pages).astype(np.int32).reshape(n, width)
        q[3] = own.standard_normal(nq * hd)
        keys[table[3]], values[table[3]] = (own.standard_normal((width, nkv, page, hd)).astype(np.float16) for _ in range(2))
        lens = np.full(n, other, np.int32)
        lens[3] = length
        with Arrays(gpu_ctx) as mem:
            po, pl = mem.up(np.zeros_like(q)), mem.up(np.zeros((n, nq), np.float32))
            S.paged_attention_decode(gpu_ctx, S.PagedCache(mem.up(keys), mem.up(values), pages, page, nkv, hd), mem.up(q),
                                     nq * hd, "f32", mem.up(table), width, width, mem.up(lens), n, nq, 0.0, po, nq * hd, pl)
            held.append((mem.down(po)[3].copy(), mem.down(pl)[3].copy()))
        mine = [t[table[3]].transpose(1, 0, 2, 3).reshape(nkv, -1, hd)[:, :length] for t in (keys, values)]
        want, _, tol, _ = attend(q[3].reshape(nq, hd), *mine, 1 / math.sqrt(hd))
        assert (np.abs(held[-1][0].reshape(nq, hd) - want) <= tol).all()
    for out, lse in held[1:]:
        assert np.array_equal(out.view(np.uint32), held[0][0].view(np.uint32))
        assert np.array_equal(lse.view(np.uint32), held[0][1].view(np.uint32))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_logprob_bits_do_not_depend_on_the_other_rows(gpu_ctx, dtype):
    rng = np.random.default_rng(25)
    x = (rng.standard_normal((40, 20000)) * 3).astype(np.float32)
    tokens = rng.integers(0, 20000, 40).astype(np.int32)
    whole = run_logprobs(gpu_ctx, x, dtype, 0.7, tokens, 9)
    for r in (0, 17, 39):
        alone = run_logprobs(gpu_ctx, x[r: r + 1], dtype, 0.7, tokens[r: r + 1], 9)
        for a, b in zip(whole[1:], alone[1:]):
            assert np.array_equal(a[r: r + 1].view(np.uint32), b.view(np.uint32))
