"""The ends of what the paged serving operators take. Tolerances are those of the operators' own tests."""
import numpy as np
import pytest

from tests.test_gpu_logprobs import run as run_logprobs, verify as verify_logprobs
from tests.test_gpu_paged import run_attention

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
