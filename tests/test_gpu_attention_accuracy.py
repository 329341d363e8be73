"""Accuracy of window attention's kernels where rounding could cost more than
a rounding."""

from __future__ import annotations

import pytest
import torch

from _gradient_checks import concentrated, gradients_in_norm, largest_share

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [32, 64, 128, 132])
@pytest.mark.parametrize("score,share", [(0.0, 0.0), (10.0, 0.9), (12.0, 0.98), (14.0, 0.997)])
def test_attention_on_a_sink(gpu, dtype, dim, score, share):
    """The gradient in a score is P (dP - delta): as P goes to one it is small
    beside both, and delta's error has to be small beside it."""
    pattern = {"window": 512, "sinks": 1}
    q, k, v, g = concentrated(dim, 1, 900, 4, 2, dim, dtype, "cuda", score)
    assert largest_share(q, k, **pattern) > share
    gradients_in_norm(gpu, q, k, v, g, f"share {share}", **pattern)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_on_a_sink_in_parts(gpu, dtype):
    """Few blocks over long spans: the keys are cut and the parts joined."""
    pattern = {"window": 4096, "sinks": 2}
    q, k, v, g = concentrated(3, 1, 5000, 1, 1, 64, dtype, "cuda", 14.0)
    q, g = q[:, -70:], g[:, -70:]
    gradients_in_norm(gpu, q, k, v, g, "parts", **pattern)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("score", [7.0, 7.5, 8.0, 8.5])
def test_attention_on_a_late_key(gpu, dtype, score):
    """A key that takes most of the softmax after others have set its maximum:
    the exponentials beside it are of a smaller one's scale, and what rounding
    takes of its own must not become a factor of delta."""
    q, k, v, g = concentrated(4, 1, 600, 2, 1, 64, dtype, "cuda", score)
    k = k.roll(300, 1)
    g[:, :300] = 0  # the queries that see it in their second tile and later
    g[:, 460:] = 0
    g[:, 300:330] = 0
    gradients_in_norm(gpu, q, k, v, g, f"score {score}", window=160)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bits", [3.3, 5.3, 6.4, 7.3, 7.7, 9.1])
def test_attention_on_two_keys(gpu, dtype, bits):
    """A sink, a later key worth some bits more, and next to nothing beside them:
    the later one's exponential is not a power of two where the sink's maximum
    stays in use."""
    q, k, v, g = concentrated(5, 1, 600, 2, 1, 64, dtype, "cuda", 0.0)
    along = q[0, :, 0].double().mean(0)
    along /= along.norm()
    score = torch.full((600,), -12.0, dtype=torch.float64, device="cuda")
    score[0] = 10.0
    score[300] = 10.0 + bits * 0.6931
    k = (k.double() * 0.25 + (score[:, None, None] * 8.0 / 16.0) * along).to(dtype)
    g[:, :330] = 0
    g[:, 460:] = 0
    gradients_in_norm(gpu, q, k, v, g, f"{bits} bits", window=160, sinks=1)
