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
