"""Accuracy of window attention's gradients on the host path."""

from __future__ import annotations

import pytest
import torch

from _gradient_checks import concentrated, gradients_in_norm, largest_share

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("score,share", [(0.0, 0.0), (9.0, 0.9), (11.0, 0.98), (13.0, 0.997)])
def test_attention_on_a_sink(cpu, dtype, score, share):
    """The gradient in a score is P (dP - delta): as P goes to one it is small
    beside both, and delta's error has to be small beside it."""
    pattern = {"window": 256, "sinks": 1}
    q, k, v, g = concentrated(1, 1, 400, 2, 1, 64, dtype, "cpu", score)
    assert largest_share(q, k, **pattern) > share
    gradients_in_norm(cpu, q, k, v, g, f"share {share}", **pattern)
