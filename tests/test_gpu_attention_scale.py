"""Window attention at scales that float32 hardly holds, or not at all."""

from __future__ import annotations

import pytest
import torch

from _attention_checks import forward_and_gradients, operands

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.0, 1e-300, 1e-46, -1e-46, 1e-45, 1e-40, 2e-38])
def test_scales_next_to_zero(gpu, dtype, scale):
    """Every score is zero: the mean of the values that are seen."""
    q, k, v, g = operands(1, 2, 150, 150, 4, 2, 64, dtype, "cuda")
    forward_and_gradients(gpu, q, k, v, g, f"{scale}", window=40, sinks=3, scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps(gpu, dtype):
    q, k, v = (torch.randn(2, n, 64).to(dtype).cuda() for n in (4, 2, 2))
    ck, cv = (torch.randn(2, 70, 2, 64).to(dtype).cuda() for _ in range(2))
    n = torch.tensor([200, 10], device="cuda")
    outs = [gpu.window_attention_step(q, k, v, ck, cv, n, window=60, scale=s) for s in (0.0, 1e-46)]
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
