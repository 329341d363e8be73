"""Window attention's float16 gradients at upstream gradients far from one:
what the products in between hold must not run out of float16's range where
the gradients themselves do not."""

from __future__ import annotations

import pytest
import torch

from _attention_checks import operands
from _gradient_checks import gradients_in_norm

pytestmark = pytest.mark.gpu

F16 = torch.float16


@pytest.mark.parametrize("power", [-20, -17, -14, -7, 0, 7, 13])
@pytest.mark.parametrize("tokens,window,sinks,dim", [(1500, 1024, 4, 64), (700, 600, 0, 128), (300, 40, 70, 32)])
def test_upstream_of_any_size(gpu, power, tokens, window, sinks, dim):
    """Small ones as a mean over many tokens gives, large ones as loss scaling
    does; 700 tokens in a window of 600 have flat rows whose dS is a thousandth
    of the upstream's."""
    q, k, v, g = operands(tokens, 1, tokens, tokens, 4, 2, dim, F16, "cuda")
    gradients_in_norm(gpu, q, k, v, g * 2.0**power, f"2^{power}", window=window, sinks=sinks)


def test_upstream_of_many_sizes(gpu):
    """Tokens whose upstream gradients differ by 2^24 beside each other: each
    row of dq is as good as alone, each key's sum as its largest terms."""
    q, k, v, g = operands(5, 1, 640, 640, 2, 2, 64, F16, "cuda")
    powers = torch.arange(640, device="cuda") % 25 - 14
    g = (g.float() * torch.exp2(powers.float())[None, :, None, None]).to(F16)
    pattern = {"window": 500, "sinks": 2}
    gradients_in_norm(gpu, q, k, v, g, "mixed", **pattern)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    dq, = torch.autograd.grad(gpu.window_attention(*leaves, **pattern), leaves[:1], g)
    for power in range(25):
        rows = (torch.arange(640, device="cuda") % 25 == power)[None, :, None, None]
        one, = torch.autograd.grad(gpu.window_attention(*leaves, **pattern), leaves[:1],
                                   torch.where(rows, g, 0))
        assert torch.equal(torch.where(rows, dq, 0), one)
