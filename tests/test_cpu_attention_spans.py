"""Window attention over spans wider than any sequence."""

from __future__ import annotations

import sys

import pytest
import torch

from _attention_checks import operands


@pytest.mark.parametrize("window,sinks", [
    (2**40 - 1, 0), (2**40, 0), (sys.maxsize, 0), (2**70, 0), (3, 2**40), (3, sys.maxsize), (3, 2**70)])
def test_wider_than_any_sequence(cpu, window, sinks):
    """The pattern is the causal one, and so are its derivatives."""
    q, k, v, g = operands(1, 2, 9, 9, 4, 2, 8, torch.float32, "cpu")

    def outputs(**pattern):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = cpu.window_attention(*leaves, **pattern)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    for got, want in zip(outputs(window=window, sinks=sinks), outputs(window=9)):
        assert torch.equal(got, want)
