"""Scales beyond float32, in which scores are made."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("scale", [3e38, 1e39, -1e300, float("inf"), float("nan")])
def test_refused(cpu, scale):
    q, k = torch.ones(1, 4, 2, 8), torch.ones(1, 4, 1, 8)
    with pytest.raises(ValueError, match="scale must be finite"):
        cpu.window_attention(q, k, k, window=2, scale=scale)
    with pytest.raises(ValueError, match="scale must be finite"):
        cpu.window_attention(q.requires_grad_(), k, k, window=2, scale=scale)
    cache = torch.ones(1, 6, 1, 8)
    with pytest.raises(ValueError, match="scale must be finite"):
        cpu.window_attention_step(q[:, 0], k[:, 0], k[:, 0], cache, cache.clone(), torch.tensor([0]),
                                  window=2, scale=scale)


def test_the_largest(cpu):
    """A score that overflows is the softmax's, not the scale's."""
    q = torch.zeros(1, 3, 1, 4)
    v = torch.arange(12.0).reshape(1, 3, 1, 4)
    assert torch.equal(cpu.window_attention(q, q, v, window=1, scale=2e38), v)
