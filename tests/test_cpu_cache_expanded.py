"""Caches that several sequences would share by expansion are refused: each
writes its own token."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dim", [0, 1, 2])
def test_expanded_caches(cpu, which, dim):
    shape = [2, 6, 2, 8]
    shape[dim] = 1
    caches = [torch.zeros(2, 6, 2, 8), torch.zeros(2, 6, 2, 8)]
    caches[which] = torch.zeros(shape).expand(2, 6, 2, 8)
    row = torch.ones(2, 2, 8)
    with pytest.raises(ValueError, match="cannot be an expanded tensor"):
        cpu.window_attention_step(torch.ones(2, 4, 8), row, row, *caches, torch.tensor([0, 1]),
                                  window=4)
    with pytest.raises(ValueError, match="cannot be an expanded tensor"):
        cpu.window_cache_store(row[:, None], row[:, None], *caches)
    assert caches[0].abs().max() == 0 and caches[1].abs().max() == 0


def test_one_sequence(cpu):
    """A dimension of one has no stride of its own."""
    ck, cv = torch.zeros(6, 1, 8).expand(1, 6, 1, 8), torch.zeros(6, 1, 8)[None]
    cpu.window_attention_step(torch.ones(1, 4, 8), torch.ones(1, 1, 8), torch.ones(1, 1, 8), ck, cv,
                              torch.tensor([2]), window=4)
    assert ck[0, 2].min() == 1 and cv[0, 2].min() == 1
