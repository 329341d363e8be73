"""Refusals of what would be cut to something else, in the operators' own words."""

from __future__ import annotations

import pytest
import torch


def test_complex_weights(cpu):
    A = cpu.csr_array((torch.ones(2), torch.tensor([0, 1]), torch.tensor([0, 1, 2])), shape=(2, 4))
    for weights in (torch.ones(2, dtype=torch.complex64), torch.tensor(1j)):
        with pytest.raises(TypeError, match="weights must be real"):
            cpu.distill_value_and_grad(torch.zeros(2, 4), A, weights)


@pytest.mark.parametrize("sinks", [4, 2**40, 2**63, 2**70])
def test_sinks_of_a_store(cpu, sinks):
    k = torch.ones(1, 3, 1, 2)
    with pytest.raises(ValueError, match="slots"):
        cpu.window_cache_store(k, k, torch.zeros(1, 4, 1, 2), torch.zeros(1, 4, 1, 2), sinks=sinks)
