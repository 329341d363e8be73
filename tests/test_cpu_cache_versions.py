"""Ring caches are written in place: torch is told, as by its own in-place
operations."""

from __future__ import annotations

import pytest
import torch


def caches():
    gen = torch.Generator().manual_seed(1)
    return [torch.randn(1, 6, 2, 8, generator=gen) for _ in range(2)]


def step(ms, ck, cv):
    ms.window_attention_step(torch.ones(1, 4, 8), torch.ones(1, 2, 8), torch.ones(1, 2, 8), ck, cv,
                             torch.tensor([3]), window=6)


def store(ms, ck, cv):
    ms.window_cache_store(torch.ones(1, 2, 2, 8), torch.ones(1, 2, 2, 8), ck, cv)


@pytest.mark.parametrize("write", [step, store])
@pytest.mark.parametrize("saved", ["whole", "view"])
def test_a_derivative_that_saved_the_cache_raises(cpu, write, saved):
    ck, cv = caches()
    k, v = (ck, cv) if saved == "whole" else (ck[:, 1:5], cv[:, 1:5])
    q = torch.randn(1, k.shape[1], 4, 8, requires_grad=True)
    out = cpu.window_attention(q, k, v, window=4)
    write(cpu, ck, cv)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("write", [step, store])
def test_versions(cpu, write):
    ck, cv = caches()
    write(cpu, ck, cv)
    assert ck._version == 1 and cv._version == 1
    with torch.inference_mode():
        ck, cv = caches()
        write(cpu, ck, cv)  # these have no versions
        assert (ck[0, 3 if write is step else 0] == 1).all()
