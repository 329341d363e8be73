"""Where ``window_cache_store`` puts a chunk whose starts and lengths are of
different index types."""

from __future__ import annotations

import pytest
import torch

I32, I64 = torch.int32, torch.int64


@pytest.mark.parametrize("first", [0, 5, 2**31 - 2, 2**31 + 5, 2**40])
@pytest.mark.parametrize("lengths", [I32, I64])
def test_starts_of_64_bits(cpu, first, lengths):
    """A start beyond 32 bits is the position that it says."""
    k = torch.arange(1.0, 4.0).reshape(1, 3, 1, 1)
    ck, cv = torch.zeros(1, 6, 1, 1), torch.zeros(1, 6, 1, 1)
    cpu.window_cache_store(k, -k, ck, cv, sinks=2, starts=torch.tensor([first], dtype=I64),
                           lengths=torch.tensor([3], dtype=lengths))
    want = torch.zeros(6)
    for t in range(3):
        p = first + t
        want[p if p < 2 else 2 + (p - 2) % 4] = t + 1.0
    assert torch.equal(ck.flatten(), want) and torch.equal(cv, -ck)


def test_lengths_of_64_bits(cpu):
    k = torch.ones(1, 3, 1, 1)
    ck, cv = torch.zeros(1, 6, 1, 1), torch.zeros(1, 6, 1, 1)
    cpu.window_cache_store(k, k, ck, cv, starts=torch.tensor([1], dtype=I32),
                           lengths=torch.tensor([2**32 + 1], dtype=I64))
    assert ck.flatten().tolist() == [0, 1, 1, 1, 0, 0]


def test_other_types_are_refused(cpu):
    k = torch.ones(1, 3, 1, 1)
    ck, cv = torch.zeros(1, 6, 1, 1), torch.zeros(1, 6, 1, 1)
    for starts, lengths in (([1.7], [3]), ([1], [3.0]), ([True], [3])):
        with pytest.raises(ValueError, match="int32 or int64"):
            cpu.window_cache_store(k, k, ck, cv, starts=torch.tensor(starts),
                                   lengths=torch.tensor(lengths))
    assert ck.abs().max() == 0
