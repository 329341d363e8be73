"""The counting check of paged attention: on the host, and that it sees what it is for."""

from __future__ import annotations

import pytest
import torch

from _attention_reference import UNIT
from _paged_counts import counted, counts_case, marks, outside

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 0), (70, 5)])
def test_on_the_host(cpu, dtype, window, sinks):
    counts_case(cpu, "cpu", dtype, [0, 40, -1, 300], tokens=3, lengths=[3, 1, 0, 2], window=window, sinks=sinks,
                size=5)
    counts_case(cpu, "cpu", dtype, [64, 32, 70], shared=2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [33, 700, 2290, 5300, 20_012])
@pytest.mark.parametrize("dim", [64, 128])
def test_that_a_mistake_is_seen(dtype, n, dim):
    """Results without a step of 32 keys, with one twice, without a part or with one twice are
    outside at every length tested; a single key more or less is while rounding allows it."""
    want = counted(n - 1, 1, dim, n)
    assert not outside(want.to(dtype), want, dtype).any()
    keys = marks(torch.arange(n), dim)
    steps = range(0, n, 32) if n < 6000 else range(0, n, 32 * 17)
    for length, starts in ((32, steps), (n // 3, (0, n // 3, n - n // 3))):
        for first in starts:
            some = keys[first:first + length]
            for sign in (-1, 1):
                wrong = (keys.sum(0) + sign * some.sum(0)) / (n + sign * len(some))
                assert outside(wrong.to(dtype), want[0], dtype).any(), (first, length, sign)
    if n * (UNIT[dtype] + 2.0**-18) * 2 < dim // 2 - 1:
        for first in range(0, n, max(n // 50, 1)):
            wrong = (keys.sum(0) - keys[first]) / (n - 1)
            assert outside(wrong.to(dtype), want[0], dtype).any(), first
