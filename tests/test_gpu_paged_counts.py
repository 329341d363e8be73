"""Paged attention that counts the keys seen: cuts, joins and the ends of pages, at
lengths where a sum over all keys would not show a lost step."""

from __future__ import annotations

import pytest
import torch

from _paged_counts import counts_case

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [33, 700, 2290, 5300, 20_012])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_sequence(gpu, dtype, n, dim):
    counts_case(gpu, "cuda", dtype, [n - 1], dim=dim, heads=8)
    counts_case(gpu, "cuda", dtype, [n - 3], dim=dim, tokens=3, heads=8, width=1400)  # cut at any length


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [16, 24])
def test_a_ragged_batch(gpu, dtype, size):
    gen = torch.Generator().manual_seed(size)
    starts = torch.exp(torch.rand(37, generator=gen) * 8.3).int().tolist()
    starts[3] = starts[9] = -1
    counts_case(gpu, "cuda", dtype, starts, dim=96, heads=6, kv_heads=2, size=size)
    counts_case(gpu, "cuda", dtype, starts, dim=64, tokens=5, lengths=[1, 5, 0, 4, 2, 3, 5] * 5 + [1, 2], size=size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start,tokens", [(0, 333), (600, 64), (5000, 250), (5000, 620), (20_000, 40)])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunks(gpu, dtype, start, tokens, dim):
    counts_case(gpu, "cuda", dtype, [start], tokens=tokens, dim=dim, heads=8)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_wide_heads(gpu, dtype):
    counts_case(gpu, "cuda", dtype, [2290, 14], dim=256)
    counts_case(gpu, "cuda", dtype, [2290, 700], tokens=90, dim=256)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window,sinks", [(700, 0), (700, 5), (2100, 33)])
@pytest.mark.parametrize("tokens", [1, 4, 130])
def test_windows(gpu, dtype, window, sinks, tokens):
    counts_case(gpu, "cuda", dtype, [5000, 90, 2300], tokens=tokens, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size,pages,tokens", [(16, 140, 1), (16, 141, 3), (24, 130, 2), (5, 841, 1)])
def test_shared_pages(gpu, dtype, size, pages, tokens):
    shared = size * pages
    starts = [shared + 7 * b % 300 for b in range(64)]
    starts[0], starts[1], starts[2] = -1, shared - 40, shared
    counts_case(gpu, "cuda", dtype, starts, tokens=tokens, shared=pages, size=size, dim=128)
