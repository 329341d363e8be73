"""Paged attention of wide heads over few keys, whole or cut by how many workgroups there are."""

from __future__ import annotations

import pytest
import torch

from _paged_checks import paged_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,keys", [(torch.float32, 240), (torch.float16, 500), (torch.bfloat16, 500)])
@pytest.mark.parametrize("dim", [200, 256])
@pytest.mark.parametrize("batch,tokens", [(8, 1), (40, 1), (40, 3), (290, 1)])
def test_wide_heads(gpu, dtype, keys, dim, batch, tokens):
    gen = torch.Generator().manual_seed(batch)
    starts = torch.randint(0, keys - tokens, (batch,), generator=gen)
    starts[::7], starts[1] = -1, keys - tokens
    paged_case(gpu, "cuda", dtype, starts.tolist(), tokens=tokens, heads=8, kv_heads=4, dim=dim, size=16,
               width=keys // 16 + 1)
