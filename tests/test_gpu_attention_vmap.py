"""torch.func.vmap of window attention and its gradients."""

from __future__ import annotations

import pytest
import torch

from _attention_vmap_checks import mapped_operands, no_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_mapped_operands(gpu, dtype):
    mapped_operands(gpu, "cuda", dtype)


def test_no_tokens(gpu):
    no_tokens(gpu, "cuda")
