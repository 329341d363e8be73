"""torch.func.vmap of window attention and its gradients on the host path."""

from __future__ import annotations

import pytest
import torch

from _attention_vmap_checks import mapped_operands, no_tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mapped_operands(cpu, dtype):
    mapped_operands(cpu, "cpu", dtype)


def test_no_tokens(cpu):
    no_tokens(cpu, "cpu")
