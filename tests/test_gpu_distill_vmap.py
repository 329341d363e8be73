"""torch.func.vmap of distillation."""

from __future__ import annotations

import pytest
import torch

from _distill_vmap_checks import mapped_students

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_mapped_students(gpu, dtype):
    mapped_students(gpu, "cuda", dtype)
