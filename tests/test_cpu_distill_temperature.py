"""Temperatures at the ends of what float32 holds."""

from __future__ import annotations

import pytest
import torch

from _distill_checks import all_forms, teacher_rows


@pytest.mark.parametrize("temperature", [1e-300, 1e-46, 1e-39, 1e-20, 1e20, 1e39, 1e300])
def test_refused(cpu, temperature):
    A = cpu.csr_array((torch.ones(2), torch.tensor([0, 1]), torch.tensor([0, 1, 2])), shape=(2, 4))
    logits = torch.zeros(2, 4)
    for f in (cpu.distill_loss, cpu.distill_value_and_grad):
        for z in (logits, logits.t().contiguous().t(), logits.clone().requires_grad_()):
            with pytest.raises(ValueError, match="temperature"):
                f(z, A, temperature=temperature)


@pytest.mark.parametrize("temperature", [1e-18, 1e-6, 1e3])
def test_taken(cpu, temperature):
    logits = torch.randn(3, 9, generator=torch.Generator().manual_seed(1))
    buffers = teacher_rows(1, 3, 9, [4, 0, 9], torch.float32, torch.int32)
    all_forms(cpu, logits, buffers, f"{temperature}", temperature=temperature, serial=9)
