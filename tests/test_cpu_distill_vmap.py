"""torch.func.vmap of distillation on the host path."""

from __future__ import annotations

import pytest
import torch

from _distill_vmap_checks import mapped_students


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mapped_students(cpu, dtype):
    mapped_students(cpu, "cpu", dtype)


def test_no_rows(cpu):
    A = cpu.CSRArray(data=torch.zeros(0), indices=torch.zeros(0, dtype=torch.int64),
                     indptr=torch.zeros(1, dtype=torch.int64), shape=(0, 4))
    assert torch.func.vmap(lambda x: cpu.distill_loss(x, A))(torch.zeros(3, 0, 4)).shape == (3, 0)


def test_mapped_teachers_are_refused(cpu):
    z, data = torch.zeros(3, 5), torch.ones(2, 3)
    indices, indptr = torch.tensor([0, 1, 2]), torch.tensor([0, 1, 2, 3])

    def loss(values):
        return cpu.distill_loss(z, cpu.CSRArray(data=values, indices=indices, indptr=indptr,
                                                shape=(3, 5)))

    with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
        torch.func.vmap(loss)(data)
