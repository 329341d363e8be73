"""Distillation on the host path, against its definition in 64 bits; and the
refusals, which come before any device is touched."""

from __future__ import annotations

import ctypes

import pytest
import torch

import _capi
from _distill_checks import all_forms, teacher_rows

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype,teacher", [(F32, F32), (F16, F32), (BF16, BF16), (F32, F16)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_losses_and_gradients(cpu, dtype, teacher, index):
    logits = (torch.randn(9, 57, generator=torch.Generator().manual_seed(1)) * 2.5).to(dtype)
    buffers = teacher_rows(1, 9, 57, [5, 0, 57, 1], teacher, index, ordered=False)
    weights = torch.linspace(-1, 2, 9)
    weights[4] = 0
    all_forms(cpu, logits, buffers, "", temperature=2.0, weights=weights, serial=57)


def test_rank_three_logits_and_views(cpu):
    logits = torch.randn(2, 6, 40, generator=torch.Generator().manual_seed(2))[:, ::2, 3:33]
    all_forms(cpu, logits, teacher_rows(2, 6, 30, [4], F32, torch.int64), "view", serial=30)


def test_rows_without_a_target(cpu):
    """None stored, all -inf, columns outside: zero, whatever the logits."""
    logits = torch.full((4, 8), float("nan"))
    logits[3] = torch.linspace(-1, 1, 8)
    data = torch.tensor([float("-inf"), float("-inf"), 1.0, 2.0, 1.0, float("-inf")])
    indices = torch.tensor([1, 2, -1, 8, 3, 5])
    indptr = torch.tensor([0, 0, 2, 4, 6])
    losses, grad = all_forms(cpu, logits, (data, indices, indptr), "empty", serial=8)
    assert losses[:3].abs().max() == 0 and grad[:3].abs().max() == 0


def test_columns_stored_twice(cpu):
    logits = torch.randn(2, 5, generator=torch.Generator().manual_seed(3))
    buffers = (torch.tensor([1.0, 0.5, 2.0, 0.0, 0.0]), torch.tensor([3, 1, 3, 2, 2]),
               torch.tensor([0, 3, 5]))
    all_forms(cpu, logits, buffers, "twice", serial=5)


def test_impossible_columns(cpu):
    """A student's -inf: no probability; an infinite loss where the teacher
    keeps the column, and none where the teacher's own is -inf."""
    logits = torch.tensor([[0.0, 1.0, float("-inf"), 0.5]]).repeat(2, 1)
    buffers = (torch.tensor([1.0, 2.0, 1.0, float("-inf")]), torch.tensor([0, 2, 1, 2]),
               torch.tensor([0, 2, 4]))
    losses, _ = all_forms(cpu, logits, buffers, "impossible", serial=4)
    assert torch.isinf(losses[0]) and torch.isfinite(losses[1])


def test_gradient_against_differences(cpu):
    logits = torch.randn(2, 7, generator=torch.Generator().manual_seed(4))
    data, indices, indptr = teacher_rows(4, 2, 7, [3], F32, torch.int32)
    A = cpu.CSRArray(data=data, indices=indices, indptr=indptr, shape=(2, 7))
    _, grad = cpu.distill_value_and_grad(logits, A, torch.tensor([0.5, 2.0]), temperature=1.5)
    h = 2.0**-6
    for i in range(logits.numel()):
        sums = []
        for sign in (h, -h):
            logits.view(-1)[i] += sign
            loss = cpu.distill_loss(logits, A, temperature=1.5).double()
            sums.append(float(0.5 * loss[0] + 2.0 * loss[1]))
            logits.view(-1)[i] -= sign
        assert abs((sums[0] - sums[1]) / (2 * h) - float(grad.view(-1)[i])) < 2e-3


def test_one_weight_for_all_and_no_rows(cpu):
    logits = torch.randn(3, 4)
    A = cpu.csr_array((torch.ones(3), torch.tensor([0, 1, 2]), torch.tensor([0, 1, 2, 3])),
                      shape=(3, 4))
    _, one = cpu.distill_value_and_grad(logits, A, 0.25)
    _, each = cpu.distill_value_and_grad(logits, A, torch.full((3,), 0.25))
    assert torch.equal(one, each)
    none = cpu.CSRArray(data=torch.zeros(0), indices=torch.zeros(0, dtype=torch.int64),
                        indptr=torch.zeros(1, dtype=torch.int64), shape=(0, 4))
    losses, grad = cpu.distill_value_and_grad(torch.zeros(0, 4), none)
    assert losses.shape == (0,) and grad.shape == (0, 4)


def test_refusals(cpu):
    logits = torch.zeros(2, 4)
    A = cpu.csr_array((torch.ones(2), torch.tensor([0, 1]), torch.tensor([0, 1, 2])), shape=(2, 4))
    for f in (cpu.distill_loss, cpu.distill_value_and_grad):
        with pytest.raises(TypeError, match="CSRArray"):
            f(logits, logits)
        with pytest.raises(TypeError, match="logits"):
            f(logits.double(), A)
        with pytest.raises(ValueError, match="teacher of shape"):
            f(torch.zeros(3, 4), A)
        with pytest.raises(ValueError, match="tokens, vocabulary"):
            f(torch.zeros(4), A)
        for t in (0.0, -1.0, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="temperature"):
                f(logits, A, temperature=t)
        with pytest.raises(ValueError, match="no derivative in the teacher"):
            f(logits, cpu.CSRArray(data=torch.ones(2, requires_grad=True), indices=A.indices,
                                   indptr=A.indptr, shape=(2, 4)))
        with pytest.raises(TypeError, match="teachers"):
            f(logits, cpu.CSRArray(data=torch.ones(2, dtype=torch.complex64), indices=A.indices,
                                   indptr=A.indptr, shape=(2, 4)))
    with pytest.raises(ValueError, match="weights"):
        cpu.distill_value_and_grad(logits, A, torch.ones(3))
    leaf = logits.clone().requires_grad_()
    first, = torch.autograd.grad(cpu.distill_loss(leaf, A).sum(), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="second-order"):
        first.sum().backward()


def test_c_entry_points_refuse():
    """Status codes, before any HIP call."""
    L = _capi.lib()
    desc = (ctypes.c_char * 256)()
    assert L.msx_distill_loss(None, None, None, None) == _capi.EINVAL
    head = ctypes.cast(desc, ctypes.POINTER(ctypes.c_int32))
    head[0] = 3
    assert L.msx_distill_loss(desc, None, None, None) == _capi.ETYPE
    head[0] = 0
    assert L.msx_distill_loss(desc, None, None, None) == _capi.EINVAL  # temperature 0
    assert "temperature" in _capi.last_error()
