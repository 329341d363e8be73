"""Distillation over an empty vocabulary or without tokens, at any rank."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("lead", [(6,), (2, 3), (3, 1, 2), (2, 0), (0, 3)])
@pytest.mark.parametrize("vocab", [0, 4])
def test_empty(cpu, lead, vocab):
    rows = 1
    for n in lead:
        rows *= n
    A = cpu.CSRArray(data=torch.zeros(0), indices=torch.zeros(0, dtype=torch.int64),
                     indptr=torch.zeros(rows + 1, dtype=torch.int64), shape=(rows, vocab))
    logits = torch.zeros(*lead, vocab, requires_grad=True)
    losses = cpu.distill_loss(logits, A)
    assert losses.shape == lead and losses.sum() == 0
    grad, = torch.autograd.grad(losses.sum(), logits)
    assert grad.shape == logits.shape and grad.abs().sum() == 0
    losses, grad = cpu.distill_value_and_grad(logits, A, torch.ones(lead))
    assert losses.shape == lead and grad.shape == logits.shape and grad.abs().sum() == 0
