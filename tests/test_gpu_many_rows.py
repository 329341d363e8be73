"""More rows than one launch holds, which counts its threads in 32 bits: a wave
or a workgroup of a wave a row, 2^26 of them."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BEYOND = 2**26 + 1000


def test_distillation(gpu):
    """A vocabulary of two, every third row without a target: with a teacher that
    keeps one column, the loss is ln(1 + exp(other - kept))."""
    logits = torch.randn(BEYOND, 2, generator=torch.Generator(device="cuda").manual_seed(1),
                         device="cuda")
    row = torch.arange(BEYOND, device="cuda", dtype=torch.int32)
    kept = row % 3 != 0
    indptr = torch.zeros(BEYOND + 1, dtype=torch.int32, device="cuda")
    indptr[1:] = kept.cumsum(0)
    columns = (row % 2)[kept]
    A = gpu.CSRArray(data=torch.ones(columns.numel(), device="cuda"), indices=columns, indptr=indptr,
                     shape=(BEYOND, 2))
    at = (row % 2).long()[:, None]
    away = (logits.gather(1, 1 - at) - logits.gather(1, at))[:, 0]
    want = torch.where(kept, torch.nn.functional.softplus(away), 0.0)
    losses = gpu.distill_loss(logits, A)
    # sums of two terms of at most 2^-21 (8 + |logit|) each, as in the other tests
    assert float((losses - want).abs().max()) < 2.0**-21 * 16 * (1 + float(want.max()))
    both, grad = gpu.distill_value_and_grad(logits, A)
    assert torch.equal(both, losses)
    p = torch.where(kept, torch.sigmoid(away), 0.0)[:, None]
    assert float((grad.gather(1, at) + p).abs().max()) < 2.0**-21 * 32
    assert float((grad.gather(1, 1 - at) - p).abs().max()) < 2.0**-21 * 32


def test_attention_by_rows(gpu):
    """Heads of one value, a window of one: every query takes its own value."""
    tokens, heads = BEYOND // 64 + 1, 64
    q = torch.ones(1, tokens, heads, 1, device="cuda")
    v = torch.arange(tokens * heads, device="cuda").reshape(1, tokens, heads, 1) % 8191 + 1.0
    leaves = [q, q.clone(), v]
    for t in leaves:
        t.requires_grad_()
    out = gpu.window_attention(*leaves, window=1)
    assert torch.equal(out, v)
    dq, dk, dv = torch.autograd.grad(out, leaves, v)
    assert torch.equal(dv, v) and dq.abs().max() == 0 and dk.abs().max() == 0


def test_a_store(gpu):
    tokens, heads = BEYOND // 64 + 1, 64
    k = (torch.arange(tokens * heads, device="cuda") % 8191 + 1.0).reshape(1, tokens, heads, 1)
    ck, cv = torch.zeros(1, tokens, heads, 1, device="cuda"), torch.zeros(1, tokens, heads, 1, device="cuda")
    gpu.window_cache_store(k, -k, ck, cv)
    assert torch.equal(ck, k) and torch.equal(cv, -k)
