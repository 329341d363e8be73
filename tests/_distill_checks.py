"""Checks of distillation that run on either device."""

from __future__ import annotations

import torch

from _distill_reference import check, reference


def teacher_rows(seed, rows, vocab, counts, dtype, index, *, ordered=True):
    """CSR buffers (CPU) of a teacher with ``counts[i]`` distinct columns in
    row i, ascending or in any order."""
    gen = torch.Generator().manual_seed(seed)
    columns, indptr = [], [0]
    for i in range(rows):
        c = torch.randperm(vocab, generator=gen)[:counts[i % len(counts)]]
        columns.append(c.sort().values if ordered else c)
        indptr.append(indptr[-1] + len(c))
    indices = torch.cat(columns) if columns else torch.zeros(0, dtype=torch.int64)
    data = (torch.randn(len(indices), generator=gen) * 2 + 6).to(dtype)
    return data, indices.to(index), torch.tensor(indptr, dtype=index)


def all_forms(ms, logits, buffers, what, *, temperature=1.0, weights=None, serial=1):
    """Losses, losses with gradient and the derivative against the definition."""
    device = logits.device
    data, indices, indptr = (t.to(device) for t in buffers)
    rows = indptr.numel() - 1
    teacher = ms.CSRArray(data=data, indices=indices, indptr=indptr,
                          shape=(rows, logits.shape[-1]))
    want, want_grad = reference(logits, data, indices, indptr, temperature=temperature,
                                weights=weights, serial=serial)
    losses = ms.distill_loss(logits.detach(), teacher, temperature=temperature)
    assert losses.dtype == torch.float32 and losses.shape == logits.shape[:-1]
    check(losses, want, f"{what} loss")
    w = None if weights is None else weights.reshape(logits.shape[:-1])
    both = ms.distill_value_and_grad(logits.detach(), teacher, w, temperature=temperature)
    check(both[0], want, f"{what} loss of both")
    assert both[1].dtype == logits.dtype and both[1].shape == logits.shape
    check(both[1], want_grad, f"{what} gradient of both")
    leaf = logits.detach().requires_grad_()
    tracked = ms.distill_loss(leaf, teacher, temperature=temperature)
    check(tracked, want, f"{what} tracked loss")
    up = torch.ones_like(tracked) if w is None else w.to(device).float()
    grad, = torch.autograd.grad(tracked, leaf, up)
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    check(grad, want_grad, f"{what} derivative")
    return both
