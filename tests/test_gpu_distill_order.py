"""Distillation from teacher rows whose columns are out of order, as a
teacher's largest logits are when they lie by value: many of them, and columns
that are stored more than once."""

from __future__ import annotations

import pytest
import torch

from _distill_checks import all_forms, teacher_rows

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def student(seed, rows, vocab, dtype):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen) * 2.5).to(dtype).cuda()


def csr(rows, dtype=F32, index=torch.int32):
    """Rows of (columns, values) as CSR buffers."""
    indptr = torch.tensor([0] + [len(c) for c, _ in rows]).cumsum(0)
    return (torch.cat([v for _, v in rows]).to(dtype), torch.cat([c for c, _ in rows]).to(index),
            indptr.to(index))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab,counts", [
    (131_072, [40_000, 131_072]), (50_257, [50_257, 3000]), (4000, [4000, 2]), (300_007, [70_000, 64])])
def test_many_columns_out_of_order(gpu, dtype, vocab, counts):
    """The reads of a row grow with its kept columns, not with their square."""
    buffers = teacher_rows(vocab, 2, vocab, counts, F32, torch.int32, ordered=False)
    all_forms(gpu, student(vocab, 2, vocab, dtype), buffers, f"{vocab}", serial=vocab // 64)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab,kept", [(40, 90), (1009, 3000), (8193, 500), (60_000, 5000), (200_003, 30_000)])
def test_columns_stored_many_times(gpu, dtype, vocab, kept):
    """Columns drawn with repetition, and one that most entries share; beyond
    one pass of marks, columns out of range among them."""
    gen = torch.Generator().manual_seed(kept)
    rows = []
    for i in range(3):
        c = torch.randint(0, vocab, (kept,), generator=gen)
        if i == 1:
            c[::2] = vocab - 1
        if i == 2:
            c = c.sort(descending=True).values
            c[5] = vocab
            c[7] = -1
        rows.append((c, torch.randn(kept, generator=gen) * 2 + 6))
    all_forms(gpu, student(kept, 3, vocab, dtype), csr(rows), f"{vocab}", serial=vocab // 64 + kept,
              weights=torch.tensor([1.0, -2.0, 0.5]))


def test_a_teacher_that_is_not_finite(gpu):
    """Its row's loss and its kept columns' gradients are NaN in any order."""
    logits = student(3, 2, 500, F32)
    columns = torch.tensor([9, 3, 400, 3])
    values = torch.tensor([1.0, float("nan"), 2.0, 0.5])
    data, indices, indptr = csr([(columns, values), (columns, torch.zeros(4))])
    A = gpu.CSRArray(data.cuda(), indices.cuda(), indptr.cuda(), shape=(2, 500))
    losses, grad = gpu.distill_value_and_grad(logits, A)
    assert torch.isnan(losses[0]) and torch.isfinite(losses[1])
    assert torch.isnan(grad[0, columns]).all() and torch.isfinite(grad[1]).all()


def test_repeated_columns_repeat(gpu):
    """The same inputs give the same bits, whatever order sums are made in."""
    gen = torch.Generator().manual_seed(4)
    rows = [(torch.randint(0, 600, (5000,), generator=gen), torch.randn(5000, generator=gen))
            for _ in range(40)]
    A = gpu.CSRArray(*(t.cuda() for t in csr(rows)), shape=(40, 700))
    logits = student(4, 40, 700, F32)
    first = gpu.distill_value_and_grad(logits, A)
    for _ in range(4):
        again = gpu.distill_value_and_grad(logits, A)
        assert all(torch.equal(a, b) for a, b in zip(again, first))
