"""Distillation's kernels against the definition in 64 bits."""

from __future__ import annotations

import pytest
import torch

from _distill_checks import all_forms, teacher_rows

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def student(seed, rows, vocab, dtype, spread=2.5):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen) * spread).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 255, 1000, 4097, 20_011])
def test_vocabularies(gpu, dtype, vocab):
    rows = 5
    buffers = teacher_rows(vocab, rows, vocab, [min(vocab, 9), 0, 1], F32, torch.int32)
    weights = torch.tensor([0.5, 1.0, -2.0, 0.0, 3.0])
    all_forms(gpu, student(vocab, rows, vocab, dtype), buffers, f"{vocab}", temperature=2.0,
              weights=weights, serial=vocab // 64 + 2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_large_vocabularies(gpu, dtype):
    for vocab in (50_001, 131_072, 200_003):
        buffers = teacher_rows(1, 3, vocab, [64, 300], BF16, torch.int64, ordered=False)
        all_forms(gpu, student(1, 3, vocab, dtype), buffers, f"{vocab}", serial=vocab // 64)


@pytest.mark.parametrize("teacher", [F32, F16, BF16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_kept_counts(gpu, teacher, index):
    """From none to every column, in any order."""
    buffers = teacher_rows(2, 6, 1500, [0, 1, 255, 256, 1025, 1500], teacher, index, ordered=False)
    all_forms(gpu, student(2, 6, 1500, BF16), buffers, "kept", temperature=0.5, serial=200)


def test_many_rows(gpu):
    buffers = teacher_rows(3, 4000, 33, [3, 0, 7], F32, torch.int32)
    all_forms(gpu, student(3, 4000, 33, F32), buffers, "rows", serial=33)


def test_views(gpu):
    z = student(4, 12, 777, BF16)
    rows = teacher_rows(4, 6, 770, [8], F32, torch.int32)
    all_forms(gpu, z[::2, 5:775], rows, "rows and columns apart", serial=64)
    all_forms(gpu, z.t().contiguous().t()[:6, :770], rows, "columns apart", serial=64)
    all_forms(gpu, z.reshape(2, 6, 777)[:1, :, :770], rows, "rank 3", serial=64)
    all_forms(gpu, z[:1, :770].expand(6, 770), rows, "one row for all", serial=64)


def test_rows_without_a_target(gpu):
    logits = torch.full((4, 600), float("nan"), device="cuda")
    logits[3] = torch.linspace(-1, 1, 600, device="cuda")
    data = torch.tensor([float("-inf"), float("-inf"), 1.0, 2.0, 1.0, float("-inf")])
    buffers = (data, torch.tensor([1, 2, -1, 600, 3, 5]), torch.tensor([0, 0, 2, 4, 6]))
    for dtype in (F32, BF16):
        losses, grad = all_forms(gpu, logits.to(dtype), buffers, "empty", serial=16)
        assert losses[:3].abs().max() == 0 and grad[:3].abs().max() == 0


def test_rows_of_weight_zero(gpu):
    """Masked by weight: gradient zero whatever the logits are."""
    logits = student(5, 3, 900, BF16)
    buffers = teacher_rows(5, 3, 900, [4], F32, torch.int32)
    weights = torch.tensor([1.0, 0.0, 2.0])
    _, want = all_forms(gpu, logits, buffers, "weight zero", weights=weights, serial=16)
    logits[1] = float("inf")
    A = gpu.CSRArray(*(t.cuda() for t in buffers), shape=(3, 900))
    _, grad = gpu.distill_value_and_grad(logits, A, weights)
    assert torch.equal(grad, want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_columns_stored_twice(gpu, dtype):
    logits = student(6, 2, 500, dtype)
    buffers = (torch.tensor([1.0, 0.5, 2.0, 0.0, 0.0]), torch.tensor([3, 1, 3, 2, 2]),
               torch.tensor([0, 3, 5]))
    all_forms(gpu, logits, buffers, "twice", serial=16)


def test_impossible_columns(gpu):
    for dtype in (F32, F16, BF16):
        logits = student(7, 2, 300, dtype)
        logits[:, 2] = float("-inf")
        logits[:, 100:250] = torch.finfo(dtype).min
        buffers = (torch.tensor([1.0, 2.0, 1.0, float("-inf")]), torch.tensor([0, 2, 1, 2]),
                   torch.tensor([0, 2, 4]))
        A = gpu.CSRArray(*(t.cuda() for t in buffers), shape=(2, 300))
        losses, grad = gpu.distill_value_and_grad(logits, A)
        assert torch.isinf(losses[0]) and torch.isfinite(losses[1]) and torch.isfinite(grad).all()
        assert grad[:, 100:250].abs().max() == 0 and grad[1, 2] == 0


def test_wide_logits(gpu):
    """Logits in the thousands of either sign."""
    buffers = teacher_rows(8, 4, 3001, [16], F32, torch.int32)
    for dtype in (F32, BF16):
        all_forms(gpu, student(8, 4, 3001, dtype, spread=800.0), buffers, "wide", serial=100)


def test_rows_repeat(gpu):
    """The same inputs give the same bits."""
    logits = student(9, 64, 10_007, BF16)
    A = gpu.CSRArray(*(t.cuda() for t in teacher_rows(9, 64, 10_007, [50], F32, torch.int32)),
                     shape=(64, 10_007))
    first = gpu.distill_value_and_grad(logits, A)
    for _ in range(3):
        again = gpu.distill_value_and_grad(logits, A)
        assert all(torch.equal(a, b) for a, b in zip(again, first))


def test_another_stream(gpu):
    logits = student(10, 8, 5000, BF16)
    A = gpu.CSRArray(*(t.cuda() for t in teacher_rows(10, 8, 5000, [50], F32, torch.int32)),
                     shape=(8, 5000))
    want = gpu.distill_value_and_grad(logits, A)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gpu.distill_value_and_grad(logits, A)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_in_a_graph(gpu):
    """Losses and gradient captured once; every replay against the eager call."""
    z = student(9, 70, 5000, BF16)
    data, indices, indptr = teacher_rows(9, 70, 5000, [20, 0, 3], F32, torch.int32)
    teacher = gpu.csr_array((data.cuda(), indices.cuda(), indptr.cuda()), (70, 5000))
    gpu.distill_value_and_grad(z, teacher)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gpu.distill_value_and_grad(z, teacher)
    for i in range(3):
        z.copy_(student(30 + i, 70, 5000, BF16))
        want = gpu.distill_value_and_grad(z, teacher)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
