"""Operands whose rows do not start at sixteen bytes run the same kernels as
those that do: the same bits come out."""

from __future__ import annotations

import pytest
import torch

from _attention_checks import operands

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def odd(t):
    """The same values, every row one value past a sixteen-byte address."""
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 16, dtype=t.dtype, device=t.device)
    wide[..., 1:1 + t.shape[-1]] = t
    return wide[..., 1:1 + t.shape[-1]]


def outputs(ms, q, k, v, g):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ms.window_attention(*leaves, window=40, sinks=3)
    with torch.no_grad():
        assert torch.equal(ms.window_attention(q, k, v, window=40, sinks=3), out)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("which", [0, 1, 2, 3, None])
def test_one_operand_or_all(gpu, dtype, which):
    args = operands(1, 2, 150, 150, 4, 2, 64, dtype, "cuda")
    want = outputs(gpu, *args)
    got = outputs(gpu, *(odd(t) if which in (i, None) else t for i, t in enumerate(args)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_of_single_places(gpu, dtype):
    """One sequence, one key head: their strides say nothing."""
    q, k, v, g = operands(2, 1, 150, 150, 4, 1, 64, dtype, "cuda")
    want = outputs(gpu, q, k, v, g)

    def loose(t):
        return t.as_strided(t.shape, (t.numel() + 1, t.stride(1), t.stride(2) if t.shape[2] > 1 else 3, 1))

    got = outputs(gpu, *map(loose, (q, k, v, g)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_upstream_of_a_concatenation(gpu):
    """The backward pass of a concatenation hands on slices of its gradient."""
    q, k, v, g = operands(3, 2, 150, 150, 4, 2, 64, BF16, "cuda")
    extra = torch.randn(2, 150, 4, 1, device="cuda").to(BF16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = gpu.window_attention(*leaves, window=40, sinks=3)
    got = torch.autograd.grad(torch.cat([extra, out], dim=3), leaves, torch.cat([extra, g], dim=3))
    assert all(torch.equal(a, b) for a, b in zip(got, outputs(gpu, q, k, v, g)[1:]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 256])
def test_steps(gpu, dtype, dim):
    q, k, v = (torch.randn(3, n, dim).to(dtype).cuda() for n in (8, 2, 2))
    caches = [torch.randn(3, 304, 2, dim).to(dtype).cuda() for _ in range(2)]
    n = torch.tensor([900, 20, 0], device="cuda")
    mirror = [c.clone() for c in caches]
    want = gpu.window_attention_step(q, k, v, *mirror, n, window=300, sinks=4)
    got = gpu.window_attention_step(odd(q), odd(k), odd(v), *caches, n, window=300, sinks=4)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(caches, mirror))


@pytest.mark.parametrize("dtype,dim", [(F16, 100), (BF16, 121), (BF16, 33), (F16, 6), (F32, 30), (F32, 127), (F32, 3)])
def test_heads_between_sixteen_bytes(gpu, dtype, dim):
    """As the same heads with zeros beyond them."""
    q, k, v, g = operands(dim, 2, 150, 150, 4, 2, dim, dtype, "cuda")
    per = 16 // q.element_size()

    def pad(t):
        return torch.nn.functional.pad(t, (0, -dim % per))

    pattern = {"window": 40, "sinks": 3, "lengths": torch.tensor([150, 70], device="cuda")}
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = gpu.window_attention(*leaves, **pattern)
    got = (out.detach(), *torch.autograd.grad(out, leaves, g))
    leaves = [pad(t).requires_grad_() for t in (q, k, v)]
    out = gpu.window_attention(*leaves, scale=dim**-0.5, **pattern)
    want = (out.detach(), *torch.autograd.grad(out, leaves, pad(g)))
    for a, b in zip(got, want):
        assert a.shape[-1] == dim and a.is_contiguous() and torch.equal(a, b[..., :dim])
    with torch.no_grad():
        assert torch.equal(gpu.window_attention(q, k, v, **pattern), got[0])
