"""Distillation of mapped students, on either device."""

from __future__ import annotations

import torch

from _distill_checks import teacher_rows


def mapped_students(ms, device, dtype=torch.float32):
    """vmap over students, weights and upstream gradients equals a loop (rows of
    40 start at sixteen bytes wherever they lie, so that sums are made in one order)."""
    gen = torch.Generator().manual_seed(1)
    z = (torch.randn(4, 6, 40, generator=gen) * 2).to(dtype).to(device)
    w = torch.rand(4, 6, generator=gen).to(device)
    data, indices, indptr = (t.to(device) for t in teacher_rows(2, 6, 40, [5, 0, 40, 1],
                                                                torch.float32, torch.int32))
    A = ms.CSRArray(data=data, indices=indices, indptr=indptr, shape=(6, 40))
    vmap, grad = torch.func.vmap, torch.func.grad

    def loss(x):
        return ms.distill_loss(x, A, temperature=1.5)

    def both(x, v):
        return ms.distill_value_and_grad(x, A, v, temperature=1.5)

    def weighted(x, v):
        return (loss(x) * v).sum()

    def stacked(f, *args):
        got = [f(*(a[i] for a in args)) for i in range(4)]
        return tuple(map(torch.stack, zip(*got))) if isinstance(got[0], tuple) else torch.stack(got)

    assert torch.equal(vmap(loss)(z), stacked(loss, z))
    last = z.movedim(0, 2).contiguous()
    assert torch.equal(vmap(loss, in_dims=2)(last), stacked(loss, z))
    for got, want in zip(vmap(both)(z, w), stacked(both, z, w)):
        assert torch.equal(got, want)
    for got, want in zip(vmap(both, in_dims=(None, 0))(z[0], w), stacked(lambda v: both(z[0], v), w)):
        assert torch.equal(got, want)
    want = stacked(grad(weighted), z, w)
    assert torch.equal(vmap(grad(weighted))(z, w), want)
    assert torch.equal(vmap(grad(weighted), in_dims=(None, 0))(z[0], w),
                       stacked(lambda v: grad(weighted)(z[0], v), w))
    assert torch.equal(grad(lambda x: (vmap(loss)(x) * w).sum())(z), want)
    # rows of one student do not depend on each other's
    jacobian = torch.func.jacrev(loss)(z[0])
    every = grad(lambda x: loss(x).sum())(z[0])
    assert torch.equal(jacobian.diagonal().movedim(-1, 0), every) and \
        int(jacobian.count_nonzero()) == int(every.count_nonzero())
    nested = z.reshape(2, 2, 6, 40)
    assert torch.equal(vmap(vmap(loss))(nested).reshape(4, 6), stacked(loss, z))
