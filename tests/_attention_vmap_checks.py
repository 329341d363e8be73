"""Window attention of mapped operands, on either device."""

from __future__ import annotations

import torch

from _attention_checks import operands


def mapped_operands(ms, device, dtype=torch.float32):
    """vmap of outputs and gradients equals a loop, whichever operands are
    mapped."""
    q, k, v, g = (t.unflatten(0, (3, 2)) for t in operands(1, 6, 13, 13, 4, 2, 16, dtype, device))
    lengths = torch.tensor([[13, 4], [0, 9], [13, 13]], device=device)
    vmap, grad = torch.func.vmap, torch.func.grad

    def attend(q, k, v, n=None):
        return ms.window_attention(q, k, v, window=5, sinks=1, lengths=n)

    def weighted(q, k, v, g, n):
        return (attend(q, k, v, n).float() * g).sum()

    every = grad(weighted, argnums=(0, 1, 2))
    want = tuple(map(torch.stack, zip(*(every(q[i], k[i], v[i], g[i], lengths[i]) for i in range(3)))))
    for got in (vmap(every)(q, k, v, g, lengths),
                grad(lambda *a: (vmap(attend)(*a, lengths).float() * g).sum(), argnums=(0, 1, 2))(q, k, v)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    mixed = vmap(every, in_dims=(None, 0, None, 1, None))(q[0], k, v[0], g.movedim(0, 1), lengths[0])
    want = tuple(map(torch.stack, zip(*(every(q[0], k[i], v[0], g[i], lengths[0]) for i in range(3)))))
    assert all(torch.equal(a, b) for a, b in zip(mixed, want))
    # one row of the Jacobian for each output value
    rows = torch.func.jacrev(lambda q: attend(q, k[0], v[0])[:, -1, 1].float().sum(0))(q[0])
    for d in range(16):
        upstream = torch.zeros_like(q[0])
        upstream[:, -1, 1, d] = 1
        leaf = q[0].clone().requires_grad_()
        assert torch.equal(rows[d], torch.autograd.grad(attend(leaf, k[0], v[0]), leaf, upstream)[0])


def no_tokens(ms, device):
    f = torch.func.vmap(lambda q, k: ms.window_attention(q, k, k, window=2))
    for shape_q, shape_k in (((3, 2, 0, 4, 8), (3, 2, 5, 2, 8)), ((3, 0, 5, 4, 8), (3, 0, 5, 2, 8)),
                             ((3, 2, 5, 4, 8), (3, 2, 0, 2, 8))):
        q = torch.ones(shape_q, device=device)
        assert f(q, torch.ones(shape_k, device=device)).shape == q.shape
