"""Calls without a derivative say so under torch.func transforms and in
forward mode, where a tangent would be lost."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd


def teacher(ms):
    return ms.csr_array((torch.ones(3), torch.tensor([0, 1, 2]), torch.tensor([0, 1, 2, 3])),
                        shape=(3, 5))


def test_value_and_grad(cpu):
    A, z = teacher(cpu), torch.randn(3, 5, generator=torch.Generator().manual_seed(1))
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda x: cpu.distill_value_and_grad(x, A)[0], (z,), (z,))
    with pytest.raises(NotImplementedError, match="distill_value_and_grad"):
        torch.func.grad(lambda x: cpu.distill_value_and_grad(x, A)[0].sum())(z)
    with pytest.raises(NotImplementedError, match="distill_value_and_grad"):
        torch.func.grad(lambda w: cpu.distill_value_and_grad(z, A, w)[1].sum())(torch.ones(3))
    with fwd.dual_level():
        dual = fwd.make_dual(z, torch.ones_like(z))
        with pytest.raises(NotImplementedError):
            cpu.distill_value_and_grad(dual, A)
        plain = cpu.distill_value_and_grad(z, A)  # operands without a tangent
    assert all(torch.equal(a, b) for a, b in zip(plain, cpu.distill_value_and_grad(z, A)))
    # of no concern to a transform of something else
    got = torch.func.grad(lambda x: (x * cpu.distill_value_and_grad(z, A)[0]).sum())(torch.ones(3))
    assert torch.equal(got, plain[0])


def test_steps_and_stores(cpu):
    q, k = torch.randn(3, 2, 4, 8), torch.randn(3, 2, 2, 8)
    ck, cv = torch.zeros(3, 2, 6, 2, 8), torch.zeros(3, 2, 6, 2, 8)
    n = torch.zeros(3, 2, dtype=torch.int32)

    def step(q, k, ck, cv, n):
        return cpu.window_attention_step(q, k, k, ck, cv, n, window=4)

    with pytest.raises(NotImplementedError, match="window_attention_step"):
        torch.func.vmap(step)(q, k, ck, cv, n)
    with pytest.raises(NotImplementedError, match="window_attention_step"):
        torch.func.grad(lambda q: step(q, k[0], ck[0], cv[0], n[0]).sum())(q[0])
    with pytest.raises(NotImplementedError, match="window_cache_store"):
        torch.func.vmap(lambda k, ck, cv: cpu.window_cache_store(k[:, None], k[:, None], ck, cv))(k, ck, cv)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="window_attention_step"):
            step(fwd.make_dual(q[0], q[0]), k[0], ck[0], cv[0], n[0])
        with pytest.raises(NotImplementedError, match="window_cache_store"):
            dual = fwd.make_dual(k[0, :, None], k[0, :, None])
            cpu.window_cache_store(dual, dual, ck[0], cv[0])
        assert ck.abs().max() == 0 and cv.abs().max() == 0
        step(q[0], k[0], ck[0], cv[0], n[0])
    assert torch.equal(ck[0, :, 0], k[0])
