"""Window attention on the host path, against its definition in 64 bits; and
the refusals, which come before any device is touched."""

from __future__ import annotations

import ctypes

import pytest
import torch

import _capi
from _attention_checks import forward_and_gradients, operands, prompt_then_steps, step
from _attention_reference import check, reference

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lq,lk,window,sinks", [
    (1, 1, 1, 0), (9, 9, 1, 0), (23, 23, 5, 2), (23, 23, 100, 7), (7, 30, 6, 3), (30, 7, 4, 1),
    (12, 12, 3, 50)])
def test_outputs_and_gradients(cpu, dtype, lq, lk, window, sinks):
    q, k, v, g = operands(1, 2, lq, lk, 4, 2, 12, dtype, "cpu")
    forward_and_gradients(cpu, q, k, v, g, f"{lq} {lk}", window=window, sinks=sinks)


def test_lengths_and_padding(cpu):
    q, k, v, g = operands(2, 4, 17, 17, 6, 3, 8, F32, "cpu")
    lengths = torch.tensor([17, 5, 0, 1], dtype=torch.int64)
    for b, n in enumerate(lengths.tolist()):
        for t in (q, k, v, g):
            t[b, n:] = float("nan")
    got = forward_and_gradients(cpu, q, k, v, g, "padded", window=4, sinks=2, lengths=lengths)
    assert got["out"][1, 5:].abs().max() == 0 and got["dk"][2].abs().max() == 0


def test_views_of_one_projection(cpu):
    packed = torch.randn(2, 11, 8, 6, generator=torch.Generator().manual_seed(3))
    q, k, v = packed.split([4, 2, 2], dim=2)
    forward_and_gradients(cpu, q, k, v, torch.randn(2, 11, 4, 6), "views", window=3, sinks=1)
    q = torch.randn(2, 4, 11, 6).transpose(1, 2)  # head-major
    forward_and_gradients(cpu, q, k, v, torch.randn(2, 4, 11, 6).transpose(1, 2), "head-major",
                          window=3, sinks=1, scale=0.3)


def test_empty_operands(cpu):
    for batch, lq, lk in ((0, 3, 3), (2, 0, 4), (2, 3, 0)):
        q, k, v, g = operands(4, batch, lq, lk, 2, 1, 4, F32, "cpu")
        forward_and_gradients(cpu, q, k, v, g, "empty", window=2)


def test_gradients_against_differences(cpu):
    """Central differences of sum(out * g) in float32: the step's error is
    h^2 of the third derivative, the rounding 2^-24 / h of the sum's terms."""
    q, k, v, g = operands(5, 1, 6, 6, 2, 1, 4, F32, "cpu", spread=0.5)
    got = forward_and_gradients(cpu, q, k, v, g, "", window=3, sinks=1)
    h = 2.0**-6
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        for i in range(t.numel()):
            sums = []
            for sign in (h, -h):
                t.view(-1)[i] += sign
                sums.append(float((cpu.window_attention(q, k, v, window=3, sinks=1).double()
                                   * g.double()).sum()))
                t.view(-1)[i] -= sign
            assert abs((sums[0] - sums[1]) / (2 * h) - float(got[name].view(-1)[i])) < 2e-3, name


def test_vmap_and_functional_grad(cpu):
    q, k, v, g = operands(6, 6, 9, 9, 2, 1, 4, F32, "cpu")
    want = cpu.window_attention(q, k, v, window=4, sinks=1)
    mapped = torch.func.vmap(lambda a, b, c: cpu.window_attention(a, b, c, window=4, sinks=1))
    halves = [t.reshape(3, 2, *t.shape[1:]) for t in (q, k, v)]
    assert torch.equal(mapped(*halves).reshape(want.shape), want)
    grads = torch.func.grad(
        lambda *a: (cpu.window_attention(*a, window=4, sinks=1) * g).sum(), argnums=(0, 1, 2))(q, k, v)
    for name, got in zip(("dq", "dk", "dv"), grads):
        check(got, reference(q, k, v, window=4, sinks=1, grad=g)[name], name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps(cpu, dtype):
    step(cpu, 1, [0, 1, 5, 9, 40, -1], 4, 2, 8, dtype, "cpu", window=6, sinks=2, index=torch.int64)
    step(cpu, 2, [3, 12], 2, 2, 5, dtype, "cpu", window=4, sinks=0, slots=20,
         unseen=float("nan"))


def test_prompt_then_steps(cpu):
    prompt_then_steps(cpu, "cpu", F32, window=7, sinks=3, prompt=[4, 25, 1], more=12)


def test_store_of_a_chunk(cpu):
    """A chunk that starts at a position of its own, longer than the ring."""
    k = torch.arange(1.0, 21.0).reshape(1, 20, 1, 1).expand(2, 20, 1, 1)
    ck = torch.zeros(2, 6, 1, 1)
    cv = torch.zeros(2, 6, 1, 1)
    cpu.window_cache_store(k, -k, ck, cv, sinks=2, starts=torch.tensor([0, 1]),
                           lengths=torch.tensor([20, 3]))
    # ring of 4: position p >= 2 in slot 2 + (p - 2) % 4; positions 16 .. 19 stay
    assert ck[0].flatten().tolist() == [1, 2, 19, 20, 17, 18]
    assert ck[1].flatten().tolist() == [0, 1, 2, 3, 0, 0]
    assert torch.equal(cv, -ck)


def test_refusals(cpu):
    q, k, v, _ = operands(7, 2, 5, 5, 4, 2, 8, F32, "cpu")
    f = cpu.window_attention
    with pytest.raises(ValueError, match="window must be at least 1"):
        f(q, k, v, window=0)
    with pytest.raises(ValueError, match="sinks must be non-negative"):
        f(q, k, v, window=1, sinks=-1)
    with pytest.raises(TypeError):
        f(q, k, v, window=2.5)
    with pytest.raises(TypeError, match="one dtype"):
        f(q, k.half(), v, window=2)
    with pytest.raises(TypeError, match="supports float32"):
        f(q.double(), k.double(), v.double(), window=2)
    with pytest.raises(ValueError, match="multiple"):
        f(q[:, :, :3], k, v, window=2)
    with pytest.raises(ValueError, match="expects q of shape"):
        f(q, k, v[:, :4], window=2)
    with pytest.raises(ValueError, match="batch or head dimension"):
        f(q[:1], k, v, window=2)
    with pytest.raises(ValueError, match="between 1 and 256"):
        f(*(t.repeat(1, 1, 1, 40) for t in (q, k, v)), window=2)
    with pytest.raises(ValueError, match="lengths"):
        f(q, k, v, window=2, lengths=torch.tensor([1, 2, 3]))
    with pytest.raises(ValueError, match="int32 or int64"):
        f(q, k, v, window=2, lengths=torch.tensor([1.0, 2.0]))
    leaf = q.clone().requires_grad_()
    first, = torch.autograd.grad((f(leaf, k, v, window=2) ** 2).sum(), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="second-order"):
        first.sum().backward()


def test_step_refusals(cpu):
    q, k = torch.zeros(2, 4, 8), torch.zeros(2, 2, 8)
    ck, cv = torch.zeros(2, 6, 2, 8), torch.zeros(2, 6, 2, 8)
    n = torch.tensor([0, 1])
    f = cpu.window_attention_step
    f(q, k, k, ck, cv, n, window=4, sinks=2)
    with pytest.raises(ValueError, match="at least sinks"):
        f(q, k, k, ck, cv, n, window=5, sinks=2)
    with pytest.raises(TypeError, match="one dtype"):
        f(q, k, k, ck.half(), cv, n, window=4)
    with pytest.raises(ValueError, match="cache_v"):
        f(q, k, k, ck, cv[:, :5], n, window=4)
    with pytest.raises(ValueError, match="require grad"):
        f(q, k, k, ck.requires_grad_(), cv, n, window=4)
    with pytest.raises(ValueError, match="adjacent"):
        f(q, k, k, torch.zeros(2, 6, 8, 2).transpose(2, 3), cv, n, window=4)
    with pytest.raises(TypeError, match="requires lengths"):
        f(q, k, k, cv, cv.clone(), None, window=4)


def test_c_entry_points_refuse():
    """Status codes, before any HIP call."""
    L = _capi.lib()
    desc = (ctypes.c_char * 512)()
    assert L.msx_window_attention(None, None, None, None, ctypes.c_size_t(0), None) == _capi.EINVAL
    head = ctypes.cast(desc, ctypes.POINTER(ctypes.c_int32))
    head[0] = 3  # complex values
    assert L.msx_window_attention(desc, None, None, None, ctypes.c_size_t(0), None) == _capi.ETYPE
    assert L.msx_window_attention_step(desc, None, None, ctypes.c_size_t(0), None) == _capi.ETYPE
    head[0] = 0
    assert L.msx_window_attention(desc, None, None, None, ctypes.c_size_t(0), None) == _capi.EINVAL  # no heads
    assert "heads" in _capi.last_error()
