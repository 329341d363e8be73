"""Rotary positions on the host: values, derivatives, transforms, refusals."""

from __future__ import annotations

import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

from _paged_checks import rotation_case
from _paged_reference import turned, within

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated", [(32, 32), (2, 2), (80, 48), (7, 4), (256, 256), (33, 30)])
def test_values_and_gradient(cpu, dtype, interleaved, dim, rotated):
    rotation_case(cpu, "cpu", dtype, dim=dim, rotated=rotated, interleaved=interleaved)


@pytest.mark.parametrize("where", ["none", "starts", "positions", "one row of positions"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("layout", ["plain", "packed", "heads first", "odd"])
def test_positions_and_layouts(cpu, where, index, layout):
    rotation_case(cpu, "cpu", torch.float32, where=where, index=index, layout=layout)


@pytest.mark.parametrize("how", [
    {"scaling": "linear", "factor": 4.0}, {"scaling": "ntk", "factor": 4.0},
    {"scaling": "yarn", "factor": 8.0, "trained": 128}, {"base": 500_000.0},
    {"magnitude": -0.5}, {"frequencies": [float(i) for i in range(16)]},
])
@pytest.mark.parametrize("far", [0, 1_500_000])
def test_frequencies(cpu, how, far):
    rotation_case(cpu, "cpu", torch.float32, far=far, **how)


def test_scalings_by_their_formulas(ms):
    n, s = 16, 8.0
    f = [10_000.0 ** (-2 * i / n) for i in range(n // 2)]
    torch.testing.assert_close(ms.Rotary(n).frequencies, torch.tensor(f, dtype=torch.float64))
    linear = ms.Rotary(n, scaling="linear", factor=s).frequencies
    torch.testing.assert_close(linear, torch.tensor(f, dtype=torch.float64) / s)
    ntk = ms.Rotary(n, scaling="ntk", factor=s).frequencies
    assert ntk[0] == 1 and math.isclose(float(ntk[-1]), f[-1] / s, rel_tol=1e-12)
    yarn = ms.Rotary(n, scaling="yarn", factor=s, trained=1000)
    assert math.isclose(yarn.magnitude, 0.1 * math.log(s) + 1)
    for got, one in zip(yarn.frequencies.tolist(), f):
        turns = 1000 * one / (2 * math.pi)
        kept = min(max((turns - 1) / 31, 0.0), 1.0)
        assert math.isclose(got, one * kept + one / s * (1 - kept), rel_tol=1e-12)
    assert yarn.frequencies[0] == 1 and math.isclose(float(yarn.frequencies[-1]), f[-1] / s)


def test_nothing_to_rotate(cpu):
    r = cpu.Rotary(4)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        x = torch.zeros(shape, requires_grad=True)
        out = cpu.rotary(x, r)
        assert out.shape == x.shape
        assert torch.autograd.grad(out.sum(), x)[0].shape == x.shape


def test_gradient_against_differences(cpu):
    """The operator is linear: a difference quotient of any step is the derivative."""
    gen = torch.Generator().manual_seed(2)
    r = cpu.Rotary(6, interleaved=True, magnitude=1.5)
    x = torch.randn(2, 3, 2, 8, generator=gen, requires_grad=True)
    d, up = (torch.randn(x.shape, generator=gen) for _ in range(2))
    grad, = torch.autograd.grad(cpu.rotary(x, r, starts=torch.tensor([3, 9])), x, up)
    with torch.no_grad():
        plus, minus = (cpu.rotary(x + s * d, r, starts=torch.tensor([3, 9])) for s in (0.5, -0.5))
    quotient = ((plus.double() - minus.double()) * up.double()).sum()
    # each value is off by 6 x 2^-24 m (|a| + |b|), the operands by their own rounding
    size = ((x.abs() + d.abs()).sum() * up.abs().max() * 1.5).double()
    off = quotient - (grad.double() * d.double()).sum()
    assert abs(float(off.detach())) <= 4 * 8 * 2**-24 * float(size.detach())


def test_second_derivatives(cpu):
    r = cpu.Rotary(8)
    x = torch.randn(1, 4, 2, 8, generator=torch.Generator().manual_seed(3), requires_grad=True)
    up = torch.ones_like(x, requires_grad=True)
    first, = torch.autograd.grad(cpu.rotary(x, r), x, up, create_graph=True)
    w = torch.randn(x.shape, generator=torch.Generator().manual_seed(4))
    second, = torch.autograd.grad((first * w).sum(), up)
    within(second, turned(w, torch.arange(4)[None], r.frequencies, 1.0, False), "second")


def test_transforms(cpu):
    r = cpu.Rotary(8, interleaved=True)
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(3, 2, 4, 2, 8, generator=gen)
    starts = torch.tensor([[1, 2], [3, 4], [5, 6]])
    one = lambda x, s: cpu.rotary(x, r, starts=s)  # noqa: E731
    want = torch.stack([one(a, s) for a, s in zip(x, starts)])
    assert torch.equal(torch.func.vmap(one)(x, starts), want)
    assert torch.equal(torch.func.vmap(one, (1, None), 1)(x.transpose(0, 1), starts[0]),
                       torch.stack([one(a, starts[0]) for a in x], 1))
    value, tangent = torch.func.jvp(lambda x: one(x, starts[0]), (x[0],), (x[1],))
    assert torch.equal(value, want[0]) and torch.equal(tangent, one(x[1], starts[0]))
    loss = lambda x: (one(x, starts[0]) * x[..., :1]).sum()  # noqa: E731
    a = x[0].clone().requires_grad_()
    assert torch.equal(torch.func.grad(loss)(x[0]), torch.autograd.grad(loss(a), a)[0])
    each = torch.func.vmap(torch.func.grad(lambda x, s: one(x, s).square().sum()))(x, starts)
    # a rotation keeps the square: its gradient is 2 x
    torch.testing.assert_close(each, 2 * x, rtol=0, atol=8 * 6 * 2**-24 * float(x.abs().max()))
    positions = torch.arange(4).expand(2, -1)
    assert torch.equal(torch.func.vmap(lambda x: cpu.rotary(x, r, positions=positions))(x),
                       torch.stack([cpu.rotary(a, r) for a in x]))
    with fwd.dual_level():
        out = fwd.unpack_dual(cpu.rotary(fwd.make_dual(x[0], x[1]), r))
        assert torch.equal(out.tangent, cpu.rotary(x[1], r))


def test_views_of_negated_and_expanded_operands(cpu):
    r = cpu.Rotary(8)
    x = torch.randn(2, 3, 2, 8, generator=torch.Generator().manual_seed(6))
    negative = torch._neg_view(x)
    assert torch.equal(cpu.rotary(negative, r), cpu.rotary(-x, r))
    wide = x[:1].expand(4, -1, -1, -1)
    assert torch.equal(cpu.rotary(wide, r), cpu.rotary(wide.contiguous(), r))
    y = x[:1].clone().requires_grad_()
    out = cpu.rotary(y.expand(4, -1, -1, -1), r, starts=torch.arange(4))
    grad, = torch.autograd.grad(out.sum(), y)
    want = sum(turned(torch.ones_like(y), torch.arange(3)[None] + b, r.frequencies, 1.0, False,
                      inverse=True)[0] for b in range(4))
    torch.testing.assert_close(grad.double(), want, rtol=0, atol=4 * 16 * 2**-24)


@pytest.mark.parametrize("bad,error,text", [
    (dict(dim=3), ValueError, "even"), (dict(dim=0), ValueError, "even"),
    (dict(dim=258), ValueError, "256"), (dict(dim=8, base=0.0), ValueError, "base"),
    (dict(dim=8, factor=-1.0), ValueError, "factor"),
    (dict(dim=8, scaling="cubic"), ValueError, "scaling"),
    (dict(dim=8, scaling="yarn", factor=2.0), ValueError, "trained"),
    (dict(dim=8, scaling="yarn", factor=2.0, trained=9, ramp=(2, 1)), ValueError, "ramp"),
    (dict(dim=8, frequencies=[1.0]), ValueError, "shape"),
    (dict(dim=4, frequencies=[1.0, math.inf]), ValueError, "finite"),
    (dict(dim=4, frequencies=[1.0, 2.0], scaling="ntk"), ValueError, "not both"),
    (dict(dim=4, magnitude=math.nan), ValueError, "magnitude"),
    (dict(dim=4, magnitude=1e39), ValueError, "magnitude"),
])
def test_refused_rotations(ms, bad, error, text):
    with pytest.raises(error, match=text):
        ms.Rotary(**bad)


def test_refusals(cpu):
    r, x = cpu.Rotary(8), torch.zeros(2, 3, 2, 8)
    with pytest.raises(TypeError, match="Rotary"):
        cpu.rotary(x, 8)
    with pytest.raises(TypeError, match="float64"):
        cpu.rotary(x.double(), r)
    with pytest.raises(ValueError, match="shape"):
        cpu.rotary(x[0], r)
    with pytest.raises(ValueError, match="rotates 8"):
        cpu.rotary(x[..., :6], r)
    with pytest.raises(ValueError, match="256"):
        cpu.rotary(torch.zeros(1, 1, 1, 300), r)
    with pytest.raises(ValueError, match="not both"):
        cpu.rotary(x, r, starts=torch.zeros(2, dtype=torch.int32),
                   positions=torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="starts"):
        cpu.rotary(x, r, starts=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions"):
        cpu.rotary(x, r, positions=torch.zeros(3, dtype=torch.int32))
    with pytest.raises((TypeError, ValueError), match="int32 or int64"):
        cpu.rotary(x, r, starts=torch.zeros(2))
