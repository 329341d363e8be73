"""Rotary positions on the GPU."""

from __future__ import annotations

import pytest
import torch

from _paged_checks import normal, rotation_case
from _paged_reference import turned, within

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated", [(64, 64), (128, 128), (80, 48), (96, 32), (256, 256),
                                         (2, 2), (33, 30), (128, 62), (100, 100), (64, 8)])
def test_values_and_gradient(gpu, dtype, interleaved, dim, rotated):
    rotation_case(gpu, "cuda", dtype, dim=dim, rotated=rotated, interleaved=interleaved, tokens=7,
                  heads=5)


@pytest.mark.parametrize("where", ["none", "starts", "positions", "one row of positions"])
@pytest.mark.parametrize("layout", ["plain", "packed", "heads first", "odd"])
@pytest.mark.parametrize("dtype", TYPES)
def test_positions_and_layouts(gpu, where, layout, dtype):
    for index in (torch.int32, torch.int64):
        rotation_case(gpu, "cuda", dtype, where=where, index=index, layout=layout, dim=64)


@pytest.mark.parametrize("batch,tokens,heads", [(1, 1, 1), (1, 1, 65), (3, 1, 40), (2, 257, 9),
                                                (1, 1030, 3), (700, 1, 2), (5, 33, 130)])
def test_shapes(gpu, batch, tokens, heads):
    rotation_case(gpu, "cuda", torch.bfloat16, batch=batch, tokens=tokens, heads=heads, dim=64)
    rotation_case(gpu, "cuda", torch.float32, batch=batch, tokens=tokens, heads=heads, dim=16,
                  interleaved=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", [
    {"scaling": "linear", "factor": 4.0}, {"scaling": "ntk", "factor": 4.0},
    {"scaling": "yarn", "factor": 8.0, "trained": 128}, {"magnitude": -0.5},
    {"frequencies": [float(i) for i in range(16)]},
])
def test_far_positions(gpu, dtype, how):
    rotation_case(gpu, "cuda", dtype, far=1_500_000, **how)


def test_all_quarters_of_a_turn(gpu):
    """Angles at and around each eighth of a turn, both directions."""
    r = gpu.Rotary(2, frequencies=[1.0])
    eighths = torch.arange(-64, 65, dtype=torch.float64) * torch.pi / 4
    f = (eighths[:, None] + torch.tensor([-1e-4, -1e-9, 0, 1e-9, 1e-4])).flatten()
    wide = gpu.Rotary(256, frequencies=f[:128])
    x = normal(torch.Generator().manual_seed(1), torch.float32, "cuda", 1, 3, 2, 256)
    for first in range(0, 512, 128):
        wide = gpu.Rotary(256, frequencies=f[first:first + 128])
        within(gpu.rotary(x, wide), turned(x, torch.arange(3)[None], wide.frequencies, 1.0, False),
               f"angles from {first}")
    assert torch.equal(gpu.rotary(x, r)[..., 2:], x[..., 2:])


def test_copied_values_keep_their_bits(gpu):
    x = torch.randint(-2**15, 2**15, (2, 3, 4, 64), dtype=torch.int16, device="cuda").view(torch.bfloat16)
    out = gpu.rotary(x, gpu.Rotary(16))
    assert torch.equal(out[..., 16:].view(torch.int16), x[..., 16:].view(torch.int16))


def test_transforms(gpu):
    r = gpu.Rotary(8, interleaved=True)
    gen = torch.Generator().manual_seed(5)
    x = normal(gen, torch.float32, "cuda", 3, 2, 4, 2, 8)
    starts = torch.tensor([[1, 2], [3, 4], [5, 6]], device="cuda")
    one = lambda x, s: gpu.rotary(x, r, starts=s)  # noqa: E731
    assert torch.equal(torch.func.vmap(one)(x, starts), torch.stack([one(a, s) for a, s in zip(x, starts)]))
    _, tangent = torch.func.jvp(lambda x: one(x, starts[0]), (x[0],), (x[1],))
    assert torch.equal(tangent, one(x[1], starts[0]))


def test_captured_and_replayed(gpu):
    r = gpu.Rotary(64)
    x = normal(torch.Generator().manual_seed(2), torch.bfloat16, "cuda", 2, 5, 3, 64).requires_grad_()
    up = torch.ones_like(x)
    starts = torch.tensor([0, 3], device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        out = gpu.rotary(x, r, starts=starts)
        torch.autograd.grad(out, x, up)
        del out
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu.rotary(x, r, starts=starts)
        grad, = torch.autograd.grad(out, x, up)
    for shift in (1, 5, 90):
        starts.add_(shift)
        with torch.no_grad():
            x.mul_(-1)
        graph.replay()
        torch.cuda.synchronize()
        y = x.detach().clone().requires_grad_()
        want = gpu.rotary(y, r, starts=starts)
        assert torch.equal(out, want)
        assert torch.equal(grad, torch.autograd.grad(want, y, up)[0])


def test_on_another_stream(gpu):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        r = gpu.Rotary(64)
        x = normal(torch.Generator().manual_seed(2), torch.float32, "cuda", 2, 5, 3, 64)
        out = gpu.rotary(x, r)
    stream.synchronize()
    within(out, turned(x, torch.arange(5).expand(2, -1), r.frequencies, 1.0, False), "stream")


def test_host_operands_move(gpu):
    r = gpu.Rotary(8)
    x = torch.randn(1, 3, 2, 8)
    out = gpu.rotary(x, r, starts=torch.tensor([4]))
    assert out.is_cuda
    within(out, turned(x, 4 + torch.arange(3)[None], r.frequencies, 1.0, False), "moved")


def test_large(gpu):
    """More values than 32 bits count, in places picked out."""
    r = gpu.Rotary(128)
    x = torch.empty(1, 140_001, 120, 128, dtype=torch.bfloat16, device="cuda").normal_()
    assert x.numel() > 2**31
    out = gpu.rotary(x, r, starts=torch.tensor([5], device="cuda"))
    for t in (0, 70_000, 139_810, 140_000):
        within(out[:, t:t + 1], turned(x[:, t:t + 1], torch.tensor([[t + 5]]), r.frequencies, 1.0,
                                       False), f"token {t}")
