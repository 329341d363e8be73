"""A rotation that a device does not have yet while a graph is captured there."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_first_used_in_a_graph(gpu):
    gpu.use_cpu()
    try:
        rotation = gpu.Rotary(64)
    finally:
        gpu.use_gpu()
    x = torch.randn(1, 3, 2, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"), torch.cuda.graph(graph):
        gpu.rotary(x, rotation)
    torch.cuda.synchronize()
    want = gpu.rotary(x, rotation)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = gpu.rotary(x, rotation)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
