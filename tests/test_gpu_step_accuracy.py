"""Accuracy of a single token's attention: memory bounds it, so its output has
the rounding of the result alone."""

from __future__ import annotations

import pytest
import torch

from _attention_reference import UNIT

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,window,sinks", [
    (3, 8, 2, 64, 700, 4), (1, 4, 4, 128, 5000, 0), (5, 20, 1, 200, 90, 2)])
def test_rounded_once(gpu, dtype, batch, heads, kv_heads, dim, window, sinks):
    """Rounding values spread over binades once costs 0.39 to 0.43 u of their
    norm (a uniform error of half a step, 0.58 u at a power of two); one more
    rounding of as many terms would make 0.55 to 0.6.  Allowed is 0.5 u, and
    for the sums in float32 (n + dim + 8) 2^-23 (1 + A), A the largest sum of
    a score's absolute terms, where they are what counts."""
    gen = torch.Generator().manual_seed(dim)
    held = window + sinks

    def normal(*shape):
        return torch.randn(shape, generator=gen).to(dtype).cuda()

    q, k, v = normal(batch, heads, dim), normal(batch, kv_heads, dim), normal(batch, kv_heads, dim)
    ck, cv = normal(batch, held, kv_heads, dim), normal(batch, held, kv_heads, dim)
    n = torch.full((batch,), 3 * held, device="cuda")
    out = gpu.window_attention_step(q, k, v, ck, cv, n, window=window, sinks=sinks)
    key, value = (t.double().cpu().repeat_interleave(heads // kv_heads, 2) for t in (ck, cv))
    terms = key * q.double().cpu()[:, None] * dim**-0.5
    p = torch.softmax(terms.sum(3), 1)
    want = (p[..., None] * value).sum(1)
    most = 0.5 * UNIT[dtype]
    if dtype == F32:
        most = (held + dim + 8) * 2.0**-23 * (1 + float(terms.abs().sum(3).max()))
    error = float((out.double().cpu() - want).norm() / want.norm())
    assert error <= most, f"off by {error:.3g}, tolerated {most:.3g}"
