"""Paged attention where one key takes nearly all of the softmax and its value is
nothing: the output is what the other keys add, however little they weigh.

Scores are exact: queries are one-hot, the first value of the keys is their score, the
scale is one.  With w the weight of a key beside the largest and u the type's unit
roundoff, a weight enters the product with the values off by u w at most, in float16
by 2^-38 where that is more (half of its smallest number beside a largest weight of
2^13 at least), and the result is rounded once (float16: to 2^-25 at least).  The
exponent, at most 24 in three roundings to float32 and made a power of two, is good to
3 x 24 x 2^-24 x 1.45 in all, and sums of n terms in float32 to n 2^-24 of them:

    (2 u + (n + 120) 2^-24) sum_j p_j |v_j| + 2^-25 + 2^-38 sum_j |v_j|
"""

from __future__ import annotations

import pytest
import torch

from _attention_reference import UNIT, check
from _paged_checks import normal, table_for

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def concentrated(ms, dtype, nats, starts, *, tokens=1, heads=4, kv_heads=2, dim=64, size=16, shared=0,
                 width=None, at=0, uniform=True, window=None, sinks=0):
    """Key ``at`` of every sequence has the score ``nats`` and the value zero, the others a
    score of zero (-1 to 0 where not ``uniform``) and values up to 1,024."""
    gen = torch.Generator().manual_seed(int(nats) + len(starts))
    batch = len(starts)
    ends = [s + tokens for s in starts]
    width = width or -(-max(ends) // size)
    total, table = table_for(gen, ends, size, width, shared=shared)
    ck = torch.zeros(total, size, kv_heads, dim)
    cv = normal(gen, F32, "cpu", total, size, kv_heads, dim).abs().clamp(0.25, 4) * 256
    if uniform:
        cv[:] = 1000.0
    else:
        ck[..., 0] = -torch.rand(ck.shape[:-1], generator=gen)
    for b in range(batch):
        page = int(table[b, at // size])
        ck[page, at % size, :, 0], cv[page, at % size] = nats, 0.0
    q = torch.zeros(batch, tokens, heads, dim)
    q[..., 0] = 1.0
    q, ck, cv = (t.to(dtype).cuda() for t in (q, ck, cv))
    out = ms.paged_attention(q, ck, cv, table.int().cuda(), starts=torch.tensor(starts).cuda(), scale=1.0,
                             window=window, sinks=sinks, shared_pages=shared)
    ck, cv = ck.double().cpu(), cv.double().cpu()
    want, tol = (torch.zeros(out.shape, dtype=torch.float64) for _ in range(2))
    most = 2.0**40 if window is None else window
    for b, start in enumerate(starts):
        j = torch.arange(start + tokens)
        k, v = (t[table[b, j // size], j % size] for t in (ck, cv))
        p = start + torch.arange(tokens)[:, None]
        seen = (j <= p) & ((p - j < most) | (j < sinks))
        for h in range(heads):
            s = torch.where(seen, k[:, h // (heads // kv_heads), 0], -torch.inf)
            of = v[:, h // (heads // kv_heads)]
            want[b, :, h] = torch.softmax(s, 1) @ of
            tol[b, :, h] = 2.0**-25 + (2.0**-38 * (seen.double() @ of) if dtype == F16 else 0)
    n = max(ends)
    check(out, (want, tol + (2 * UNIT[dtype] + (n + 120) * 2.0**-24) * want),
          f"{dtype} {nats} nats, {starts[:4]} tokens {tokens} of {dim}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nats", [8, 12, 14, 16, 18, 20, 24])
@pytest.mark.parametrize("uniform", [True, False])
def test_single_tokens(gpu, dtype, nats, uniform):
    concentrated(gpu, dtype, nats, [499], uniform=uniform)  # a workgroup a sequence
    concentrated(gpu, dtype, nats, [4100, 90], uniform=uniform, dim=128, width=600)  # cut


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nats", [8, 12, 14, 16, 18, 20, 24])
@pytest.mark.parametrize("dim", [32, 64, 128, 256])
def test_chunks(gpu, dtype, nats, dim):
    concentrated(gpu, dtype, nats, [430], tokens=70, dim=dim)
    concentrated(gpu, dtype, nats, [300, 0], tokens=130, dim=dim, uniform=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nats", [14, 17, 20])
def test_long_chunk(gpu, dtype, nats):
    concentrated(gpu, dtype, nats, [6000], tokens=300, heads=2, kv_heads=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nats", [14, 17, 20, 24])
@pytest.mark.parametrize("tokens", [1, 4])
def test_shared_pages(gpu, dtype, nats, tokens):
    starts = [2240 + 7 * b % 90 for b in range(64)]
    concentrated(gpu, dtype, nats, starts, tokens=tokens, shared=140, dim=128)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 70])
@pytest.mark.parametrize("at", [40, 300])
def test_late_keys(gpu, dtype, tokens, at):
    """The largest score comes after others, or not far above them."""
    for nats in (0.25, 0.75, 1.5, 3.0, 5.5, 6.0, 11.0, 18.0):
        concentrated(gpu, dtype, nats, [430], tokens=tokens, at=at, uniform=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 70])
def test_sinks_before_a_window(gpu, dtype, tokens):
    concentrated(gpu, dtype, 18, [2000, 700], tokens=tokens, window=400, sinks=1, dim=128)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 70])
def test_the_largest_values(gpu, dtype, tokens):
    """Sums of unnormalised weights times values near the type's largest stay finite."""
    gen = torch.Generator().manual_seed(1)
    total, table = table_for(gen, [900], 16, 57)
    ck = normal(gen, dtype, "cuda", total, 16, 1, 64)
    cv = torch.full_like(ck, 32768.0 if dtype == F16 else 2.0**100)
    q = normal(gen, dtype, "cuda", 1, tokens, 4, 64)
    out = gpu.paged_attention(q, ck, cv, table.cuda(), starts=torch.tensor([900 - tokens]).cuda())
    assert out.isfinite().all()
    want = cv[0, 0, 0, 0].double()
    assert ((out.double() - want).abs() <= 2 * (UNIT[dtype] + 1020 * 2.0**-24) * want).all()
