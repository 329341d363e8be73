"""Rotary positions and attention over paged caches by their definitions, in 64
bits on the CPU, with what rounding may take from a result.

Rotary.  With u the unit roundoff of the storage type (2^-24, 2^-11, 2^-8), m
the magnitude and (a, b) a pair: the angle is off by 2 pi p f 2^-53 / (2 pi)
times some, 2^-30 at the positions tested.  For 16-bit values its cosine and sine
are float32's of an angle of at most pi / 4 in float32 (three roundings of at
most 2^-24 pi / 4, the series' own 2 x 2^-24): off by 2^-22 m; for float32 values
they are 64-bit, rounded: 2^-24 m.  Two products, a sum and the magnitude add 4 x
2^-24 m (|a| + |b|), and the result is rounded once.  So

    16-bit:  u |want| + 2^-21 m (|a| + |b|)      float32:  6 x 2^-24 m (|a| + |b|)

and half a step of float16's subnormals, 2^-25.

Attention: as derived in _attention_reference.py, with n the most keys that a
query sees: (3 u + (n + dim + 8) 2^-23 (1 + A)) sum_j p_j |v_j|.
"""

from __future__ import annotations

import math

import torch

from _attention_reference import UNIT


def turned(x, position, frequencies, magnitude, interleaved, inverse=False):
    """(value, tolerance) of ``x`` (..., heads, dim) at ``position`` (...)."""
    dtype = x.dtype
    x = x.detach().cpu().double()
    f = torch.as_tensor(frequencies, dtype=torch.float64)
    r = 2 * f.numel()
    angle = position.cpu().double()[..., None, None] * f
    cos, sin = angle.cos() * magnitude, angle.sin() * magnitude * (-1 if inverse else 1)
    y, size = x.clone(), torch.zeros_like(x)
    first = torch.arange(r // 2) * 2 if interleaved else torch.arange(r // 2)
    second = first + 1 if interleaved else first + r // 2
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    both = (a.abs() + b.abs()) * abs(magnitude)
    size[..., first], size[..., second] = both, both
    if dtype == torch.float32:
        return y, 6 * 2.0**-24 * size
    tol = UNIT[dtype] * y.abs() + 2.0**-21 * size
    tol[..., r:] = 0
    if dtype == torch.float16:
        tol[..., :r] += 2.0**-25
    return y, tol


def within(got, want, what):
    value, tol = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    off = (got - value).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst off "
                           f"{float(off[bad].max())} of {float(tol[bad].max())}")


def attention(q, cache_k, cache_v, pages, starts, lengths=None, window=None, sinks=0, scale=None):
    """(value, tolerance); ``starts``, ``lengths``: lists or None."""
    dtype = q.dtype
    q, cache_k, cache_v = (t.detach().cpu().double() for t in (q, cache_k, cache_v))
    pages = pages.cpu().long()
    batch, tokens, heads, dim = q.shape
    n_pages, size, kv_heads = cache_k.shape[:3]
    group = heads // kv_heads
    scale = dim**-0.5 if scale is None else scale
    window = 2**40 if window is None else window
    value, tol = torch.zeros_like(q), torch.full_like(q, 1e-37)
    largest, most, widest = 0.0, 1, 1.0
    sizes = torch.zeros_like(q)
    for b in range(batch):
        start = 0 if starts is None else int(starts[b])
        n = tokens if lengths is None else min(max(int(lengths[b]), 0), tokens)
        if start < 0 or n == 0:
            continue
        end = min(start + n, pages.shape[1] * size)
        j = torch.arange(end)
        page = pages[b][j // size] if end else j
        there = (page >= 0) & (page < n_pages)
        j, page = j[there], page[there]
        # (of positions that far nothing is cached, and 64 bits hold their sums)
        p = min(start, 2**62) + torch.arange(n)[:, None]
        seen = (j <= p) & ((p - j < window) | (j < sinks))
        used = seen.any(0)
        j, page, seen = j[used], page[used], seen[:, used]
        k, v = cache_k[page, j % size], cache_v[page, j % size]
        most = max(most, int(seen.sum(1).max()) if j.numel() else 1)
        for h in range(heads):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[b, :n, h]
            # a key that one query does not see is no part of it, whatever it holds
            s = torch.where(seen, (qq @ kk.T) * scale, -math.inf)
            if seen.any():
                absolute = torch.where(seen, (qq.abs() @ kk.abs().T) * abs(scale), 0.0)
                largest = max(largest, float(absolute.nan_to_num(0, 0, 0).max()))
            a = torch.softmax(s, 1) if j.numel() else s
            a = torch.where(seen.any(1, keepdim=True), a, 0.0)
            terms = torch.where(seen[:, :, None], a[:, :, None] * vv, 0.0)
            value[b, :n, h] = terms.sum(1)
            sizes[b, :n, h] = terms.abs().sum(1)
            widest = max(widest, float(vv.nan_to_num(0, 0, 0).abs().max()) if j.numel() else 0.0)
    eps = 3 * UNIT[dtype] + (most + dim + 8) * 2.0**-23 * (1 + largest)
    tol = eps * sizes + tol
    if dtype == torch.float16:
        tol = tol + 2.0**-24 * (1 + widest)
    return value, tol
