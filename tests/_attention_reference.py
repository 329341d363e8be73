"""Window attention by its definition, in 64 bits on the CPU, with the
magnitudes that a result's rounding errors scale with.

Tolerances.  With u the unit roundoff of the storage type (2^-24, 2^-11,
2^-8), sums of n products in float32 and A the largest sum of a score's
absolute terms:

- a score is off by at most (dim + 2) 2^-24 A, its probability by that share
  (twice with the normaliser), and the probability's own rounding to the
  storage type by u;
- every output is a sum of products, off by (n + dim) 2^-24 of the sum of
  their absolute values (its magnitude), and rounded once: u;
- delta = grad . out takes out's rounding: u of the sum of |grad out|, which
  the magnitude of dS holds.

So |got - want| <= (3 u + (n + dim + 8) 2^-23 (1 + A)) magnitude, and in
float16 each rounded factor may lose 2^-24 absolutely (its subnormals).
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def seen_mask(lq, lk, window, sinks, n):
    p = torch.arange(lq)[:, None] + (lk - lq)
    j = torch.arange(lk)[None, :]
    return (j <= p) & (j < n) & (p < n) & ((p - j < window) | (j < sinks))


def reference(q, k, v, *, window, sinks=0, scale=None, lengths=None, grad=None):
    """{name: (value, magnitude)} of out (and dq, dk, dv), in float64."""
    dtype = q.dtype
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    batch, lq, heads, dim = q.shape
    lk, kv_heads = k.shape[1], k.shape[2]
    group = heads // kv_heads
    scale = dim**-0.5 if scale is None else scale
    grad = None if grad is None else grad.detach().cpu().double()
    names = ("out",) if grad is None else ("out", "dq", "dk", "dv")
    like = {"out": q, "dq": q, "dk": k, "dv": v}
    value = {n: torch.zeros_like(like[n]) for n in names}
    size = {n: torch.zeros_like(like[n]) for n in names}
    largest, most = 0.0, 1
    for b in range(batch):
        n = lk if lengths is None else min(max(int(lengths[b]), 0), lk)
        seen = seen_mask(lq, lk, window, sinks, n)
        most = max(most, int(seen.sum(1).max()) if lk and lq else 1,
                   group * int(seen.sum(0).max()) if lk and lq else 1)
        rows, keys = seen.any(1), seen.any(0)
        for h in range(heads):
            # what no query sees, and queries that see nothing, take no part
            qq = torch.where(rows[:, None], q[b, :, h], 0.0)
            kk = torch.where(keys[:, None], k[b, :, h // group], 0.0)
            vv = torch.where(keys[:, None], v[b, :, h // group], 0.0)
            s = torch.where(seen, (qq @ kk.T) * scale, -math.inf)
            if seen.any():
                largest = max(largest, float((((qq.abs() @ kk.abs().T) * abs(scale)) * seen).max()))
            p = torch.softmax(s, 1) if lk else s
            p = torch.where(seen.any(1, keepdim=True), p, 0.0)
            o = p @ vv
            value["out"][b, :, h] = o
            size["out"][b, :, h] = p @ vv.abs()
            if grad is None:
                continue
            g = torch.where(rows[:, None], grad[b, :, h], 0.0)
            ds = p * (g @ vv.T - (g * o).sum(1, keepdim=True))
            ds_size = p * (g.abs() @ vv.abs().T + (g.abs() * (p @ vv.abs())).sum(1, keepdim=True))
            value["dq"][b, :, h] = ds @ kk * scale
            size["dq"][b, :, h] = ds_size @ kk.abs() * abs(scale)
            value["dk"][b, :, h // group] += ds.T @ qq * scale
            size["dk"][b, :, h // group] += ds_size.T @ qq.abs() * abs(scale)
            value["dv"][b, :, h // group] += p.T @ g
            size["dv"][b, :, h // group] += p.T @ g.abs()
    u = UNIT[dtype]
    eps = 3 * u + (most + dim + 8) * 2.0**-23 * (1 + largest)
    floor = 1e-37
    if dtype == torch.float16:
        operands = [t for t in (q, k, v, grad) if t is not None and t.numel()]
        widest = max([float(t.nan_to_num(0, 0, 0).abs().max()) for t in operands] + [1.0])
        floor = 2.0**-24 * (1 + most * widest)
    return {n: (value[n], eps * size[n] + floor) for n in names}


def check(got, want, what):
    value, tol = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - value).abs()
    bad = off > tol
    if bad.any():
        worst = (off / tol).argmax()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                             f"{float(off.flatten()[worst])} of {float(tol.flatten()[worst])} at "
                             f"{int(worst)}")


def ring_reference(q, k, v, cache_k, cache_v, lengths, *, window, sinks, scale=None):
    """(out (value, tolerance), caches after the step) of a single token."""
    cache_k, cache_v = cache_k.detach().cpu().clone(), cache_v.detach().cpu().clone()
    batch, heads, dim = q.shape
    ring = cache_k.shape[1] - sinks
    values, tols = [], []
    for b in range(batch):
        p = int(lengths[b])
        if p < 0:
            values.append(torch.zeros(heads, dim, dtype=torch.float64))
            tols.append(torch.full((heads, dim), 1e-37, dtype=torch.float64))
            continue
        slot = [j if j < sinks else sinks + (j - sinks) % ring for j in range(p + 1)]
        cache_k[b, slot[p]] = k[b].cpu()
        cache_v[b, slot[p]] = v[b].cpu()
        at = sorted(set(range(min(sinks, p + 1))) | set(range(max(0, p - window + 1), p + 1)))
        rows = [slot[j] for j in at]
        n = len(at)
        # one query at the end of the keys it sees
        got = reference(q[b:b + 1, None].cpu(), cache_k[b:b + 1, rows], cache_v[b:b + 1, rows],
                        window=n, sinks=0, scale=scale)["out"]
        values.append(got[0][0, 0])
        tols.append(got[1][0, 0])
    empty = torch.zeros(0, heads, dim, dtype=torch.float64)
    return ((torch.stack(values) if values else empty, torch.stack(tols) if tols else empty),
            cache_k, cache_v)
