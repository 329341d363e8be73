"""Distillation by its definition, in 64 bits on the CPU, with tolerances.

With A the largest |logit| / T of either side, u the storage type's unit
roundoff: a scaled logit is off by 2^-23 A, the logarithm of a sum of
exponentials by (levels of the sum + 4) 2^-23 and that; so

- loss / T^2 = sum p (ln p - ln q): off by 2^-21 (8 + A) (1 + sum p |ln p -
  ln q|);
- gradient = weight T (q - p): off by u of itself (its rounding) and by
  2^-21 (8 + A) (q + p) weight T; in float16 by 2^-25 more (subnormals).

The sums have at most 20 levels where they are added pairwise by the threads
of a row, each of which adds up to n of them in turn: n 2^-24 more.
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def reference(logits, data, indices, indptr, *, temperature=1.0, weights=None, serial=1):
    """(losses, tolerance), (gradient, tolerance); ``serial``: terms a thread
    adds in turn."""
    dtype = logits.dtype
    z = logits.detach().cpu().double().reshape(-1, logits.shape[-1]) / temperature
    t = data.detach().cpu().double() / temperature
    indices, indptr = indices.cpu().tolist(), indptr.cpu().tolist()
    rows, vocab = z.shape
    w = torch.ones(rows, dtype=torch.float64) if weights is None else weights.cpu().double()
    loss, loss_tol = torch.zeros(rows, dtype=torch.float64), torch.full((rows,), 1e-37).double()
    grad, grad_tol = torch.zeros_like(z), torch.full_like(z, 1e-37)
    for i in range(rows):
        kept = [e for e in range(indptr[i], indptr[i + 1])
                if 0 <= indices[e] < vocab and float(t[e]) != -math.inf]
        if not kept:
            continue
        columns = torch.tensor([indices[e] for e in kept])
        log_p = torch.log_softmax(t[kept], 0)
        p = log_p.exp()
        log_q = torch.log_softmax(z[i], 0)
        terms = torch.where(p > 0, p * (log_p - log_q[columns]), 0.0)
        finite = z[i][torch.isfinite(z[i])]
        top = max(float(finite.abs().max()), float(t[kept].abs().max()))
        eps = (2.0**-21 * (8 + top) + (serial + len(kept)) * 2.0**-24)
        loss[i] = terms.sum() * temperature**2
        loss_tol[i] += eps * (1 + float(terms.abs().sum())) * temperature**2
        if float(w[i]) == 0:
            continue
        summed = torch.zeros(vocab, dtype=torch.float64).index_add_(0, columns, p)
        factor = w[i] * temperature
        grad[i] = (log_q.exp() - summed) * factor
        grad_tol[i] += (UNIT[dtype] * grad[i].abs()
                        + eps * (log_q.exp() + summed) * factor.abs()
                        + (2.0**-25 if dtype == torch.float16 else 0.0))
    return (loss, loss_tol), (grad, grad_tol)


def check(got, want, what):
    value, tol = want
    got = got.detach().cpu().double().reshape(value.shape)
    same = torch.isinf(value) & (got == value)
    off = torch.where(same, 0.0, (got - value).abs())
    bad = ~(off <= tol) & ~same
    if bad.any():
        at = int(bad.flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {at}: "
                             f"{float(got.flatten()[at])}, want {float(value.flatten()[at])} "
                             f"within {float(tol.flatten()[at])}")
