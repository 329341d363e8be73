"""Accuracy of window attention's gradients where rounding could cost more than
a rounding: attention concentrated on a sink, upstream gradients at the ends
of float16's range.

Tolerances, as norms over a whole tensor, u the unit roundoff of the storage
type.  A rounding of each term of a sum, or of the result, costs u of the
norm at most:

- out: probabilities and the result, 2 u;
- dv: the same, 2 u;
- dq, dk: dS, the result, and delta = sum_j P_j dP_j, which enters as
  P (dP - delta) and so has to be good to u of dP - delta, 3 u.

Scores, statistics and sums are float32: (n + dim + 8) 2^-23 (1 + A) with A
the largest sum of a score's absolute terms, n the longest sum.  Of dP and
delta, sums of dim products of either sign, the partial sums' roundings come
to 0.3 2^-24 |grad| |v| in the mean square each; allowed is 2 each, weighted
by P (whose squares over a row sum to one at most) and carried on to dq and dk
by the widest key or query, a row beside the other.  float16 results lose
what rounding the exact ones to its subnormals costs.
"""

from __future__ import annotations

import torch

from _attention_reference import UNIT, reference

ROUNDINGS = {"out": 2, "dq": 3, "dk": 3, "dv": 2}


def concentrated(seed, batch, tokens, heads, kv_heads, dim, dtype, device, score):
    """(q, k, v, grad) where key 0 is worth ``score`` to every query and the
    others a standard normal score: a share of the softmax that any count of
    them cannot take from it."""
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, dtype=torch.float64)

    along = normal(dim)
    along /= along.norm()
    q, k = normal(batch, tokens, heads, dim), normal(batch, tokens, kv_heads, dim)
    q -= (q @ along)[..., None] * along
    k -= (k @ along)[..., None] * along
    q += 16.0 * along
    k[:, 0] = along * (score * dim**0.5 / 16.0)
    v, g = normal(batch, tokens, kv_heads, dim), normal(batch, tokens, heads, dim)
    return tuple(t.to(dtype).to(device) for t in (q, k, v, g))


def largest_share(q, k, *, window, sinks):
    """Mean over the queries of their largest probability (head 0 of each)."""
    q, k = q[0, :, 0].double().cpu(), k[0, :, 0].double().cpu()
    s = q @ k.T * q.shape[1]**-0.5
    i = torch.arange(len(q))
    seen = (i[:, None] >= i) & ((i[:, None] - i < window) | (i < sinks))
    return float(torch.softmax(s.masked_fill(~seen, -torch.inf), 1).amax(1).mean())


def gradients_in_norm(ms, q, k, v, grad, what, **pattern):
    """Output and gradients against the definition, each in its norm."""
    dtype = q.dtype
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ms.window_attention(*leaves, **pattern)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, grad)), out=out.detach())
    want = {n: value for n, (value, _) in reference(q, k, v, grad=grad, **pattern).items()}
    seen = min(q.shape[1], pattern["window"] + pattern.get("sinks", 0))
    scale = pattern.get("scale") or q.shape[3]**-0.5
    size = float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * abs(scale)
    sums = (seen + q.shape[3] + 8) * 2.0**-23 * (1 + size)

    def widest(t):
        return float(t.double().norm(dim=-1).max())

    ds = 4 * 2.0**-24 * widest(grad) * widest(v) * abs(scale) * (q[..., 0].numel())**0.5
    carried = {"dq": ds * widest(k), "dk": ds * widest(q)}
    errors = {}
    for name, value in got.items():
        exact = want[name]
        assert torch.isfinite(value).all(), f"{what} {name}: not finite"
        floor = 0.0
        if dtype == torch.float16:
            once = exact.to(dtype).double()
            assert torch.isfinite(once).all(), "the inputs' exact result fits"
            floor = float((once - exact).norm())
        errors[name] = float((value.cpu().double() - exact).norm())
        most = (ROUNDINGS[name] * UNIT[dtype] + sums) * float(exact.norm()) + floor
        most += carried.get(name, 0.0)
        assert errors[name] <= most, (f"{what} {name}: off by {errors[name]:.3g} of "
                                      f"{float(exact.norm()):.3g}, tolerated {most:.3g}")
    return errors
