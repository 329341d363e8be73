"""Checks of window attention that run on either device."""

from __future__ import annotations

import torch

from _attention_reference import check, reference, ring_reference


def operands(seed, batch, lq, lk, heads, kv_heads, dim, dtype, device, spread=1.0):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return (torch.randn(shape, generator=gen) * spread).to(dtype).to(device)

    return (normal(batch, lq, heads, dim), normal(batch, lk, kv_heads, dim),
            normal(batch, lk, kv_heads, dim), normal(batch, lq, heads, dim))


def forward_and_gradients(ms, q, k, v, grad, what, **pattern):
    """Output and gradients against the definition."""
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out = ms.window_attention(q, k, v, **pattern)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), grad)), out=out)
    want = reference(q, k, v, grad=grad, **pattern)
    for name, value in got.items():
        assert value.dtype == q.dtype
        check(value, want[name], f"{what} {name}")
    with torch.no_grad():
        assert torch.equal(ms.window_attention(q, k, v, **pattern), out), f"{what}: without grad"
    return got


def step(ms, seed, lengths, heads, kv_heads, dim, dtype, device, *, window, sinks, slots=None,
         index=torch.int32, spread=1.0, unseen=None):
    """One step against the definition; ``unseen``: what the slots hold that
    nothing has been written to, or that the query does not see."""
    gen = torch.Generator().manual_seed(seed)
    batch = len(lengths)
    slots = slots or window + sinks

    def normal(*shape):
        return (torch.randn(shape, generator=gen) * spread).to(dtype).to(device)

    q, k, v = normal(batch, heads, dim), normal(batch, kv_heads, dim), normal(batch, kv_heads, dim)
    ck, cv = normal(batch, slots, kv_heads, dim), normal(batch, slots, kv_heads, dim)
    ring = slots - sinks
    if unseen is not None:
        for b, p in enumerate(lengths):
            at = set(range(min(sinks, p + 1))) | set(range(max(0, p - window + 1), p + 1))
            held = {j if j < sinks else sinks + (j - sinks) % ring for j in at}
            if p >= 0:
                held.discard(p if p < sinks else sinks + (p - sinks) % ring)
            free = [s for s in range(slots) if s not in held]
            ck[b, free] = unseen
            cv[b, free] = unseen
    before = ck.clone(), cv.clone()
    n = torch.tensor(lengths, dtype=index, device=device)
    want, want_k, want_v = ring_reference(q, k, v, ck, cv, lengths, window=window, sinks=sinks)
    out = ms.window_attention_step(q, k, v, ck, cv, n, window=window, sinks=sinks)
    check(out, want, f"step {lengths} window={window} sinks={sinks} slots={slots} dim={dim}")
    for got, expect, old in ((ck, want_k, before[0]), (cv, want_v, before[1])):
        assert torch.equal(got.cpu().view(torch.uint8), expect.view(torch.uint8))
        assert got.shape == old.shape
    return out


def prompt_then_steps(ms, device, dtype, *, window, sinks, prompt, more, heads=4, kv_heads=2,
                      dim=32, batch=3):
    """Steps after a stored prompt equal the rows of one long product."""
    total = max(prompt) + more
    q, k, v, _ = operands(9, batch, total, total, heads, kv_heads, dim, dtype, device)
    lengths = torch.tensor(prompt, dtype=torch.int32, device=device)
    whole = reference(q, k, v, window=window, sinks=sinks)["out"]
    slots = window + sinks
    ck = torch.full((batch, slots, kv_heads, dim), float("nan"), dtype=dtype, device=device)
    cv = ck.clone()
    ms.window_cache_store(k, v, ck, cv, sinks=sinks, lengths=lengths)
    rows = torch.arange(batch, device=device)
    for _ in range(more):
        at = lengths.long()
        out = ms.window_attention_step(q[rows, at], k[rows, at], v[rows, at], ck, cv, lengths,
                                       window=window, sinks=sinks)
        cpu = at.cpu()
        check(out, tuple(t[torch.arange(batch), cpu] for t in whole), f"step at {cpu.tolist()}")
        lengths = lengths + 1
