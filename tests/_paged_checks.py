"""Checks of rotary positions and paged caches that run on either device."""

from __future__ import annotations

import torch

from _attention_reference import check
from _paged_reference import attention, turned, within


def normal(gen, dtype, device, *shape, spread=1.0):
    return (torch.randn(shape, generator=gen) * spread).to(dtype).to(device)


def rotation_case(ms, device, dtype, *, batch=2, tokens=5, heads=3, dim=32, rotated=0,
                  interleaved=False, where="starts", index=torch.int64, layout="plain", seed=1,
                  far=0, **how):
    """Values and gradient at starts, positions or neither."""
    gen = torch.Generator().manual_seed(seed)
    rotation = ms.Rotary(rotated or dim, interleaved=interleaved, **how)
    if layout == "plain":
        x = normal(gen, dtype, device, batch, tokens, heads, dim)
    elif layout == "packed":  # a view of a projection
        x = normal(gen, dtype, device, batch, tokens, heads + 2, dim)[:, :, 1:-1]
    elif layout == "heads first":
        x = normal(gen, dtype, device, batch, heads, tokens, dim).transpose(1, 2)
    else:  # "odd": rows at odd addresses
        x = normal(gen, dtype, device, batch, tokens, heads, dim + 1)[..., 1:]
    at = torch.arange(tokens).expand(batch, -1)
    kwargs = {}
    if where == "starts":
        starts = torch.randint(0, 100, (batch,), generator=gen) + far
        at = at + starts[:, None]
        kwargs["starts"] = starts.to(index).to(device)
    elif where == "positions":
        at = torch.randint(-50, 100, (batch, tokens), generator=gen) + far
        kwargs["positions"] = at.to(index).to(device)
    elif where == "one row of positions":
        at = (torch.randperm(tokens, generator=gen) + far).expand(batch, -1)
        kwargs["positions"] = at[0].to(index).to(device).expand(batch, -1)
    x = x.detach().requires_grad_()
    out = ms.rotary(x, rotation, **kwargs)
    what = f"{dtype} {tuple(x.shape)} {rotation} {where} {layout}"
    assert out.dtype == dtype and out.is_contiguous()
    f, m = rotation.frequencies, rotation.magnitude
    within(out, turned(x, at, f, m, interleaved), what)
    up = normal(gen, dtype, device, *x.shape)
    got, = torch.autograd.grad(out, x, up)
    within(got, turned(up, at, f, m, interleaved, inverse=True), f"{what}: gradient")
    with torch.no_grad():
        assert torch.equal(ms.rotary(x, rotation, **kwargs), out)
    return x, out


def table_for(gen, ends, size, width, extra=3, wrong=True, shared=0):
    """(pages of the cache, a table of scattered pages): sequence b holds its
    first ``ends[b]`` positions; what is behind names no page that is there."""
    need = [max(-(-min(max(n, 0), width * size) // size), shared if n > 0 else 0) for n in ends]
    total = sum(max(n - shared, 0) for n in need) + shared + extra
    order = torch.randperm(total, generator=gen).tolist()
    common = [order.pop() for _ in range(shared)]
    table = torch.full((len(ends), width), -1, dtype=torch.int64)
    if wrong:
        table[:, 1::2] = total + 7
    table[:, :shared] = torch.tensor(common, dtype=torch.int64)
    for b, n in enumerate(need):
        for e in range(shared, n):
            table[b, e] = order.pop()
    return total, table


def paged_case(ms, device, dtype, starts, *, tokens=1, heads=4, kv_heads=2, dim=32, size=16,
               lengths=None, window=None, sinks=0, scale=None, shared=0, width=None,
               index=torch.int32, table_index=torch.int32, layout="plain", poison=True, seed=3,
               spread=1.0, holes=(), change=None):
    """paged_attention against the definition.  ``poison``: what no query sees is
    NaN; ``holes``: (sequence, entry) of pages that are not there."""
    gen = torch.Generator().manual_seed(seed)
    batch = len(starts)
    new = [tokens] * batch if lengths is None else lengths
    ends = [0 if s < 0 else s + min(max(n, 0), tokens) for s, n in zip(starts, new)]
    if width is None:
        width = max([-(-n // size) for n in ends] + [shared, 0]) + 1
    total, table = table_for(gen, ends, size, width, shared=shared)
    for b, e in holes:
        table[b, e] = -1 if (b + e) % 2 else total
    if layout == "plain":
        ck = normal(gen, dtype, device, total, size, kv_heads, dim, spread=spread)
        cv = normal(gen, dtype, device, total, size, kv_heads, dim, spread=spread)
        q = normal(gen, dtype, device, batch, tokens, heads, dim, spread=spread)
    elif layout == "packed":  # keys and values side by side, heads before slots
        both = normal(gen, dtype, device, total, 2, kv_heads, size, dim, spread=spread)
        ck, cv = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
        q = normal(gen, dtype, device, batch, tokens, heads + 2, dim, spread=spread)[:, :, 1:-1]
    else:  # "odd": caches and queries at odd addresses
        ck = normal(gen, dtype, device, total, size, kv_heads, dim + 1, spread=spread)[..., 1:]
        cv = normal(gen, dtype, device, total, size, kv_heads, dim + 1, spread=spread)[..., 1:]
        q = normal(gen, dtype, device, batch, tokens, heads, dim + 1, spread=spread)[..., 1:]
    if poison:
        seen = torch.zeros(total, size, dtype=torch.bool)
        for b, (s, end) in enumerate(zip(starts, ends)):
            for j in range(max(min(end, width * size), 0)):
                low = 0 if window is None else max(s - window + 1, 0)
                page = int(table[b, j // size])
                if (j >= low or j < sinks) and 0 <= page < total:
                    seen[page, j % size] = True
        ck[~seen.to(device)] = float("nan")
        cv[~seen.to(device)] = float("nan")
    if change is not None:
        change(q, ck, cv, table)
    kwargs = {"window": window, "sinks": sinks, "scale": scale}
    out = ms.paged_attention(q, ck, cv, table.to(table_index).to(device),
                             starts=torch.tensor(starts).to(index).to(device),
                             lengths=None if lengths is None
                             else torch.tensor(lengths).to(index).to(device),
                             shared_pages=shared, **kwargs)
    want = attention(q, ck, cv, table, starts, lengths, **kwargs)
    what = (f"{dtype} {starts} tokens {tokens} heads {heads}/{kv_heads} of {dim} pages of {size} "
            f"window {window} sinks {sinks} shared {shared} {layout}")
    assert out.dtype == dtype and out.is_contiguous()
    if change is None:
        check(out, want, what)
    return out, want


def append_case(ms, device, dtype, starts, *, tokens=1, heads=4, kv_heads=2, dim=32, size=16,
                lengths=None, rotated=0, interleaved=False, with_q=True, width=None,
                index=torch.int32, table_index=torch.int64, layout="plain", rotate=True, seed=5,
                holes=(), **how):
    """paged_cache_append: what is written is right, and nothing else is."""
    gen = torch.Generator().manual_seed(seed)
    batch = len(starts)
    new = [tokens] * batch if lengths is None else [min(max(n, 0), tokens) for n in lengths]
    ends = [0 if s < 0 else s + n for s, n in zip(starts, new)]
    if width is None:
        width = max([-(-n // size) for n in ends] + [0]) + 1
    total, table = table_for(gen, ends, size, width)
    for b, e in holes:
        table[b, e] = -1 if (b + e) % 2 else total
    pad = 1 if layout == "odd" else 0
    packed = normal(gen, dtype, device, batch, tokens, heads + 2 * kv_heads, dim + pad)[..., pad:]
    q, k, v = packed.split([heads, kv_heads, kv_heads], dim=2)
    if layout == "packed":
        both = normal(gen, dtype, device, total, 2, kv_heads, size, dim)
        ck, cv = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    else:
        ck = normal(gen, dtype, device, total, size, kv_heads, dim + pad)[..., pad:]
        cv = normal(gen, dtype, device, total, size, kv_heads, dim + pad)[..., pad:]
    rotation = ms.Rotary(rotated or dim, interleaved=interleaved, **how) if rotate else None
    want_k, want_v = ck.detach().cpu().double(), cv.detach().cpu().clone()
    tol_k = torch.zeros_like(want_k)
    want_q, tol_q = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, (s, n) in enumerate(zip(starts, new)):
        if s < 0:
            continue
        at = s + torch.arange(n)
        if rotate:
            f = (rotation.frequencies, rotation.magnitude, interleaved)
            want_q[b, :n], tol_q[b, :n] = turned(q[b, :n], at, *f)
            turn_k = turned(k[b, :n], at, *f)
        else:
            turn_k = k[b, :n].cpu().double(), torch.zeros(n, kv_heads, dim, dtype=torch.float64)
        for t in range(n):
            j = s + t
            page = int(table[b, j // size]) if j < width * size else -1
            if 0 <= page < total:
                want_k[page, j % size], tol_k[page, j % size] = turn_k[0][t], turn_k[1][t]
                want_v[page, j % size] = v[b, t].cpu()
    got = ms.paged_cache_append(
        k, v, ck, cv, table.to(table_index).to(device),
        starts=torch.tensor(starts).to(index).to(device),
        lengths=None if lengths is None else torch.tensor(lengths).to(index).to(device),
        rotation=rotation, q=q if with_q and rotate else None)
    what = f"{dtype} {starts} tokens {tokens} of {dim} pages of {size} {rotation} {layout}"
    within(ck, (want_k, tol_k), f"{what}: keys")
    assert torch.equal(cv.cpu(), want_v), f"{what}: values"
    if with_q and rotate:
        within(got, (want_q, tol_q), f"{what}: queries")
    else:
        assert got is None


def prompt_then_steps(ms, device, dtype, *, prompt=(21, 7, 12), more=4, chunk=8, heads=4,
                      kv_heads=2, dim=32, size=8, window=None, sinks=0):
    """A prompt in chunks, then single tokens: each row equals that of one
    product over the whole sequence, rotated as a whole."""
    gen = torch.Generator().manual_seed(9)
    batch, total = len(prompt), max(prompt) + more
    q = normal(gen, dtype, device, batch, total, heads, dim)
    k = normal(gen, dtype, device, batch, total, kv_heads, dim)
    v = normal(gen, dtype, device, batch, total, kv_heads, dim)
    rotation = ms.Rotary(dim, scaling="linear", factor=2.0)
    rq, rk = ms.rotary(q, rotation), ms.rotary(k, rotation)
    whole = ms.window_attention(rq, rk, v, window=window or total, sinks=sinks)
    width = -(-total // size)
    pages = torch.randperm(batch * width, generator=gen).reshape(batch, width).int().to(device)
    ck = torch.full((batch * width, size, kv_heads, dim), float("nan"), dtype=dtype, device=device)
    cv = ck.clone()
    left = torch.tensor(prompt)
    start = torch.zeros(batch, dtype=torch.int32)
    rows = torch.arange(batch)

    # both are within a tolerance of the definition, so within two of one another
    def compare(out, at, n):
        for b in range(batch):
            m = int(n[b])
            first = int(at[b])
            ref = attention(rq[b:b + 1, :total].cpu(), *single(rk, v, b), [0], None, window, sinks)
            close = ref[0][:, first:first + m], 2 * ref[1][:, first:first + m]
            check(out[b:b + 1, :m], close, f"sequence {b} from {first}")
            check(whole[b:b + 1, first:first + m], close, f"sequence {b} from {first}: whole")
            assert (out[b, m:] == 0).all()

    def single(rk, v, b):
        k1, v1 = (t[b, :total].cpu().unsqueeze(0) for t in (rk, v))
        return k1, v1, torch.zeros(1, 1, dtype=torch.int64)

    while left.max() > 0:
        n = left.clamp(max=chunk).int()
        at = (start.long()[:, None] + torch.arange(chunk)).clamp(max=total - 1)
        pick = lambda t: t[rows[:, None].to(device), at.to(device)]  # noqa: E731
        s, l = start.to(device), n.to(device)
        got = ms.paged_cache_append(pick(k), pick(v), ck, cv, pages, starts=s, lengths=l,
                                    rotation=rotation, q=pick(q))
        out = ms.paged_attention(got, ck, cv, pages, starts=s, lengths=l, window=window, sinks=sinks)
        compare(out, start, n)
        start, left = start + n, left - n
    for _ in range(more):
        at = start.long()[:, None]
        pick = lambda t: t[rows[:, None].to(device), at.to(device)]  # noqa: E731
        s = start.to(device)
        got = ms.paged_cache_append(pick(k), pick(v), ck, cv, pages, starts=s, rotation=rotation,
                                    q=pick(q))
        out = ms.paged_attention(got, ck, cv, pages, starts=s, window=window, sinks=sinks)
        compare(out, start, [1] * batch)
        start = start + 1
