"""Attention that counts keys: queries of zeros weigh all keys alike, and values say which
key they are, so that an output is a count over the number of keys seen.

The first half of a head's values is one-hot in the key's place among `dim / 2` neighbours, the
second in the number of the `dim / 2` it lies in.  A lost key, step or part, one joined twice, or
one too many moves a count of some n / (dim / 2) by one at least.  The weights are the same number
for every key, so that sums lose nothing but that number's rounding; a quotient and the output's
own rounding are left, together within (u + 2^-18) of the count: a key more or less of n is seen
while n < dim / 2 / (u + 2^-18), a step of 32 of them up to 32 times that.
"""

from __future__ import annotations

import torch

from _attention_reference import UNIT
from _paged_checks import table_for


def marks(j, dim):
    """What the value of key j holds."""
    half = dim // 2
    out = torch.zeros(len(j), dim, dtype=torch.float64)
    rows = torch.arange(len(j))
    out[rows, j % half] = 1.0
    out[rows, half + j // half % half] = 1.0
    return out


def counted(start, tokens, dim, capacity, window=None, sinks=0):
    """(queries, dim): what each of a sequence's queries has to give."""
    end = min(start + tokens, capacity)
    j = torch.arange(end)
    p = start + torch.arange(tokens)[:, None]
    seen = ((j <= p) & ((p - j < (window or 2**40)) | (j < sinks))).double()
    return seen @ marks(j, dim) / seen.sum(1, keepdim=True).clamp(min=1)


def outside(got, want, dtype):
    """Values that are off by more than rounding takes."""
    tol = (UNIT[dtype] + 2.0**-18) * want + (2.0**-25 if dtype == torch.float16 else 0)
    return ~((got.double().cpu() - want).abs() <= tol)


def counts_case(ms, device, dtype, starts, *, tokens=1, lengths=None, heads=4, kv_heads=2, dim=64, size=16,
                window=None, sinks=0, shared=0, width=None):
    gen = torch.Generator().manual_seed(len(starts) + tokens)
    new = [tokens] * len(starts) if lengths is None else lengths
    ends = [0 if s < 0 else s + n for s, n in zip(starts, new)]
    width = width or max(-(-max(ends) // size), shared)
    total, table = table_for(gen, ends, size, width, shared=shared)
    cv = torch.full((total, size, kv_heads, dim), 1000.0)  # seen by nobody
    for b, end in enumerate(ends):
        j = torch.arange(min(end, width * size))
        cv[table[b, j // size], j % size] = marks(j, dim).float()[:, None].expand(-1, kv_heads, -1)
    ck = torch.randn(total, size, kv_heads, dim, generator=gen)
    q = torch.zeros(len(starts), tokens, heads, dim)
    q, ck, cv = (t.to(dtype).to(device) for t in (q, ck, cv))
    out = ms.paged_attention(q, ck, cv, table.int().to(device), starts=torch.tensor(starts).to(device),
                             lengths=None if lengths is None else torch.tensor(lengths).to(device),
                             window=window, sinks=sinks, shared_pages=shared)
    for b, (start, n) in enumerate(zip(starts, new)):
        if start < 0:
            assert (out[b] == 0).all()
            continue
        want = counted(start, n, dim, width * size, window, sinks)[:, None].expand(-1, heads, -1)
        bad = outside(out[b, :n], want, dtype)
        assert not bad.any(), (f"{dtype} sequence {b} from {start}: {int(bad.sum())} of {bad.numel()} outside, "
                               f"first at {bad.nonzero()[0].tolist()}")
        assert (out[b, n:] == 0).all()
