"""Rotary positions, paged caches and the attention that reads them: workloads
for timing the package's operators and comparing them with their plain forms.

Each case is one pass:

- ``rotate``: ``rotary`` over queries and keys that lie side by side, where
  ``grad`` is set with its gradient;
- ``append``: ``paged_cache_append``, keys rotated into a paged cache beside
  their values, the queries rotated in the same call;
- ``attend``: ``paged_attention``, the last tokens of every sequence (one, a
  few drafts, a chunk of a prompt) against its pages; where ``shared`` is set,
  the batch shares its first pages.

``own`` false runs the plain forms: products, sums, exponentials, indexing, in
32 bits (angles in 64), rounded once at the end.
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_INDEX = {"i32": torch.int32, "i64": torch.int64}
_BASE = 10_000.0
_TRAINED = 4096  # positions before a context was made longer


def _rotate(batch, tokens, heads, dim, dtype="bf16", *, rotated=0, interleaved=False, scaling="",
            far=False, grad=False, name=None):
    """``rotated``: leading values of a head, 0 for all; ``far``: sequences
    go on at positions beyond a million, else they begin at zero."""
    case = {"op": "rotate", "batch": batch, "tokens": tokens, "heads": heads, "dim": dim,
            "rotated": rotated or dim, "interleaved": interleaved, "scaling": scaling, "far": far,
            "grad": grad, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def _append(batch, tokens, heads, kv_heads, dim, page, keys, dtype="bf16", *, rotated=0,
            interleaved=False, scaling="", ragged=False, index="i32", name=None):
    """``keys``: places a sequence's pages hold; ``ragged``: sequences bring
    from one to ``tokens`` tokens, and some slots of the batch have none."""
    case = {"op": "append", "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "keys": max(keys, tokens),
            "rotated": rotated or dim, "interleaved": interleaved, "scaling": scaling,
            "ragged": ragged, "index": index, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def _attend(batch, tokens, heads, kv_heads, dim, page, keys, dtype="bf16", *, spread="full",
            shared=0, window=0, sinks=0, index="i32", name=None):
    """``keys``: the longest sequence, the new tokens among them; ``spread``:
    "full", all are as long; "ragged", from the shortest on, evenly over the
    logarithm, and some slots of the batch are without a sequence; ``shared``:
    leading tokens that all have in common; ``window`` 0: every key is seen."""
    case = {"op": "attend", "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "keys": max(keys, shared + tokens),
            "spread": spread, "shared": shared // page * page, "window": window, "sinks": sinks,
            "index": index, "dtype": dtype}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a short prompt of a small model in full precision, a part of each head rotated
        _rotate(1, 129, 10, 80, "f32", rotated=48, interleaved=True, name="rotate_small"),
        # a training batch: queries and keys of one layer, forward and back
        _rotate(4, 2048, 20, 128, grad=True, name="rotate_train"),
        # a chunk of a very long document, a context longer than the trained one
        _rotate(1, 16_384, 40, 128, scaling="yarn", far=True, name="rotate_long"),
        # one token of each conversation of a serving batch: latency bound
        _append(64, 1, 32, 8, 128, 16, 512, name="append_batch"),
        # prompts of every length into the cache, odd sizes
        _append(5, 2049, 16, 8, 128, 64, 2100, "f16", scaling="linear", ragged=True,
                name="append_prompts"),
        # one conversation with a small model: latency bound
        _attend(1, 1, 8, 2, 64, 16, 700, name="attend_one"),
        # a serving batch of conversations of every length, pages of an odd size
        _attend(37, 1, 24, 8, 96, 24, 5000, "f16", spread="ragged", index="i64",
                name="attend_ragged"),
        # a large serving batch, few long sequences among many short ones
        _attend(64, 1, 32, 8, 128, 16, 16_384, spread="ragged", name="attend_batch"),
        # one very long document: its keys are all the work there is to share
        _attend(1, 1, 32, 8, 128, 64, 131_072, name="attend_long"),
        # a chunk of a long prompt against the pages before it
        _attend(1, 2048, 16, 8, 128, 64, 18_432, "f16", name="attend_chunk"),
        # a serving batch behind one long instruction
        _attend(64, 1, 32, 8, 128, 16, 9200, spread="ragged", shared=8192, name="shared_batch"),
        # a few drafted tokens of each conversation behind a short instruction
        _attend(9, 4, 16, 4, 64, 16, 1300, "f16", spread="ragged", shared=1040,
                name="shared_drafts"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(high, low))))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "append", "append", "attend", "attend", "attend",
                     "drafts", "chunk", "shared", "shared"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
    dim = rng.choice([64, 64, 128, 128, 128, 32, 80, 96, 256])
    size = _BYTES[dtype]
    part = {"rotated": rng.choice([0, 0, 0, dim // 2, dim // 4 * 2 - 2 or 2]),
            "interleaved": rng.random() < 0.4,
            "scaling": rng.choice(["", "", "linear", "ntk", "yarn"])}
    if op == "rotate":
        grad = rng.random() < 0.5
        batch, wide = rng.choice([1, 1, 2, 5]), heads + kv_heads
        most = 1.6e8 / (size * dim * wide * batch * (2 if grad else 1))
        return _rotate(batch, _log(rng, 1, max(1, min(20_000, most))), wide, dim, dtype,
                       far=rng.random() < 0.4, grad=grad, **part)
    page = rng.choice([16, 16, 32, 64, 64, 128, 1, 5, 24])
    index = rng.choice(["i32", "i32", "i64"])
    row = 2 * size * kv_heads * dim  # bytes of a token's key and value
    if op == "append":
        if rng.random() < 0.5:
            batch = _log(rng, 1, 200)
            keys = _log(rng, 16, max(16, min(2000, 2e8 / (row * batch))))
            return _append(batch, 1, heads, kv_heads, dim, page, keys, dtype,
                           ragged=rng.random() < 0.5, index=index, **part)
        batch = rng.choice([1, 1, 2, 5])
        tokens = _log(rng, 2, max(2, min(8000, 8e7 / (row * batch))))
        return _append(batch, tokens, heads, kv_heads, dim, page, tokens + _log(rng, 1, 500), dtype,
                       ragged=batch > 1, index=index, **part)
    window, sinks = rng.choice([(0, 0), (0, 0), (0, 0), (_log(rng, 16, 4000), rng.choice([0, 4]))])
    spread = rng.choice(["full", "ragged", "ragged"])
    more = {"spread": spread, "window": window, "sinks": sinks, "index": index}
    if op == "chunk":
        batch = rng.choice([1, 1, 2])
        # products of the largest listed one; full precision an eighth of them
        most = 6e10 / (8 if dtype == "f32" else 1) / (heads * dim * batch)
        keys = _log(rng, 200, min(20_000, most / 32))
        tokens = _log(rng, 17, max(17, min(keys, 3000, most / keys)))
        return _attend(batch, tokens, heads, kv_heads, dim, page, keys, dtype, **more)
    tokens = rng.choice([2, 3, 5, 8]) if op == "drafts" else rng.choice([1, 1, 1, 4])
    if op == "attend":
        tokens = 1
    batch = _log(rng, 1, 96)
    keys = _log(rng, 16, max(16, min(130_000, 4e8 / (row * batch))))
    if op == "shared":
        keys = max(keys, 2 * page)
        more["shared"] = rng.randint(page, max(page, keys - tokens))
    return _attend(batch, tokens, heads, kv_heads, dim, page, keys, dtype, **more)


# -- inputs -------------------------------------------------------------------
def _frequencies(case):
    """(radians a position for each pair, magnitude) in 64 bits."""
    r, factor = case["rotated"], 8.0
    exponent = torch.arange(0, r, 2, dtype=torch.float64) / r
    base = _BASE * factor ** (r / (r - 2)) if case["scaling"] == "ntk" and r > 2 else _BASE
    f = base ** -exponent
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "yarn":
        turns = _TRAINED * f / (2 * math.pi)
        kept = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        return kept * f + (1 - kept) * f / factor, 0.1 * math.log(factor) + 1.0
    return f, 1.0


@functools.lru_cache(maxsize=1)
def _package():
    pkg = str(Path(__file__).resolve().parents[1] / "mlx-sparse_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mlx_sparse

    return mlx_sparse


def _rotation(case):
    """What a program keeps beside its weights."""
    if not own:
        frequencies, magnitude = _frequencies(case)
        return frequencies.cuda(), magnitude
    return _package().Rotary(case["rotated"], base=_BASE, interleaved=case["interleaved"],
                             scaling=case["scaling"] or None,
                             factor=8.0 if case["scaling"] else 1.0, trained=_TRAINED)


def _counts(case, seed):
    """(tokens of each sequence before the new ones, new ones), as lists; a
    slot without a sequence has -1 before."""
    gen = torch.Generator().manual_seed(seed)
    n, tokens, keys = case["batch"], case["tokens"], case["keys"]
    if case["op"] == "append":
        new = torch.full((n,), tokens)
        if case["ragged"] and tokens > 1:
            new = torch.randint(1, tokens + 1, (n,), generator=gen)
        before = (torch.rand(n, generator=gen) * (keys - tokens + 1)).long()
    else:
        new = torch.full((n,), tokens)
        before = torch.full((n,), keys - tokens)
        if case["spread"] == "ragged":
            least = case["shared"]
            over = math.log(keys - tokens - least + 1)
            before = least + (torch.exp(torch.rand(n, generator=gen, dtype=torch.float64) * over)
                              - 1).long()
            before[0] = keys - tokens
    if case.get("ragged") or case.get("spread") == "ragged":
        before[2::13] = -1
    return before.tolist(), new.tolist()


def _pool(case, before, new):
    """(pages of the cache, pages of each sequence, shared pages)"""
    page = case["page"]
    shared = case.get("shared", 0) // page
    held = [max(-(-(s + t) // page), shared) if s >= 0 else 0 for s, t in zip(before, new)]
    if case["op"] == "append":  # as many as the batch may come to hold
        return case["batch"] * -(-case["keys"] // page) + 3, held, shared
    return sum(max(h - shared, 0) for h in held) + shared + 3, held, shared


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    batch, tokens, dim = case["batch"], case["tokens"], case["dim"]
    if case["op"] == "rotate":
        state = {"case": case, "x": normal(batch, tokens, case["heads"], dim),
                 "rotation": _rotation(case), "starts": None}
        if case["far"]:
            state["starts"] = torch.randint(1_000_000, 2_000_000, (batch,), generator=gen,
                                            device="cuda")
        if case["grad"]:
            state["x"].requires_grad_()
            state["upstream"] = normal(batch, tokens, case["heads"], dim)
        return state
    heads, kv_heads, page = case["heads"], case["kv_heads"], case["page"]
    index = _INDEX[case["index"]]
    before, new = _counts(case, seed)
    n_pages, held, shared = _pool(case, before, new)
    width = -(-case["keys"] // page)
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    common = [order.pop() for _ in range(shared)]
    # what is behind a sequence's pages is what was there before: other pages
    table = torch.randint(0, n_pages, (batch, width),
                          generator=torch.Generator().manual_seed(seed + 1))
    for b, n in enumerate(held):
        mine = common + [order.pop() for _ in range(n - shared)] if n else common
        table[b, :len(mine)] = torch.tensor(mine, dtype=torch.int64)
    state = {"case": case, "pages": table.to(index).cuda(),
             "starts": torch.tensor(before).to(index).cuda(), "lengths": None,
             "cache_k": normal(n_pages, page, kv_heads, dim),
             "cache_v": normal(n_pages, page, kv_heads, dim)}
    if case["op"] == "attend":
        return state | {"q": normal(batch, tokens, heads, dim)}
    # queries, keys and values as the views of one projection
    packed = normal(batch, tokens, heads + 2 * kv_heads, dim)
    q, k, v = packed.split([heads, kv_heads, kv_heads], dim=2)
    if case["ragged"]:
        state["lengths"] = torch.tensor(new).to(index).cuda()
    return state | {"q": q, "k": k, "v": v, "rotation": _rotation(case)}


# -- one pass -----------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["op"] == "rotate":
            return _plain_rotate(case, state)
        if case["op"] == "append":
            return _plain_append(case, state)
        return _plain_attend(case, state)


def _run_own(case, state):
    ms = _package()
    if case["op"] == "rotate":
        out = ms.rotary(state["x"], state["rotation"], starts=state["starts"])
        if not case["grad"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, state["x"], state["upstream"]))
    if case["op"] == "append":
        q = ms.paged_cache_append(state["k"], state["v"], state["cache_k"], state["cache_v"],
                                  state["pages"], starts=state["starts"],
                                  lengths=state["lengths"], rotation=state["rotation"],
                                  q=state["q"])
        return q, state["cache_k"], state["cache_v"]
    return ms.paged_attention(state["q"], state["cache_k"], state["cache_v"], state["pages"],
                              starts=state["starts"], window=case["window"] or None,
                              sinks=case["sinks"], shared_pages=case["shared"] // case["page"])


def _turned(x, position, rotation, case, sign=1.0):
    """``x`` in 32 bits, rotated at ``position`` (batch x tokens)."""
    frequencies, magnitude = rotation
    angle = position[:, :, None, None].double() * frequencies
    cos, sin = (angle.cos() * magnitude).float(), (angle.sin() * (magnitude * sign)).float()
    r, y = case["rotated"], x.float().clone()
    if case["interleaved"]:
        a, b = x[..., 0:r:2].float(), x[..., 1:r:2].float()
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :r // 2].float(), x[..., r // 2:r].float()
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    return y


def _positions(starts, tokens, batch, device):
    at = torch.arange(tokens, device=device).expand(batch, -1)
    return at if starts is None else at + starts.long()[:, None]


def _plain_rotate(case, state):
    x = state["x"].detach()
    position = _positions(state["starts"], x.shape[1], x.shape[0], x.device)
    out = _turned(x, position, state["rotation"], case).to(x.dtype)
    if not case["grad"]:
        return out
    return out, _turned(state["upstream"], position, state["rotation"], case, -1.0).to(x.dtype)


def _plain_append(case, state):
    q, k, v = state["q"], state["k"], state["v"]
    batch, tokens = k.shape[:2]
    position = _positions(state["starts"], tokens, batch, k.device)
    live = (state["starts"] >= 0)[:, None].expand(-1, tokens)
    if state["lengths"] is not None:
        live = live & (torch.arange(tokens, device=k.device) < state["lengths"][:, None])
    q = _turned(q, position, state["rotation"], case)
    q = torch.where(live[:, :, None, None], q, 0.0).to(k.dtype)
    k = _turned(k, position, state["rotation"], case).to(k.dtype)
    b, t = live.nonzero(as_tuple=True)
    at = position[b, t]
    page = state["pages"].long()[b, at // case["page"]]
    state["cache_k"][page, at % case["page"]] = k[b, t]
    state["cache_v"][page, at % case["page"]] = v[b, t]
    return q, state["cache_k"], state["cache_v"]


def _plain_attend(case, state):
    """Some sequences and some queries of them at a time: their pages side by
    side, scores, softmax, sums."""
    q, dev = state["q"], state["q"].device
    batch, tokens, heads, dim = q.shape
    kv_heads = state["cache_k"].shape[2]
    group = heads // kv_heads
    table, starts = state["pages"].long(), state["starts"].long()
    keys = table.shape[1] * case["page"]
    key = torch.arange(keys, device=dev)
    some = max(1, (1 << 29) // (keys * kv_heads * dim))
    out = torch.empty_like(q)
    for b in range(0, batch, some):
        mine = slice(b, min(b + some, batch))
        n = mine.stop - b
        k = state["cache_k"][table[mine]].reshape(n, keys, kv_heads, dim)
        v = state["cache_v"][table[mine]].reshape(n, keys, kv_heads, dim)
        k = k.permute(0, 2, 3, 1).float().contiguous()
        v = v.permute(0, 2, 1, 3).float().contiguous()
        few = max(1, (1 << 28) // (keys * heads * n))
        for t in range(0, tokens, few):
            rows = slice(t, min(t + few, tokens))
            p = starts[mine, None, None] + torch.arange(t, rows.stop, device=dev)[:, None]
            seen = (key <= p) & (starts[mine] >= 0)[:, None, None]
            if case["window"]:
                seen &= (p - key < case["window"]) | (key < case["sinks"])
            seen = seen[:, None, :, None].expand(-1, -1, -1, group, -1)
            qq = q[mine, rows].float().view(n, -1, kv_heads, group, dim).transpose(1, 2)
            s = (qq.reshape(n, kv_heads, -1, dim) @ k).mul_(dim ** -0.5)
            s = s.view(n, kv_heads, -1, group, keys).masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            e = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
            total = e.sum(-1, keepdim=True)
            e = e.div_(total.masked_fill(total == 0, 1.0)).view(n, kv_heads, -1, keys)
            o = (e @ v).view(n, kv_heads, -1, group, dim).transpose(1, 2)
            out[mine, rows] = o.reshape(n, -1, heads, dim).to(q.dtype)
    return out


# -- what a pass cannot do without ---------------------------------------------
def work(case):
    size, dim = _BYTES[case["dtype"]], case["dim"]
    if case["op"] == "rotate":
        values = case["batch"] * case["tokens"] * case["heads"]
        passes = 2 if case["grad"] else 1
        return {"bytes": 2 * size * dim * values * passes,
                "flops": 3 * case["rotated"] * values * passes}
    heads, kv_heads, tokens = case["heads"], case["kv_heads"], case["tokens"]
    before, new = _counts(case, 1)
    live = [(s, t) for s, t in zip(before, new) if s >= 0]
    if case["op"] == "append":
        count = sum(t for _, t in live)
        return {"bytes": 2 * size * dim * (heads + 2 * kv_heads) * count,
                "flops": 3 * case["rotated"] * (heads + kv_heads) * count}
    window, sinks = case["window"] or 1 << 40, case["sinks"]
    pairs = held = 0
    for s, t in live:
        low = max(0, s - window + 1)  # of the first query: no later one sees below
        held += s + t - low + min(sinks, low)
        p = torch.arange(s, s + t, dtype=torch.int64)
        first = (p - window + 1).clamp(min=0)
        pairs += int((p + 1 - first + first.clamp(max=sinks)).sum())
    if not case["window"]:
        held -= (len(live) - 1) * case["shared"]
    return {"bytes": size * dim * (2 * held * kv_heads + 2 * case["batch"] * tokens * heads),
            "flops": 4 * dim * heads * pairs}


# -- the definition in 64 bits -------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "rotate":
            return _exact_rotate(case, state)
        if case["op"] == "append":
            return _exact_append(case, state)
        return _exact_attend(case, state)


def _exact_turn(x, case, position):
    """``x`` times e^(i position f) as complex numbers; ``position`` one a token."""
    frequencies, magnitude = _frequencies(case)
    angle = torch.outer(position.double(), frequencies.to(x.device))[:, None, :]
    turn = torch.polar(torch.full_like(angle, magnitude), angle)
    r, y = case["rotated"], x.double()
    if case["interleaved"]:
        pairs = y[..., :r].unflatten(-1, (-1, 2))
    else:
        pairs = y[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
    pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    done = pairs if case["interleaved"] else pairs.transpose(-1, -2)
    return torch.cat([done.flatten(-2), y[..., r:]], dim=-1)


def _exact_rotate(case, state):
    x = state["x"].detach()
    out, grad = [], []
    for b in range(case["batch"]):
        start = 0 if state["starts"] is None else int(state["starts"][b])
        position = start + torch.arange(case["tokens"], device=x.device)
        out.append(_exact_turn(x[b], case, position))
        if case["grad"]:
            # a rotation's transpose is its inverse, but for the magnitude
            grad.append(_exact_turn(state["upstream"][b], case, -position))
    if not case["grad"]:
        return torch.stack(out)
    return torch.stack(out), torch.stack(grad)


def _exact_append(case, state):
    """A sequence at a time; the values are copies, not computed."""
    q = torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    cache_k, table = state["cache_k"].double(), state["pages"].tolist()
    new = [case["tokens"]] * case["batch"] if state["lengths"] is None \
        else state["lengths"].tolist()
    for b, (start, n) in enumerate(zip(state["starts"].tolist(), new)):
        if start < 0:
            continue
        position = start + torch.arange(n, device=q.device)
        q[b, :n] = _exact_turn(state["q"][b, :n], case, position)
        k = _exact_turn(state["k"][b, :n], case, position)
        for first in range(start, start + n):
            if first % case["page"] and first != start:
                continue
            last = min((first // case["page"] + 1) * case["page"], start + n)
            cache_k[table[b][first // case["page"]],
                    first % case["page"]:first % case["page"] + last - first] = \
                k[first - start:last - start]
    return q, cache_k, None


def _exact_attend(case, state):
    """A sequence, a key head and at most 512 queries at a time."""
    group, page, window = case["heads"] // case["kv_heads"], case["page"], case["window"]
    q = state["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, start in enumerate(state["starts"].tolist()):
        if start < 0:
            continue
        n = start + case["tokens"]
        mine = state["pages"][b, :-(-n // page)].long()
        j = torch.arange(n, device=q.device)
        for h in range(case["kv_heads"]):
            k = state["cache_k"][mine, :, h].reshape(-1, case["dim"])[:n].double()
            v = state["cache_v"][mine, :, h].reshape(-1, case["dim"])[:n].double()
            heads = slice(h * group, (h + 1) * group)
            for first in range(0, case["tokens"], 512):
                rows = slice(first, min(first + 512, case["tokens"]))
                p = torch.arange(start + first, start + rows.stop, device=q.device)[:, None]
                hidden = j > p
                if window:
                    hidden |= (p - j >= window) & (j >= case["sinks"])
                s = q[b, rows, heads].double().transpose(0, 1) @ k.t() / math.sqrt(case["dim"])
                out[b, rows, heads] = (torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1)
                                       @ v).transpose(0, 1)
    return out
