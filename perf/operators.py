"""Window attention with sinks, and distillation from a teacher's top logits:
workloads for timing the package's operators and comparing them with their
plain forms.

Each case is one pass:

- ``prompt``: ``window_attention`` over a prompt, or over a chunk of one
  whose earlier keys are there (``lk > lq``);
- ``train``: the same with its gradients in queries, keys and values;
- ``step``: ``window_attention_step``, one token of every sequence against
  its ring cache, which the pass updates;
- ``loss``: ``distill_loss``, the rows' losses alone (evaluation);
- ``grad``: ``distill_value_and_grad``, the rows' losses and the gradient of
  their weighted sum in the student's logits.

``own`` false runs the plain forms: products, sums, exponentials, indexing,
in 32 bits, rounded once at the end.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_INDEX = {"i32": torch.int32, "i64": torch.int64}


def _attention(op, batch, lq, heads, kv_heads, dim, window, sinks, dtype="bf16", *, lk=0,
               ragged=False, name=None):
    """``lk``: keys, 0 for as many as queries; ``ragged``: the sequences of
    the batch have lengths of their own, padded to ``lk``."""
    case = {"op": op, "batch": batch, "lq": lq, "lk": lk or lq, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "window": window, "sinks": sinks, "dtype": dtype,
            "ragged": ragged}
    if name:
        case["name"] = name
    return case


def _step(batch, heads, kv_heads, dim, window, sinks, dtype="bf16", *, filled="all", name=None):
    """``filled``: "all", every ring has wrapped; "ragged", sequences of
    every length from the empty one on, and slots without a sequence."""
    case = {"op": "step", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": sinks, "dtype": dtype, "filled": filled}
    if name:
        case["name"] = name
    return case


def _distill(op, rows, vocab, kept, dtype="bf16", *, teacher="f32", index="i32", temperature=1.0,
             ragged=False, name=None):
    """``kept``: the teacher's logits a row; ``ragged``: from none to twice
    as many, with rows without a target."""
    case = {"op": op, "rows": rows, "vocab": vocab, "kept": kept, "dtype": dtype,
            "teacher": teacher, "index": index, "temperature": temperature, "ragged": ragged}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # a short prompt of a small model: latency bound
        _attention("prompt", 1, 129, 8, 2, 64, 64, 4, name="prompt_small"),
        # an ordinary prompt: eight sequences to a window eight times shorter
        _attention("prompt", 1, 8192, 32, 8, 128, 1024, 4, name="prompt_8k"),
        # a chunk of a long document in f16, odd length, against the keys before it
        _attention("prompt", 1, 4099, 16, 8, 128, 4096, 16, "f16", lk=20_001, name="prompt_chunk"),
        # gradient checks and small models in full precision, ragged batch
        _attention("train", 3, 517, 6, 3, 64, 200, 0, "f32", ragged=True, name="train_small_f32"),
        # an ordinary training batch
        _attention("train", 4, 2048, 16, 4, 128, 512, 4, name="train_batch"),
        # one long sequence: the keys that all queries see against the short window
        _attention("train", 1, 16_384, 16, 8, 128, 1024, 4, name="train_long"),
        # one conversation: latency bound
        _step(1, 8, 2, 64, 256, 4, name="step_one"),
        # a serving batch of conversations of every length, odd sizes
        _step(37, 24, 8, 96, 1000, 1, "f16", filled="ragged", name="step_ragged"),
        # a large serving batch with full windows
        _step(64, 32, 8, 128, 4096, 4, name="step_batch"),
        # a small student in full precision
        _distill("grad", 65, 1009, 8, "f32", temperature=2.0, name="grad_small_f32"),
        # evaluation of a batch, odd sizes, 64-bit indices, tokens without a target
        _distill("loss", 2049, 50_001, 32, "f16", teacher="f16", index="i64", ragged=True,
                 name="loss_eval"),
        # a training batch over a large vocabulary
        _distill("grad", 4096, 131_072, 64, temperature=2.0, name="grad_large"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "train", "train", "step", "step", "loss", "grad", "grad"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    if op in ("loss", "grad"):
        vocab = _log(rng, 500, 140_000)
        rows = _log(rng, 1, min(20_000, (2e8 if op == "loss" else 4e8) / vocab))
        return _distill(op, rows, vocab, _log(rng, 1, 200), dtype,
                        teacher=rng.choice(["f32", dtype]), index=rng.choice(["i32", "i64"]),
                        temperature=rng.choice([1.0, 1.0, 2.0, 0.7]),
                        ragged=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
    dim = rng.choice([64, 64, 128, 128, 128, 32, 80, 96])
    window = _log(rng, 16, 4096)
    sinks = rng.choice([0, 1, 4, 4, 16, 100])
    if op == "step":
        most = 4e8 / (2 * (window + sinks) * kv_heads * dim)
        return _step(_log(rng, 1, max(1, min(128, most))), heads, kv_heads, dim, window, sinks,
                     dtype, filled=rng.choice(["all", "ragged"]))
    batch = rng.choice([1, 1, 2, 5])
    # products of the largest listed ones; full precision an eighth of them
    most = (1.1e11 if op == "prompt" else 3.3e10) / (8 if dtype == "f32" else 1)
    most = most / (batch * heads * dim * (window + sinks))
    lq = _log(rng, 1, max(1, min(12_000, most)))
    lk = lq + (_log(rng, 1, 8000) if op == "prompt" and rng.random() < 0.4 else 0)
    return _attention(op, batch, lq, heads, kv_heads, dim, window, sinks, dtype, lk=lk,
                      ragged=batch > 1 and rng.random() < 0.6)


# -- inputs -------------------------------------------------------------------
def _lengths(case, seed):
    """Tokens of each sequence (attention: counted; step: already there, -1
    for a slot without a sequence)."""
    gen = torch.Generator().manual_seed(seed)
    n = case["batch"]
    if case["op"] == "step":
        held = case["window"] + case["sinks"]
        if case["filled"] == "all":
            return torch.randint(held, 8 * held, (n,), generator=gen, dtype=torch.int32)
        got = torch.randint(0, 2 * held, (n,), generator=gen, dtype=torch.int32)
        got[0] = 0
        got[2::11] = -1
        return got
    return torch.randint(max(1, case["lk"] // 3), case["lk"] + 1, (n,), generator=gen,
                         dtype=torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, spread=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=dtype)).mul_(spread)

    if case["op"] in ("loss", "grad"):
        rows, vocab, kept = case["rows"], case["vocab"], min(case["kept"], case["vocab"])
        counts = torch.full((rows,), kept, device="cuda")
        if case["ragged"]:
            most = min(2 * kept, vocab)
            counts = torch.randint(0, most + 1, (rows,), generator=gen, device="cuda")
            counts[::7] = 0
        indptr = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
        indptr[1:] = counts.cumsum(0)
        nnz = int(indptr[-1])
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), counts)
        nth = torch.arange(nnz, device="cuda") - indptr[row]
        # one column in each of the row's equal parts of the vocabulary
        part = torch.rand(nnz, generator=gen, device="cuda", dtype=torch.float64)
        column = ((nth + part) * vocab / counts[row].clamp(min=1)).long()
        first = (nth * vocab + counts[row] - 1) // counts[row].clamp(min=1)
        column = torch.maximum(column, first).clamp(max=vocab - 1)
        index = _INDEX[case["index"]]
        weights = torch.full((rows,), 1.0 / rows, device="cuda")
        return {"case": case, "logits": normal(rows, vocab, spread=2.5),
                "values": torch.randn(nnz, generator=gen, device="cuda").mul_(2).add_(6)
                .to(_DTYPES[case["teacher"]]),
                "indices": column.to(index), "indptr": indptr.to(index), "weights": weights}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "step":
        slots = case["window"] + case["sinks"]
        return {"case": case, "q": normal(case["batch"], heads, dim),
                "k": normal(case["batch"], kv_heads, dim), "v": normal(case["batch"], kv_heads, dim),
                "cache_k": normal(case["batch"], slots, kv_heads, dim),
                "cache_v": normal(case["batch"], slots, kv_heads, dim),
                "lengths": _lengths(case, seed).cuda()}
    # queries, keys and values as the views of one projection, where they are as many
    lq, lk, batch = case["lq"], case["lk"], case["batch"]
    if lq == lk:
        packed = normal(batch, lq, heads + 2 * kv_heads, dim)
        q, k, v = packed.split([heads, kv_heads, kv_heads], dim=2)
    else:
        q, k, v = normal(batch, lq, heads, dim), normal(batch, lk, kv_heads, dim), \
            normal(batch, lk, kv_heads, dim)
    state = {"case": case, "q": q, "k": k, "v": v,
             "lengths": _lengths(case, seed).cuda() if case["ragged"] else None}
    if case["op"] == "train":
        state |= {"q": q.detach().requires_grad_(), "k": k.detach().requires_grad_(),
                  "v": v.detach().requires_grad_(), "upstream": normal(batch, lq, heads, dim)}
    return state


# -- one pass -----------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] in ("loss", "grad"):
        return _plain_distill(state, case["op"] == "grad")
    with torch.no_grad():
        if case["op"] == "step":
            return _plain_step(state)
        return _plain_attention(state, state.get("upstream"))


def _run_own(case, state):
    pkg = str(Path(__file__).resolve().parents[1] / "mlx-sparse_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mlx_sparse as ms

    if case["op"] in ("loss", "grad"):
        teacher = ms.CSRArray(data=state["values"], indices=state["indices"],
                              indptr=state["indptr"], shape=(case["rows"], case["vocab"]))
        if case["op"] == "loss":
            return ms.distill_loss(state["logits"], teacher, temperature=case["temperature"])
        return ms.distill_value_and_grad(state["logits"], teacher, state["weights"],
                                         temperature=case["temperature"])
    if case["op"] == "step":
        out = ms.window_attention_step(state["q"], state["k"], state["v"], state["cache_k"],
                                       state["cache_v"], state["lengths"],
                                       window=case["window"], sinks=case["sinks"])
        return out, state["cache_k"], state["cache_v"]
    q, k, v = state["q"], state["k"], state["v"]
    out = ms.window_attention(q, k, v, window=case["window"], sinks=case["sinks"],
                              lengths=state["lengths"])
    if case["op"] == "prompt":
        return out
    return (out.detach(), *torch.autograd.grad(out, (q, k, v), state["upstream"]))


def _plain_attention(state, upstream):
    """Blocks of queries against the keys that any of a block's sees: the
    first ``sinks``, and the block's own span and the window before it."""
    case, q, k, v = state["case"], state["q"], state["k"], state["v"]
    batch, lq, heads, dim = q.shape
    lk, kv_heads, window, sinks = k.shape[1], k.shape[2], case["window"], case["sinks"]
    dev, group, scale = q.device, heads // kv_heads, dim ** -0.5
    size = min(max(window, 64), lq)
    blocks = -(-lq // size)
    at = torch.arange(blocks * size, device=dev).reshape(blocks, size) + (lk - lq)
    near = at[:, :1] - window + 1 + torch.arange(window - 1 + size, device=dev)
    far = torch.arange(min(sinks, lk), device=dev).expand(blocks, -1)
    keys = torch.cat([far, near], dim=1)  # blocks x n
    # a key among the first ones counts in its own place there, not again in the window's span
    fresh = torch.cat([torch.ones_like(far, dtype=torch.bool), near >= sinks], dim=1)
    ahead = at[:, :, None] - keys[:, None, :]  # blocks x size x n
    seen = (ahead >= 0) & ((ahead < window) | (keys[:, None, :] < sinks))
    seen &= (fresh & (keys >= 0) & (keys < lk))[:, None, :] & (at < lk)[:, :, None]
    seen = seen[None].expand(batch, -1, -1, -1)
    if state["lengths"] is not None:
        n = state["lengths"].long()[:, None, None, None]
        seen = seen & (keys[None, :, None, :] < n) & (at[None, :, :, None] < n)
    seen = seen[:, :, None, None]  # batch x blocks x 1 x 1 x size x n
    place = keys.clamp(0, lk - 1)

    def blocked(t, per):  # batch x blocks x kv_heads x per * size x dim
        t = torch.nn.functional.pad(t.float(), (0, 0, 0, 0, 0, blocks * size - lq))
        t = t.reshape(batch, blocks, size, kv_heads, per, dim).permute(0, 1, 3, 4, 2, 5)
        return t.reshape(batch, blocks, kv_heads, per * size, dim)

    def whole(t):  # back to batch x lq x heads x dim
        t = t.reshape(batch, blocks, kv_heads, group, size, dim).permute(0, 1, 4, 2, 3, 5)
        return t.reshape(batch, blocks * size, heads, dim)[:, :lq]

    qb = blocked(q, group)
    kb = k.float()[:, place].permute(0, 1, 3, 2, 4).contiguous()
    vb = v.float()[:, place].permute(0, 1, 3, 2, 4).contiguous()
    s = (qb @ kb.transpose(-1, -2)).mul_(scale)
    shape = (batch, blocks, kv_heads, group, size, keys.shape[1])
    s = s.view(shape).masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill(total == 0, 1.0)).reshape(qb.shape[:-1] + (keys.shape[1],))
    ob = p @ vb
    out = whole(ob).to(q.dtype)
    if upstream is None:
        return out
    gb = blocked(upstream, group)
    dv = p.transpose(-1, -2) @ gb
    dp = gb @ vb.transpose(-1, -2)
    ds = dp.sub_((gb * ob).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = whole(ds @ kb)
    dk = ds.transpose(-1, -2) @ qb

    def gathered(t):  # the blocks' shares of each key's gradient
        t = t.permute(0, 1, 3, 2, 4).reshape(batch, -1, kv_heads, dim)
        return torch.zeros(batch, lk, kv_heads, dim, device=dev).index_add_(1, place.reshape(-1), t)

    return out, dq.to(q.dtype), gathered(dk).to(q.dtype), gathered(dv).to(q.dtype)


def _plain_step(state):
    case, q, lengths = state["case"], state["q"], state["lengths"].long()
    cache_k, cache_v = state["cache_k"], state["cache_v"]
    batch, heads, dim = q.shape
    slots, kv_heads = cache_k.shape[1:3]
    window, sinks = case["window"], case["sinks"]
    ring, dev = slots - sinks, q.device
    live = lengths >= 0

    def slot(position):
        return torch.where(position < sinks, position, sinks + (position - sinks) % ring)

    each = torch.arange(batch, device=dev)
    mine = slot(lengths.clamp(min=0))
    for cache, new in ((cache_k, state["k"]), (cache_v, state["v"])):
        cache[each, mine] = torch.where(live[:, None, None], new, cache[each, mine])
    p = lengths[:, None]
    far = torch.arange(sinks, device=dev).expand(batch, -1)
    near = p - window + 1 + torch.arange(window, device=dev)
    at = torch.cat([far, near], dim=1)
    seen = (at >= 0) & (at <= p) & torch.cat([far >= 0, near >= sinks], dim=1)
    place = slot(at.clamp(min=0))
    kb = cache_k[each[:, None], place].float().permute(0, 2, 3, 1).contiguous()
    vb = cache_v[each[:, None], place].float().permute(0, 2, 1, 3).contiguous()
    s = (q.float().view(batch, kv_heads, -1, dim) @ kb) * dim ** -0.5
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    out = (e / total.masked_fill(total == 0, 1.0)) @ vb
    return out.reshape(batch, heads, dim).to(q.dtype), cache_k, cache_v


def _plain_distill(state, with_grad):
    case, t = state["case"], state["case"]["temperature"]
    rows, nnz = case["rows"], state["values"].numel()
    dev = state["logits"].device
    z = state["logits"].float() / t
    top = z.amax(1, keepdim=True)
    log_total = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    row = torch.searchsorted(state["indptr"].long(), torch.arange(nnz, device=dev), right=True) - 1
    column = state["indices"].long()
    kept = state["values"].float() / t
    best = torch.full((rows,), -math.inf, device=dev).scatter_reduce_(0, row, kept, "amax")
    e = torch.exp(kept - best[row])
    total = torch.zeros(rows, device=dev).index_add_(0, row, e)
    log_p = kept - best[row] - torch.log(total)[row]
    p = e / total[row]
    log_q = z[row, column] - log_total[row, 0]
    losses = torch.zeros(rows, device=dev).index_add_(0, row, p * (log_p - log_q)) * (t * t)
    if not with_grad:
        return losses
    held = (state["indptr"][1:] > state["indptr"][:-1])[:, None]
    grad = torch.exp(z.sub_(log_total))
    grad.view(-1).index_add_(0, row * case["vocab"] + column, -p)
    grad.mul_(torch.where(held, state["weights"][:, None] * t, 0.0))
    return losses, grad.to(state["logits"].dtype)


# -- what a pass cannot do without ---------------------------------------------
def _pairs(case, lengths):
    """(query, key) pairs that are seen, over the batch, one head; and the
    keys that any query sees."""
    lq, lk, w, s = case["lq"], case["lk"], case["window"], case["sinks"]
    pairs = 0
    for n in lengths:
        p = torch.arange(max(0, lk - lq), min(lk, n), dtype=torch.int64)
        low = (p - w + 1).clamp(min=0)
        pairs += int((p + 1 - low + torch.minimum(low, torch.tensor(min(s, lk)))).sum())
    used = min(lk, min(lk, lq + w - 1) + s)
    return pairs, used


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] in ("loss", "grad"):
        cells = case["rows"] * case["vocab"]
        kept = case["rows"] * min(case["kept"], case["vocab"]) \
            * (_BYTES[case["teacher"]] + (8 if case["index"] == "i64" else 4))
        return {"bytes": cells * size * (2 if case["op"] == "grad" else 1) + kept + 4 * case["rows"],
                "flops": cells * (6 if case["op"] == "grad" else 4)}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "step":
        held = case["window"] + case["sinks"]
        lengths = torch.full((case["batch"],), held) if case["filled"] == "all" \
            else (_lengths(case, 1) + 1).clamp(0, held)
        seen = int(lengths.sum())
        return {"bytes": size * dim * (2 * seen * kv_heads + 2 * case["batch"] * (heads + kv_heads)),
                "flops": 4 * dim * heads * seen}
    lengths = _lengths(case, 1).tolist() if case["ragged"] else [case["lk"]] * case["batch"]
    pairs, used = _pairs(case, lengths)
    queries, keys = case["batch"] * case["lq"] * heads, case["batch"] * used * kv_heads
    train = case["op"] == "train"
    return {"bytes": size * dim * (2 * queries + 2 * keys) * (2 if train else 1),
            "flops": (14 if train else 4) * dim * heads * pairs}


# -- the definition in 64 bits -------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("loss", "grad"):
            return _exact_distill(case, state)
        if case["op"] == "step":
            return _exact_step(case, state)
        return _exact_attention(case, state)


def _exact_attention(case, state):
    """One head and at most 2,048 queries at a time against all keys."""
    q, k, v = (state[n].detach().double() for n in "qkv")
    lq, lk = case["lq"], case["lk"]
    group = case["heads"] // case["kv_heads"]
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    up = state["upstream"].double() if case["op"] == "train" else None
    key = torch.arange(lk, device=q.device)
    for b in range(case["batch"]):
        n = int(state["lengths"][b]) if state["lengths"] is not None else lk
        for first in range(0, lq, 2048):
            rows = slice(first, min(first + 2048, lq))
            p = torch.arange(rows.start, rows.stop, device=q.device)[:, None] + (lk - lq)
            hidden = (key > p) | (key >= n) | (p >= n) \
                | ((p - key >= case["window"]) & (key >= case["sinks"]))
            for h in range(case["heads"]):
                kk, vv, qq = k[b, :, h // group], v[b, :, h // group], q[b, rows, h]
                s = torch.matmul(qq, kk.t()) / math.sqrt(case["dim"])
                a = torch.softmax(s.masked_fill(hidden, -math.inf), dim=1).nan_to_num(0.0)
                out[b, rows, h] = a @ vv
                if up is not None:
                    g = up[b, rows, h]
                    dv[b, :, h // group] += a.t() @ g
                    da = g @ vv.t()
                    ds = a * (da - (a * da).sum(1, keepdim=True)) / math.sqrt(case["dim"])
                    dq[b, rows, h] = ds @ kk
                    dk[b, :, h // group] += ds.t() @ qq
    return out if up is None else (out, dq, dk, dv)


def _exact_step(case, state):
    """A slot at a time of the batch; the caches are copies, not computed."""
    window, sinks = case["window"], case["sinks"]
    ring = state["cache_k"].shape[1] - sinks
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=state["q"].device)
    for b, n in enumerate(state["lengths"].tolist()):
        if n < 0:
            continue
        at = sorted(set(range(min(sinks, n + 1))) | set(range(max(0, n - window + 1), n + 1)))
        place = torch.tensor([j if j < sinks else sinks + (j - sinks) % ring for j in at],
                             device=out.device)
        k = state["cache_k"][b, place].double()
        v = state["cache_v"][b, place].double()
        k[-1], v[-1] = state["k"][b].double(), state["v"][b].double()
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = (k * state["q"][b].double()).sum(2) / math.sqrt(case["dim"])
        out[b] = (torch.softmax(s, dim=0)[:, :, None] * v).sum(0)
    return out, None, None


def _exact_distill(case, state):
    rows, vocab, t = case["rows"], case["vocab"], case["temperature"]
    dev = state["logits"].device
    losses = torch.zeros(rows, dtype=torch.float64, device=dev)
    grad = torch.zeros(rows, vocab, dtype=torch.float64, device=dev) if case["op"] == "grad" \
        else None
    indptr = state["indptr"].long()
    many = max(1, (1 << 26) // vocab)
    for first in range(0, rows, many):
        last = min(first + many, rows)
        begin, end = int(indptr[first]), int(indptr[last])
        counts = indptr[first + 1:last + 1] - indptr[first:last]
        row = torch.repeat_interleave(torch.arange(last - first, device=dev), counts)
        column = state["indices"][begin:end].long()
        teacher = torch.full((last - first, vocab), -math.inf, dtype=torch.float64, device=dev)
        teacher[row, column] = state["values"][begin:end].double() / t
        log_p = torch.log_softmax(teacher, dim=1)[row, column]
        log_q = torch.log_softmax(state["logits"][first:last].double() / t, dim=1)
        p = log_p.exp()
        losses[first:last].index_put_((row,), p * (log_p - log_q[row, column]) * t * t,
                                      accumulate=True)
        if grad is not None:
            g = log_q.exp_()
            g[row, column] -= p
            g *= (t * state["weights"][first:last].double() * (counts > 0))[:, None]
            grad[first:last] = g
    return losses if grad is None else (losses, grad)
