"""Window attention with sinks: attention over the sparse pattern of a band and
a few dense columns.

The query at position ``p`` sees the last ``window`` keys, its own among them,
and the first ``sinks`` keys of its sequence.  As a CSR matrix that pattern
would hold ``window + sinks`` columns a row, its scores would be one value
gradient (a sampled product), its output one SpMM; here the two integers are
the pattern, and scores and probabilities exist only inside the kernels.

- :func:`window_attention`: a whole sequence, a prompt or a chunk of one, with
  derivatives in queries, keys and values;
- :func:`window_attention_step`: one token of every sequence against a ring
  cache that holds no more than what can still be seen;
- :func:`window_cache_store`: a prompt's keys and values into that cache.
"""

from __future__ import annotations

import inspect
import operator

import torch
from torch.autograd import forward_ad

import mlx_sparse._native as _native
from mlx_sparse._autograd import _call
from mlx_sparse._device import default_device_index, default_torch_device
from mlx_sparse._ext_loader import extension
from mlx_sparse._validation import ensure_array

_REAL = (torch.float32, torch.float16, torch.bfloat16)
_INDEX = {torch.int32, torch.int64}


def _span(name: str, window, sinks) -> tuple[int, int]:
    window, sinks = operator.index(window), operator.index(sinks)
    if window < 1:
        raise ValueError(f"{name} window must be at least 1, got {window}.")
    if sinks < 0:
        raise ValueError(f"{name} sinks must be non-negative, got {sinks}.")
    # no sequence is as long: wider spans are the same pattern
    return min(window, 2**40), min(sinks, 2**40)


def _operand(value, device) -> torch.Tensor:
    """On ``device``, its own values in memory, the last dimension adjacent."""
    t = ensure_array(value, device=device)
    if t.is_neg():
        t = t.resolve_neg()
    if t.ndim and t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t


def _counts(value, device) -> torch.Tensor | None:
    return None if value is None else ensure_array(value, device=device).contiguous()


def _check_dtypes(name: str, q: torch.Tensor, **others: torch.Tensor) -> None:
    if q.dtype not in _REAL:
        raise TypeError(f"{name} supports float32, float16 and bfloat16, got {q.dtype}.")
    for other, t in others.items():
        if t.dtype != q.dtype:
            raise TypeError(f"{name} requires one dtype for all operands, got {q.dtype} and "
                            f"{other} of {t.dtype}.")


def _check_heads(name: str, heads: int, kv_heads: int, dim: int) -> None:
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{name} query heads ({heads}) must be a multiple of the key and value "
                         f"heads ({kv_heads}).")
    if not 1 <= dim <= 256:
        raise ValueError(f"{name} head dimension must be between 1 and 256, got {dim}.")


def _scale(scale, dim: int) -> float:
    return dim ** -0.5 if scale is None else float(scale)


def _transformed() -> bool:
    """A torch.func transform or a forward-mode level is active."""
    return torch._C._are_functorch_transforms_active() or forward_ad._current_level >= 0


def _refuse_transforms(name: str, *operands) -> None:
    """For calls that write in place and have no derivative."""
    for t in operands:
        if not isinstance(t, torch.Tensor):
            continue
        if torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise NotImplementedError(f"{name} does not support torch.func transforms of its "
                                      "operands.")
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has no forward-mode derivative.")


def _folded(t: torch.Tensor, dim: int | None, n: int) -> torch.Tensor:
    """The mapped axis joins the batch."""
    t = t.unsqueeze(0).expand(n, *t.shape) if dim is None else t.movedim(dim, 0)
    return t.reshape(n * t.shape[1], *t.shape[2:])


def _unfolded(outputs, n: int) -> tuple:
    return tuple(t if t is None else t.unflatten(0, (n, t.shape[0] // n)) for t in outputs)


class _WindowAttention(torch.autograd.Function):
    """``(out, lse, low)``; the last two are the backward pass's and have no
    derivative (``low``: what rounding left of a 16-bit ``out``, else None).
    Takes the calls under a transform; others have a node of the native
    module's, whose backward pass does not enter the interpreter."""

    @staticmethod
    def forward(q, k, v, lengths, window, sinks, scale):
        return _native.window_attention(q, k, v, lengths, window, sinks, scale, True)

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, v, lengths, window, sinks, scale = inputs
        out, lse, low = output
        ctx.mark_non_differentiable(*(t for t in (lse, low) if t is not None))
        ctx.set_materialize_grads(False)
        ctx.pattern = (window, sinks, scale)
        ctx.save_for_backward(q, k, v, lengths, out, lse, low)

    @staticmethod
    def backward(ctx, grad, *_):
        if grad is None:
            return (None,) * 7
        got = _call(_WindowGradients, *ctx.saved_tensors, grad, *ctx.pattern)
        return (*(g if needed else None for g, needed in zip(got, ctx.needs_input_grad)),
                None, None, None, None)

    @staticmethod
    def vmap(info, in_dims, q, k, v, lengths, window, sinks, scale):
        n = info.batch_size
        q, k, v = (_folded(t, d, n) for t, d in zip((q, k, v), in_dims))
        if lengths is not None:
            lengths = _folded(lengths, in_dims[3], n).contiguous()
        got = _WindowAttention.apply(q, k, v, lengths, window, sinks, scale)
        return _unfolded(got, n), tuple(t if t is None else 0 for t in got)


class _WindowGradients(torch.autograd.Function):
    """``(dq, dk, dv)``; no derivative of their own."""

    @staticmethod
    def forward(q, k, v, lengths, out, lse, low, grad, window, sinks, scale):
        return _native.window_attention_backward(q, k, v, lengths, out, lse, low,
                                                 _operand(grad, grad.device), window, sinks, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("second-order derivatives of window_attention are not supported.")

    @staticmethod
    def vmap(info, in_dims, q, k, v, lengths, out, lse, low, grad, window, sinks, scale):
        n = info.batch_size
        q, k, v, grad = (_folded(t, d, n) for t, d in zip((q, k, v, grad), (*in_dims[:3], in_dims[7])))
        lengths, out, lse, low = (
            t if t is None else _folded(t, d, n).contiguous()
            for t, d in zip((lengths, out, lse, low), in_dims[3:7]))
        got = _WindowGradients.apply(q, k, v, lengths, out, lse, low, grad, window, sinks, scale)
        return _unfolded(got, n), (0, 0, 0)


for _function in (_WindowAttention, _WindowGradients):
    _function.forward.__signature__ = inspect.signature(_function.forward)


def window_attention(q, k, v, *, window: int, sinks: int = 0, scale: float | None = None,
                     lengths=None) -> torch.Tensor:
    """Attention of every query over the last ``window`` keys and the first
    ``sinks`` keys of its sequence.

    Query ``i`` stands at position ``p = i + k_tokens - q_tokens`` (a chunk of
    a prompt ends where its keys end) and sees key ``j`` where ``j <= p`` and
    either ``p - j < window`` or ``j < sinks``.  A query that sees nothing
    gives zeros.

    Args:
        q: Queries, shape ``(batch, q_tokens, heads, dim)``.
        k: Keys, shape ``(batch, k_tokens, kv_heads, dim)``; ``heads`` is a
            multiple of ``kv_heads``, and consecutive query heads share one.
        v: Values, shaped as ``k``.
        window: Keys a query sees, its own position included.
        sinks: First keys that stay visible.
        scale: Factor of the scores, ``dim ** -0.5`` by default.
        lengths: Tokens of each sequence, shape ``(batch,)``, int32 or int64:
            keys and queries at or beyond them are padding (a padding query
            gives zeros and takes no part in the gradients).

    Returns:
        Shape ``(batch, q_tokens, heads, dim)``, the dtype of ``q``.
        Differentiable once in ``q``, ``k`` and ``v``.

    Operands are float32, float16 or bfloat16, of one dtype, ``dim`` at most
    256; strides with adjacent head values whose rows start at sixteen bytes
    are read in place, others copied.  Heads above 128 do not run on the matrix
    cores yet: 60 to 100 times slower than heads of 128, 250 and more with
    gradients (the single-token step takes them as fast as any).

    Scores, softmax and sums are float32; 16-bit operands round probabilities
    to their own type for the products with values, which costs no more than
    the rounding of the result.  A call with gradients keeps 16 bits more of
    each 16-bit output for them.  Gradients are summed in a fixed order; a
    visible token that is not finite reaches those of tokens near it too.

    Raises:
        TypeError: dtypes differ or are unsupported.
        ValueError: shapes, ``window`` or ``sinks`` are out of range.
    """
    transformed = _transformed()
    if not transformed:
        out = extension().window_attention_plain(q, k, v, lengths, window, sinks, scale,
                                                 default_device_index())
        if out is not None:
            return out
    window, sinks = _span("window_attention", window, sinks)
    device = default_torch_device()
    q, k, v = _operand(q, device), _operand(k, device), _operand(v, device)
    lengths = _counts(lengths, device)
    _check_dtypes("window_attention", q, k=k, v=v)
    if q.ndim != 4 or k.ndim != 4 or v.shape != k.shape:
        raise ValueError("window_attention expects q of shape (batch, q_tokens, heads, dim) and "
                         "k and v of shape (batch, k_tokens, kv_heads, dim), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}.")
    if q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("window_attention q and k differ in batch or head dimension: "
                         f"{tuple(q.shape)} and {tuple(k.shape)}.")
    _check_heads("window_attention", q.shape[2], k.shape[2], q.shape[3])
    scale = _scale(scale, q.shape[3])
    if not transformed:
        out = extension().window_attention_plain(q, k, v, lengths, window, sinks, scale,
                                                 default_device_index())
        if out is not None:
            return out
    # (an operand that no rule above names is named by the native checks)
    return _WindowAttention.apply(q, k, v, lengths, window, sinks, scale)[0]


def _cache(name: str, cache, device) -> torch.Tensor:
    """Caches are written in place, so none is moved or copied."""
    if not isinstance(cache, torch.Tensor):
        raise TypeError(f"{name} caches must be torch tensors.")
    if cache.device != device:
        raise ValueError(f"{name} caches must be on {device}, got {cache.device}.")
    if cache.requires_grad:
        raise ValueError(f"{name} caches are updated in place and cannot require grad.")
    return cache


def window_attention_step(q, k, v, cache_k, cache_v, lengths, *, window: int, sinks: int = 0,
                          scale: float | None = None) -> torch.Tensor:
    """One token of every sequence: its key and value go into the ring cache,
    its query attends to what it sees there.

    Position ``j`` of a sequence lies in slot ``j`` while ``j < sinks`` and in
    slot ``sinks + (j - sinks) % (slots - sinks)`` from there on, so ``sinks +
    window`` slots serve a sequence of any length; a cache with a slot for
    every position never wraps.

    Args:
        q: Queries, shape ``(batch, heads, dim)``.
        k, v: The tokens' keys and values, shape ``(batch, kv_heads, dim)``.
        cache_k, cache_v: Ring caches, shape ``(batch, slots, kv_heads,
            dim)``, updated in place; on the selected device.  Rows that do not
            start at sixteen bytes (a ``dim`` of 100 float16 values) take
            slower kernels, one wave a query head.
        lengths: Tokens before this one, shape ``(batch,)``, int32 or int64
            (not changed: one counter serves the caches of all layers).  A
            negative length marks a slot of the batch without a sequence: its
            caches are left alone and it gives zeros.
        window, sinks, scale: As in :func:`window_attention`.

    Returns:
        Shape ``(batch, heads, dim)``, the dtype of ``q``.  Not
        differentiable.
    """
    name = "window_attention_step"
    if _transformed():
        _refuse_transforms(name, q, k, v, cache_k, cache_v, lengths)
    out = extension().window_attention_step_plain(q, k, v, cache_k, cache_v, lengths, window,
                                                  sinks, scale, default_device_index())
    if out is not None:
        return out
    window, sinks = _span(name, window, sinks)
    device = default_torch_device()
    q, k, v = (_operand(t, device).detach() for t in (q, k, v))
    cache_k, cache_v = _cache(name, cache_k, device), _cache(name, cache_v, device)
    lengths = _counts(lengths, device)
    if lengths is None:
        raise TypeError(f"{name} requires lengths.")
    _check_dtypes(name, q, k=k, v=v, cache_k=cache_k, cache_v=cache_v)
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape:
        raise ValueError(f"{name} expects q of shape (batch, heads, dim) and k and v of shape "
                         f"(batch, kv_heads, dim), got {tuple(q.shape)}, {tuple(k.shape)} and "
                         f"{tuple(v.shape)}.")
    _check_heads(name, q.shape[1], k.shape[1], q.shape[2])
    if cache_k.ndim == 4 and sinks + window > cache_k.shape[1]:
        raise ValueError(f"{name} cache needs at least sinks + window = {sinks + window} slots, "
                         f"got {cache_k.shape[1]}.")
    return _native.window_attention_step(q, k, v, cache_k, cache_v, lengths, window, sinks,
                                         _scale(scale, q.shape[2]))


def window_cache_store(k, v, cache_k, cache_v, *, sinks: int = 0, starts=None,
                       lengths=None) -> None:
    """A prompt's keys and values into ring caches (the layout of
    :func:`window_attention_step`): of the tokens given, those that lie among
    the first ``sinks`` positions or among the last ``slots - sinks``.

    Args:
        k, v: Shape ``(batch, tokens, kv_heads, dim)``.
        cache_k, cache_v: Shape ``(batch, slots, kv_heads, dim)``, updated in
            place.
        sinks: First positions that keep their slots.
        starts: Position of each sequence's first token here, shape
            ``(batch,)``; zero by default.
        lengths: Tokens of each sequence here, all by default.
    """
    name = "window_cache_store"
    if _transformed():
        _refuse_transforms(name, k, v, cache_k, cache_v, starts, lengths)
    _, sinks = _span(name, 1, sinks)
    device = default_torch_device()
    k, v = _operand(k, device).detach(), _operand(v, device).detach()
    cache_k, cache_v = _cache(name, cache_k, device), _cache(name, cache_v, device)
    starts, lengths = _counts(starts, device), _counts(lengths, device)
    _check_dtypes(name, k, v=v, cache_k=cache_k, cache_v=cache_v)
    if starts is not None and lengths is not None and {starts.dtype, lengths.dtype} == _INDEX:
        starts, lengths = starts.long(), lengths.long()
    _native.window_cache_store(k, v, cache_k, cache_v, starts, lengths, sinks)
