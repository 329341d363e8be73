"""Paged caches: the keys and values of sequences that grow to any length, in
pages that sequences take as they need them and may share.

A cache has the shape ``(pages, page_size, kv_heads, dim)``; row ``b`` of a page
table ``pages`` lists the pages of sequence ``b``, whose position ``j`` lies in
slot ``j % page_size`` of page ``pages[b, j // page_size]``.  Numbers outside the
cache are pages that are not there: nothing is written to them, and their keys
are not seen.

- :func:`paged_cache_append`: new tokens' keys and values, the keys (and queries
  beside them) rotated on the way;
- :func:`paged_attention`: the new tokens' attention over what is cached, one of
  them, a few, or a chunk of a prompt; a prefix that a batch shares is read once.
"""

from __future__ import annotations

import operator

import torch

import mlx_sparse._native as _native
from mlx_sparse._attention import (_INDEX, _cache, _check_dtypes, _check_heads, _counts, _operand,
                                   _refuse_transforms, _scale, _span, _transformed)
from mlx_sparse._device import default_device_index, default_torch_device
from mlx_sparse._ext_loader import extension
from mlx_sparse._rotary import Rotary, _check_rotated


def _table(name: str, pages, device) -> torch.Tensor:
    pages = _operand(pages, device)
    if pages.dtype not in _INDEX:
        raise TypeError(f"{name} pages must be int32 or int64, got {pages.dtype}.")
    if pages.ndim != 2:
        raise ValueError(f"{name} pages must have shape (batch, pages of a sequence), got "
                         f"{tuple(pages.shape)}.")
    return pages


def _one_type(starts, lengths):
    if starts is not None and lengths is not None and {starts.dtype, lengths.dtype} == _INDEX:
        return starts.long(), lengths.long()
    return starts, lengths


def paged_cache_append(k, v, cache_k, cache_v, pages, *, starts=None, lengths=None,
                       rotation: Rotary | None = None, q=None) -> torch.Tensor | None:
    """New tokens' keys and values into a paged cache.

    Token ``t`` of sequence ``b`` goes to position ``starts[b] + t``; with
    ``rotation`` its key is rotated by that position, and so is its query ``q``,
    in the same launch.

    Args:
        k, v: Shape ``(batch, tokens, kv_heads, dim)``, float32, float16 or
            bfloat16; strides with adjacent head values are read in place.
        cache_k, cache_v: Shape ``(pages, page_size, kv_heads, dim)``, updated in
            place; on the selected device.
        pages: The table, shape ``(batch, pages of a sequence)``, int32 or int64.
            Tokens whose page is not there, or that lie beyond the table, are
            dropped.
        starts: Tokens of each sequence that are cached already, shape
            ``(batch,)``, int32 or int64; zero by default.  A negative start marks
            a slot of the batch without a sequence.
        lengths: Tokens of each sequence here, all by default.
        rotation: Rotary positions of the keys (and queries); none by default.
        q: Queries, shape ``(batch, tokens, heads, dim)``; needs ``rotation``.

    Returns:
        The rotated queries (zeros for tokens that are not there), None without
        ``q``.  Not differentiable.

    The tokens of one call have to go to different places: where two sequences
    are given the same slot, each value kept there is that of either.
    """
    name = "paged_cache_append"
    if rotation is not None and not isinstance(rotation, Rotary):
        raise TypeError(f"{name} expects a Rotary, got {type(rotation).__name__}.")
    if _transformed():
        _refuse_transforms(name, k, v, cache_k, cache_v, pages, starts, lengths, q)
    ordinal = default_device_index()
    how = None if rotation is None else rotation._on(ordinal)
    done = extension().paged_cache_append_plain(k, v, cache_k, cache_v, pages, starts, lengths,
                                                how, q, ordinal)
    if done is not None:
        return done[0]
    device = default_torch_device()
    k, v = _operand(k, device).detach(), _operand(v, device).detach()
    cache_k, cache_v = _cache(name, cache_k, device), _cache(name, cache_v, device)
    starts, lengths = _one_type(_counts(starts, device), _counts(lengths, device))
    pages = _table(name, pages, device)
    _check_dtypes(name, k, v=v, cache_k=cache_k, cache_v=cache_v)
    if k.ndim != 4 or v.shape != k.shape:
        raise ValueError(f"{name} expects k and v of shape (batch, tokens, kv_heads, dim), got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}.")
    if rotation is not None:
        _check_rotated(name, rotation, k.shape[3])
    if q is not None:
        if rotation is None:
            raise ValueError(f"{name} takes q to rotate it, and has no rotation.")
        q = _operand(q, device).detach()
        _check_dtypes(name, k, queries=q)
    return _native.paged_cache_append(k, v, cache_k, cache_v, pages, starts, lengths, how, q)


def paged_attention(q, cache_k, cache_v, pages, *, starts=None, lengths=None,
                    window: int | None = None, sinks: int = 0, scale: float | None = None,
                    shared_pages: int = 0) -> torch.Tensor:
    """Attention of every sequence's last tokens over its pages.

    Query ``t`` of sequence ``b`` stands at position ``p = starts[b] + t`` and
    sees key ``j`` where ``j <= p`` and either ``p - j < window`` or ``j <
    sinks``; its own key has to be cached before
    (:func:`paged_cache_append`).  A query that sees nothing gives zeros.

    Args:
        q: Queries, shape ``(batch, tokens, heads, dim)``: one token of each
            sequence, a few drafted ones, or a chunk of a prompt.
        cache_k, cache_v: Shape ``(pages, page_size, kv_heads, dim)``; ``heads``
            is a multiple of ``kv_heads``, and consecutive query heads share
            one.  On the selected device, never copied: rows that do not start at
            sixteen bytes (a ``dim`` of 100 float16 values) take slower
            kernels, a wave a query and head.
        pages: The table, shape ``(batch, pages of a sequence)``, int32 or int64.
            Pages that no position up to the last query's needs may be anything.
            Lengths are not read on the host: how the work is cut goes by the
            table's width, so that short sequences are served fastest from a table
            that is cut to the longest (``pages[:, :n]``, no copy).
        starts: Tokens of each sequence before the first query, shape
            ``(batch,)``, int32 or int64; zero by default.  A negative start
            marks a slot of the batch without a sequence: it gives zeros.
        lengths: Queries of each sequence, all by default; those beyond give
            zeros.
        window: Keys a query sees, its own position included; all by default.
        sinks: First keys that stay visible.
        scale: Factor of the scores, ``dim ** -0.5`` by default.
        shared_pages: The first so many pages of every row of the table are the same
            (slots without a sequence, or with no query here, need not have
            them): a batch behind one long instruction.  Few queries a
            sequence then read them once for all.

    Returns:
        Shape and dtype of ``q``.  Not differentiable.

    Scores, softmax and sums are float32.  16-bit operands round the softmax's
    weights for the product with the values: to two numbers of their own type,
    so that the result has its own rounding alone, where up to 16 queries and
    heads share a kv head (17 to 32 where the tables together hold little) and
    over shared pages; to one, which adds about as much as the rounding of the result,
    where more do.  In float16 a weight below ``2**-38`` of a row's largest may
    count as nothing.
    """
    name = "paged_attention"
    if _transformed():
        _refuse_transforms(name, q, cache_k, cache_v, pages, starts, lengths)
    out = extension().paged_attention_plain(q, cache_k, cache_v, pages, starts, lengths, window,
                                            sinks, scale, shared_pages, default_device_index())
    if out is not None:
        return out
    window, sinks = _span(name, 2**40 if window is None else window, sinks)
    shared_pages = operator.index(shared_pages)
    device = default_torch_device()
    q = _operand(q, device).detach()
    for cache in (cache_k, cache_v):
        _cache(name, cache, device)
    starts, lengths = _one_type(_counts(starts, device), _counts(lengths, device))
    pages = _table(name, pages, device)
    _check_dtypes(name, q, cache_k=cache_k, cache_v=cache_v)
    if q.ndim != 4 or cache_k.ndim != 4 or cache_v.shape != cache_k.shape:
        raise ValueError(f"{name} expects q of shape (batch, tokens, heads, dim) and caches of "
                         "shape (pages, page_size, kv_heads, dim), got "
                         f"{tuple(q.shape)}, {tuple(cache_k.shape)} and {tuple(cache_v.shape)}.")
    _check_heads(name, q.shape[2], cache_k.shape[2], q.shape[3])
    if not 0 <= shared_pages <= pages.shape[1]:
        raise ValueError(f"{name} shared_pages must be between 0 and {pages.shape[1]}, the pages "
                         f"of a sequence, got {shared_pages}.")
    return _native.paged_attention(q, cache_k, cache_v, pages, starts, lengths, window, sinks,
                                   _scale(scale, q.shape[3]), shared_pages)
