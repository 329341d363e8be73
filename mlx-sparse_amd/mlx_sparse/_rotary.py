"""Rotary positions: pairs of a head's values turned by an angle that grows with
the token's position, so that a query's product with a key depends on how far
apart they are.

With ``r`` rotated values of a head and ``f_i = base ** (-2 i / r)`` radians a
position for pair ``i`` of ``r / 2``:

    (a, b) -> magnitude (a cos(p f_i) - b sin(p f_i), a sin(p f_i) + b cos(p f_i))

- :class:`Rotary`: the layout, the frequencies, what makes them longer;
- :func:`rotary`: queries and keys rotated, with derivatives of any order.

Keys on their way into a cache are rotated by
:func:`mlx_sparse.paged_cache_append`.
"""

from __future__ import annotations

import inspect
import math
import operator

import torch

import mlx_sparse._native as _native
from mlx_sparse._attention import _REAL, _counts, _folded, _operand, _transformed
from mlx_sparse._autograd import _call
from mlx_sparse._device import default_device_index, default_torch_device
from mlx_sparse._ext_loader import extension
from mlx_sparse._validation import ensure_array


class Rotary:
    """How heads are rotated.

    Args:
        dim: Leading values of a head that are rotated, even; the others stay.
        base: Of the frequencies ``base ** (-2 i / dim)``, radians a position.
        interleaved: Pairs are the values ``(2 i, 2 i + 1)``, else
            ``(i, i + dim / 2)``.
        scaling: For contexts ``factor`` times longer than those trained on:
            ``"linear"``, positions divided by ``factor``; ``"ntk"``, ``base``
            times ``factor ** (dim / (dim - 2))``, which divides the lowest
            frequency by ``factor`` and leaves the highest; ``"yarn"`` (Peng
            et al., 2023), frequencies that turn more than ``ramp[1]`` times
            within the ``trained`` positions stay, those below ``ramp[0]``
            are divided by ``factor``, those between go from one to the
            other in proportion to their turns, and ``magnitude`` is ``0.1
            ln(factor) + 1``.  (Models whose ramp goes by the pairs' numbers,
            between rounded bounds, take ``frequencies``.)
        factor: See ``scaling``.
        trained: Positions trained on ("yarn").
        ramp: Turns within them ("yarn").
        frequencies: Radians a position, shape ``(dim / 2,)``, in place of those
            above.
        magnitude: Factor of the rotated values, in place of the one above.

    The frequencies are put on the selected device when the object is made; on
    another one the first call there copies them (not while a graph is
    captured).  Like any operand the object lives until work that was given to
    other streams with it is done, and as long as a captured graph that reads it.
    """

    __slots__ = ("_dim", "_interleaved", "_magnitude", "_frequencies", "_held")

    def __init__(self, dim: int, *, base: float = 10_000.0, interleaved: bool = False,
                 scaling: str | None = None, factor: float = 1.0, trained: int | None = None,
                 ramp: tuple[float, float] = (1.0, 32.0), frequencies=None,
                 magnitude: float | None = None) -> None:
        dim = operator.index(dim)
        if dim < 2 or dim % 2 or dim > 256:
            raise ValueError(f"Rotary dim must be even, between 2 and 256, got {dim}.")
        base, factor = float(base), float(factor)
        if not (base > 0 and math.isfinite(base)):
            raise ValueError(f"Rotary base must be positive and finite, got {base}.")
        if not (factor > 0 and math.isfinite(factor)):
            raise ValueError(f"Rotary factor must be positive and finite, got {factor}.")
        if scaling not in (None, "linear", "ntk", "yarn"):
            raise ValueError("Rotary scaling must be None, 'linear', 'ntk' or 'yarn', got "
                             f"{scaling!r}.")
        if frequencies is not None:
            if scaling is not None:
                raise ValueError("Rotary takes frequencies or scaling, not both.")
            f = torch.as_tensor(frequencies).detach().to("cpu", torch.float64).contiguous().clone()
            if f.shape != (dim // 2,):
                raise ValueError(f"Rotary frequencies must have shape ({dim // 2},), got "
                                 f"{tuple(f.shape)}.")
            if not torch.isfinite(f).all():
                raise ValueError("Rotary frequencies must be finite.")
        else:
            if scaling == "ntk" and dim > 2:
                base *= factor ** (dim / (dim - 2))
            f = base ** -(torch.arange(0, dim, 2, dtype=torch.float64) / dim)
            if scaling == "linear":
                f = f / factor
            elif scaling == "yarn":
                low, high = (float(t) for t in ramp)
                if trained is None or not trained > 0:
                    raise ValueError("Rotary scaling 'yarn' needs trained, the positions trained "
                                     f"on, got {trained}.")
                if not high > low:
                    raise ValueError(f"Rotary ramp must rise, got {(low, high)}.")
                kept = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
                f = kept * f + (1 - kept) * f / factor
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0
        magnitude = float(magnitude)
        if not math.isfinite(magnitude) or abs(magnitude) > torch.finfo(torch.float32).max:
            raise ValueError(f"Rotary magnitude must be finite in float32, got {magnitude}.")
        self._dim, self._interleaved, self._magnitude = dim, bool(interleaved), magnitude
        self._frequencies = f
        self._held = {}
        self._on(default_device_index())

    @property
    def dim(self) -> int:
        return self._dim

    @property
    def interleaved(self) -> bool:
        return self._interleaved

    @property
    def magnitude(self) -> float:
        return self._magnitude

    @property
    def frequencies(self) -> torch.Tensor:
        """Radians a position, float64 on the host (a copy)."""
        return self._frequencies.clone()

    def _on(self, device: int) -> tuple:
        """(turns a position, dim, interleaved, magnitude) for a device's ordinal
        (-1: the host)."""
        held = self._held.get(device)
        if held is None:
            turns = self._frequencies / (2 * math.pi)
            if device >= 0:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError(
                        "Rotary has no frequencies on this device, and none can be copied while a "
                        "graph is captured: make it, or call it once, on the device before.")
                turns = turns.to(torch.device("cuda", device))
            held = (turns, self._dim, self._interleaved, self._magnitude)
            self._held[device] = held
        return held

    def __repr__(self) -> str:
        return (f"Rotary(dim={self._dim}, interleaved={self._interleaved}, "
                f"magnitude={self._magnitude:g})")


def _ordinal(device: torch.device) -> int:
    return -1 if device.type == "cpu" else device.index


class _Rotary(torch.autograd.Function):
    """Takes the calls under a transform; others have a node of the native
    module's, whose backward pass does not enter the interpreter."""

    @staticmethod
    def forward(x, starts, positions, rotation, inverse):
        return _native.rotary(_operand(x, x.device), starts, positions,
                              rotation._on(_ordinal(x.device)), inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, starts, positions, rotation, inverse = inputs
        ctx.set_materialize_grads(False)
        ctx.how = (rotation, inverse)
        ctx.save_for_backward(starts, positions)
        ctx.save_for_forward(starts, positions)

    @staticmethod
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 5
        rotation, inverse = ctx.how
        return (_call(_Rotary, grad, *ctx.saved_tensors, rotation, not inverse),
                None, None, None, None)

    @staticmethod
    def jvp(ctx, tangent, *_):
        if tangent is None:
            return None
        return _call(_Rotary, tangent, *ctx.saved_tensors, *ctx.how)

    @staticmethod
    def vmap(info, in_dims, x, starts, positions, rotation, inverse):
        n = info.batch_size
        x = _folded(x, in_dims[0], n)
        starts, positions = (t if t is None else _folded(t, d, n).contiguous()
                             for t, d in zip((starts, positions), in_dims[1:3]))
        out = _call(_Rotary, x, starts, positions, rotation, inverse)
        return out.unflatten(0, (n, out.shape[0] // n)), 0


_Rotary.forward.__signature__ = inspect.signature(_Rotary.forward)


def rotary(x, rotation: Rotary, *, starts=None, positions=None) -> torch.Tensor:
    """Queries or keys (or both, side by side as heads of one tensor) rotated
    by their tokens' positions.

    Args:
        x: Shape ``(batch, tokens, heads, dim)``, float32, float16 or bfloat16,
            ``dim`` at most 256; strides with adjacent head values are read in place.
        rotation: How.
        starts: Position of each sequence's first token, shape ``(batch,)``,
            int32 or int64; zero by default.
        positions: Position of each token, shape ``(batch, tokens)``, in place of
            ``starts``; read in place (rows may be expanded).

    Returns:
        Shape and dtype of ``x``, differentiable in ``x`` to any order.

    Angles are worked out in 64 bits (positions of a million lose nothing),
    products in float32, rounded once.  A backward pass is captured into a graph
    as any of torch's is: no eager graph of ``x`` may be alive meanwhile.
    """
    if not isinstance(rotation, Rotary):
        raise TypeError(f"rotary expects a Rotary, got {type(rotation).__name__}.")
    device = default_device_index()
    transformed = _transformed()
    if not transformed:
        out = extension().rotary_plain(x, starts, positions, rotation._on(device), device)
        if out is not None:
            return out
    target = default_torch_device()
    x = _operand(x, target)
    starts = _counts(starts, target)
    if positions is not None:
        positions = ensure_array(positions, device=target)
        if positions.is_neg():
            positions = positions.resolve_neg()
    if x.dtype not in _REAL:
        raise TypeError(f"rotary supports float32, float16 and bfloat16, got {x.dtype}.")
    if x.ndim != 4:
        raise ValueError("rotary expects x of shape (batch, tokens, heads, dim), got "
                         f"{tuple(x.shape)}.")
    _check_rotated("rotary", rotation, x.shape[3])
    if starts is not None and positions is not None:
        raise ValueError("rotary takes starts or positions, not both.")
    if not transformed:
        out = extension().rotary_plain(x, starts, positions, rotation._on(device), device)
        if out is not None:
            return out
    # (an operand that no rule above names is named by the native checks)
    return _Rotary.apply(x, starts, positions, rotation, False)


def _check_rotated(name: str, rotation: Rotary, dim: int) -> None:
    if not 1 <= dim <= 256:
        raise ValueError(f"{name} head dimension must be between 1 and 256, got {dim}.")
    if rotation.dim > dim:
        raise ValueError(f"{name} rotates {rotation.dim} values of a head, which has {dim}.")
