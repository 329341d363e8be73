"""Distillation from a teacher's top logits, which are a sparse matrix: row
``i`` of a ``CSRArray`` of shape ``(tokens, vocabulary)`` holds the logits
that the teacher kept for token ``i``, an empty row is a token without a
target.

With ``q`` the softmax of a student's row over the temperature ``T`` and
``p`` the softmax of the kept logits over ``T``:

    loss = T^2 sum_r p_r (ln p_r - ln q_r)      (r over the kept columns)
    gradient in the student's logits = weight T (q - p)

- :func:`distill_loss`: the rows' losses, differentiable in the logits;
- :func:`distill_value_and_grad`: losses and gradient in one call, which reads
  the logits from memory once where the derivative of :func:`distill_loss`
  reads them again.
"""

from __future__ import annotations

import inspect
import math

import torch
from torch.autograd import forward_ad

import mlx_sparse._native as _native
from mlx_sparse._autograd import _call
from mlx_sparse._csr import CSRArray
from mlx_sparse._device import default_device_index, default_torch_device
from mlx_sparse._ext_loader import extension
from mlx_sparse._validation import ensure_array

_REAL = (torch.float32, torch.float16, torch.bfloat16)


def _prepared(name: str, logits, teacher: CSRArray, temperature: float):
    """The logits as rows, the teacher's buffers beside them, T."""
    if not isinstance(teacher, CSRArray):
        raise TypeError(f"{name} expects a CSRArray teacher, got {type(teacher).__name__}.")
    device = default_torch_device()
    logits = ensure_array(logits, device=device)
    if logits.dtype not in _REAL:
        raise TypeError(f"{name} supports float32, float16 and bfloat16 logits, got "
                        f"{logits.dtype}.")
    if teacher.dtype not in _REAL:
        raise TypeError(f"{name} supports float32, float16 and bfloat16 teachers, got "
                        f"{teacher.dtype}.")
    if logits.ndim < 2:
        raise ValueError(f"{name} expects logits of shape (..., tokens, vocabulary), got "
                         f"{tuple(logits.shape)}.")
    rows = math.prod(logits.shape[:-1])
    if teacher.shape != (rows, logits.shape[-1]):
        raise ValueError(f"{name} expects a teacher of shape {(rows, logits.shape[-1])}, got "
                         f"{teacher.shape}.")
    if teacher.data.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} has no derivative in the teacher: detach its values.")
    temperature = float(temperature)
    if not (temperature > 0.0 and math.isfinite(temperature)):
        raise ValueError(f"{name} temperature must be positive and finite, got {temperature}.")
    tiny, largest = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max
    if not tiny**0.5 <= temperature <= largest**0.5:
        raise ValueError(f"{name} temperature must have a square that float32 holds, got "
                         f"{temperature}.")
    return logits, teacher.buffers(device), temperature


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """(rows, vocabulary) with adjacent columns, in place where they are."""
    z = logits if logits.ndim == 2 else logits.flatten(0, -2)
    if z.is_neg():
        z = z.resolve_neg()
    usable = (z.shape[1] < 2 or z.stride(1) == 1) and (z.shape[0] < 2 or z.stride(0) >= z.shape[1])
    return z if usable else z.contiguous()


def _mapped(t: torch.Tensor, dim: int | None, n: int) -> torch.Tensor:
    """``n`` of ``t`` one after the other along its first dimension."""
    t = t.unsqueeze(0).expand(n, *t.shape) if dim is None else t.movedim(dim, 0)
    return t.reshape(n * t.shape[1], *t.shape[2:])


def _teachers(n: int, in_dims, data, indices, indptr):
    """The CSR buffers of a teacher for ``n`` mapped students, its rows once for each."""
    if any(d is not None for d in in_dims):
        raise ValueError("distillation vmap supports batching only the logits and weights: the "
                         "teacher must be unmapped.")
    nnz = data.shape[0]
    if indptr.dtype == torch.int32 and n * nnz > torch.iinfo(torch.int32).max:
        indices, indptr = indices.long(), indptr.long()
    first = torch.arange(n, dtype=indptr.dtype, device=indptr.device)[:, None] * nnz
    # of a row that ends a student's, the next one's start is the same entry
    starts = (first + indptr[:-1]).reshape(-1)
    return data.repeat(n), indices.repeat(n), torch.cat([starts, indptr[-1:] + (n - 1) * nnz])


class _DistillLoss(torch.autograd.Function):
    """``(losses, lse)`` of rows of logits, under a transform; other calls
    have a node of the native module's."""

    @staticmethod
    def forward(z, data, indices, indptr, temperature):
        return _native.distill_loss(z, data, indices, indptr, temperature, True)

    @staticmethod
    def setup_context(ctx, inputs, output):
        z, data, indices, indptr, temperature = inputs
        ctx.temperature = temperature
        ctx.mark_non_differentiable(output[1])
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(z, data, indices, indptr, output[1])

    @staticmethod
    def backward(ctx, grad, _lse):
        if grad is None or not ctx.needs_input_grad[0]:
            return (None,) * 5
        z, data, indices, indptr, lse = ctx.saved_tensors
        return (_call(_DistillGradient, z, data, indices, indptr, grad, lse, ctx.temperature),
                None, None, None, None)

    @staticmethod
    def vmap(info, in_dims, z, data, indices, indptr, temperature):
        """The mapped students' rows are rows of one matrix."""
        n, rows = info.batch_size, indptr.shape[0] - 1
        buffers = _teachers(n, in_dims[1:4], data, indices, indptr)
        got = _DistillLoss.apply(_rows(_mapped(z, in_dims[0], n)), *buffers, temperature)
        return tuple(t.reshape(n, rows) for t in got), (0, 0)


class _DistillGradient(torch.autograd.Function):
    """The gradient in the logits; no derivative of its own."""

    @staticmethod
    def forward(z, data, indices, indptr, grad, lse, temperature):
        return _native.distill_grad(z, data, indices, indptr, grad.resolve_neg(), lse, temperature)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("second-order derivatives of distill_loss are not supported.")

    @staticmethod
    def vmap(info, in_dims, z, data, indices, indptr, grad, lse, temperature):
        n, rows = info.batch_size, indptr.shape[0] - 1
        buffers = _teachers(n, in_dims[1:4], data, indices, indptr)
        z = _rows(_mapped(z, in_dims[0], n))
        got = _DistillGradient.apply(z, *buffers, _mapped(grad, in_dims[4], n),
                                     _mapped(lse, in_dims[5], n).contiguous(), temperature)
        return got.reshape(n, rows, z.shape[1]), 0


class _DistillBoth(torch.autograd.Function):
    """``(losses, gradient)`` under a transform, which must not lose a
    derivative: there is none."""

    @staticmethod
    def forward(z, data, indices, indptr, weights, temperature):
        return _native.distill_loss_grad(z, data, indices, indptr, weights, temperature)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("derivatives of distill_value_and_grad are not supported: "
                                  "distill_loss has one.")

    @staticmethod
    def vmap(info, in_dims, z, data, indices, indptr, weights, temperature):
        n, rows = info.batch_size, indptr.shape[0] - 1
        buffers = _teachers(n, in_dims[1:4], data, indices, indptr)
        z = _rows(_mapped(z, in_dims[0], n))
        weights = None if weights is None else _mapped(weights, in_dims[4], n)
        losses, grad = _DistillBoth.apply(z, *buffers, weights, temperature)
        return (losses.reshape(n, rows), grad.reshape(n, rows, z.shape[1])), (0, 0)


for _function in (_DistillLoss, _DistillGradient, _DistillBoth):
    _function.forward.__signature__ = inspect.signature(_function.forward)


def _transformed() -> bool:
    """A torch.func transform or a forward-mode level is active."""
    return torch._C._are_functorch_transforms_active() or forward_ad._current_level >= 0


def distill_loss(logits, teacher: CSRArray, *, temperature: float = 1.0) -> torch.Tensor:
    """Per-token divergence of a student from a teacher's kept logits.

    Args:
        logits: The student's logits, shape ``(..., vocabulary)``, float32,
            float16 or bfloat16.
        teacher: ``CSRArray`` of shape ``(tokens, vocabulary)``, ``tokens`` the
            product of the leading dimensions: the teacher's kept logits (of
            any of the three dtypes), columns in any order (that of
            ``topk``, too); a column stored twice counts twice.
        temperature: Divides both sides' logits; between 1.1e-19 and 1.8e19,
            where float32 holds its square.

    Returns:
        float32 losses of shape ``logits.shape[:-1]``, ``temperature**2`` times
        the divergence; differentiable once in ``logits``.  A row without a
        kept logit (none stored, all ``-inf``) has loss and gradient zero
        whatever its logits are; so has the gradient of a row whose upstream
        gradient is zero.

    Raises:
        TypeError: ``teacher`` is not a CSRArray or a dtype is unsupported.
        ValueError: shapes or ``temperature`` do not fit.
    """
    transformed = _transformed()
    if not transformed and type(teacher) is CSRArray:
        losses = extension().distill_loss_plain(logits, teacher.data, teacher.indices,
                                                teacher.indptr, *teacher.shape, temperature,
                                                default_device_index())
        if losses is not None:
            return losses
    logits, (data, indices, indptr), temperature = _prepared("distill_loss", logits, teacher,
                                                             temperature)
    z = _rows(logits)
    losses = None
    if not transformed:
        losses = extension().distill_loss_plain(z, data, indices, indptr, *teacher.shape,
                                                temperature, default_device_index())
    if losses is None:  # (an operand that no rule above names is named by the native checks)
        losses = _DistillLoss.apply(z, data, indices, indptr, temperature)[0]
    return losses if logits.ndim == 2 else losses.reshape(logits.shape[:-1])


def distill_value_and_grad(logits, teacher: CSRArray, weights=None, *,
                           temperature: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows' losses and the gradient of their weighted sum, in one call.

    ``logits.backward(gradient)`` continues the derivative from here.

    Args:
        logits, teacher, temperature: As in :func:`distill_loss`.
        weights: Weight of each token, shape ``logits.shape[:-1]`` (a number
            for one of all); ones by default.  A row of weight zero has
            gradient zero whatever its logits are.

    Returns:
        ``(losses, gradient)``: float32 losses as :func:`distill_loss` returns
        them (not weighted), and the gradient of ``(weights * losses).sum()``,
        shaped as ``logits`` and of their dtype.
    """
    name = "distill_value_and_grad"
    transformed = _transformed()
    if not transformed and type(teacher) is CSRArray:
        both = extension().distill_loss_grad_plain(logits, teacher.data, teacher.indices,
                                                   teacher.indptr, weights, *teacher.shape,
                                                   temperature, default_device_index())
        if both is not None:
            return both
    logits, (data, indices, indptr), temperature = _prepared(name, logits, teacher, temperature)
    lead = logits.shape[:-1]
    if weights is not None:
        if not isinstance(weights, torch.Tensor):
            weights = torch.as_tensor(weights, dtype=torch.float32)
        if weights.is_complex():
            raise TypeError(f"{name} weights must be real, got {weights.dtype}.")
        if not transformed:
            weights = weights.detach()
        weights = weights.to(device=logits.device, dtype=torch.float32).resolve_neg()
        if weights.ndim == 0:
            weights = weights.expand(lead)
        if weights.shape != lead:
            raise ValueError(f"{name} weights must have shape {tuple(lead)}, got "
                             f"{tuple(weights.shape)}.")
        if weights.ndim != 1:
            weights = weights.reshape(-1)
    if transformed:
        losses, grad = _DistillBoth.apply(_rows(logits), data, indices, indptr, weights, temperature)
    else:
        losses, grad = _native.distill_loss_grad(_rows(logits.detach()), data, indices, indptr,
                                                 weights, temperature)
    if logits.ndim == 2:
        return losses, grad
    return losses.reshape(lead), grad.reshape(logits.shape)
