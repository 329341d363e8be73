"""Dispatch shim to the native module (reference: mlx_sparse/_native.py:179-189,
286-296).

The reference routes to ``_ext`` or, when the extension is missing, to a
NumPy fallback.  Here there is no fallback: a missing extension raises, so a
result always comes from the HIP kernels (GPU operands) or the native CPU
path (``use_cpu()``).
"""

from __future__ import annotations

import torch

from mlx_sparse._ext_loader import extension
from mlx_sparse._typing import Shape2D


def csr_matvec(data, indices, indptr, x, shape: Shape2D, plan=None) -> torch.Tensor:
    return extension().csr_matvec(data, indices, indptr, x, shape[0], shape[1], plan=plan)


def csr_matmul(data, indices, indptr, rhs, shape: Shape2D, plan=None) -> torch.Tensor:
    return extension().csr_matmul(data, indices, indptr, rhs, shape[0], shape[1], plan=plan)


def csr_batched_matvec(data, indices, indptr, rhs, shape: Shape2D) -> torch.Tensor:
    """(reference: mlx_sparse/_native.py:218-228)"""
    return extension().csr_batched_matvec(data, indices, indptr, rhs, shape[0], shape[1])


def csr_batched_matmul(data, indices, indptr, rhs, shape: Shape2D) -> torch.Tensor:
    """(reference: mlx_sparse/_native.py:325-335)"""
    return extension().csr_batched_matmul(data, indices, indptr, rhs, shape[0], shape[1])


def csr_transpose(data, indices, indptr, shape: Shape2D):
    """CSR buffers of A^T, shape (n_cols, n_rows) (reference:
    mlx_sparse/_native.py:464-473)."""
    return tuple(extension().csr_transpose(data, indices, indptr, shape[0], shape[1]))


def csr_transpose_positions(indices, indptr, shape: Shape2D):
    """(t_pos, t_indices, t_indptr): the structure of A^T and, per entry, the
    position of A it holds (int32; -1 for dropped values).  GPU only."""
    return tuple(extension().csr_transpose_positions(indices, indptr, shape[0], shape[1]))


def csr_transpose_values(data, positions, conjugate: bool, out) -> None:
    """out[i] = data[positions[i]] (conjugated on request), in place.  GPU only."""
    extension().csr_transpose_values(data, positions, conjugate, out)


def csr_transpose_layout(positions, like):
    """(slot1, src1, slot2): the layout of the two-pass regather of a
    transpose's values (dtype of ``like``), from its positions."""
    return tuple(extension().csr_transpose_layout(positions, like))


def csr_transpose_values_layout(data, layout, conjugate: bool, scratch, out) -> None:
    """``out`` = the regathered values through ``layout`` (``scratch``: as
    many values as ``data``, overwritten)."""
    slot1, src1, slot2 = layout
    extension().csr_transpose_values_layout(data, slot1, src1, slot2, conjugate, scratch, out)


def csr_matvec_transpose(data, indices, indptr, x, shape: Shape2D) -> torch.Tensor:
    """A^T x, without conjugation (reference: mlx_sparse/_native.py:260-270)."""
    return extension().csr_matvec_transpose(data, indices, indptr, x, shape[0], shape[1])


def csr_matmul_transpose(data, indices, indptr, rhs, shape: Shape2D) -> torch.Tensor:
    """A^T X, without conjugation (reference: mlx_sparse/_native.py:367-377)."""
    return extension().csr_matmul_transpose(data, indices, indptr, rhs, shape[0], shape[1])


def csr_matvec_data_vjp(indices, indptr, x, cotangent, shape: Shape2D, plan=None) -> torch.Tensor:
    """cot[row(p)] * x[col(p)] per stored value (reference:
    src/sparse/csr_matvec_data_vjp/csr_matvec_data_vjp.cpp); ``plan``: the
    matrix's GPU plan, whose panel layout (if any) serves the gather of x."""
    return extension().csr_matvec_data_vjp(indices, indptr, x, cotangent, shape[0], shape[1],
                                           plan=plan)


def csr_matmul_data_vjp(indices, indptr, rhs, cotangent, shape: Shape2D) -> torch.Tensor:
    """sum_q cot[row(p), q] * X[col(p), q] per stored value (reference:
    src/sparse/csr_matmul_data_vjp/csr_matmul_data_vjp.cpp)."""
    return extension().csr_matmul_data_vjp(indices, indptr, rhs, cotangent, shape[0], shape[1])


def csr_cg(data, indices, indptr, b, x0, shape: Shape2D, *, rtol: float, atol: float,
           maxiter: int, plan=None):
    """(x, info, residual, iterations) (reference: mlx_sparse/_native.py:883-905)."""
    return extension().csr_cg(data, indices, indptr, b, x0, shape[0], shape[1], rtol, atol,
                              maxiter, plan=plan)


def csr_pcg_jacobi(data, indices, indptr, b, x0, inv_diag, shape: Shape2D, *, rtol: float,
                   atol: float, maxiter: int, plan=None):
    """(x, info, residual, iterations) (reference: mlx_sparse/_native.py:1139-1166)."""
    return extension().csr_pcg_jacobi(data, indices, indptr, b, x0, inv_diag, shape[0], shape[1],
                                      rtol, atol, maxiter, plan=plan)


def csr_bicgstab(data, indices, indptr, b, x0, shape: Shape2D, *, rtol: float, atol: float,
                 maxiter: int, plan=None):
    """(x, info, residual, iterations) (reference: mlx_sparse/_native.py csr_bicgstab)."""
    return extension().csr_bicgstab(data, indices, indptr, b, x0, shape[0], shape[1], rtol, atol,
                                    maxiter, plan=plan)


def csr_bicgstab_jacobi(data, indices, indptr, b, x0, inv_diag, shape: Shape2D, *, rtol: float,
                        atol: float, maxiter: int, plan=None):
    """(x, info, residual, iterations) of Jacobi-preconditioned BiCGSTAB
    (reference: mlx_sparse/_native.py csr_bicgstab_jacobi)."""
    return extension().csr_bicgstab_jacobi(data, indices, indptr, b, x0, inv_diag, shape[0],
                                           shape[1], rtol, atol, maxiter, plan=plan)


def csr_minres(data, indices, indptr, b, x0, shape: Shape2D, *, rtol: float, atol: float,
               maxiter: int, shift: float = 0.0, plan=None):
    """(x, info, residual, iterations) of (A - shift I) x = b (reference:
    mlx_sparse/_native.py csr_minres)."""
    return extension().csr_minres(data, indices, indptr, b, x0, shape[0], shape[1], rtol, atol,
                                  maxiter, shift, plan=plan)


def csr_minres_jacobi(data, indices, indptr, b, x0, inv_diag, shape: Shape2D, *, rtol: float,
                      atol: float, maxiter: int, shift: float = 0.0, plan=None):
    """(x, info, residual, iterations) of Jacobi-preconditioned MINRES on
    (A - shift I) x = b (reference: mlx_sparse/_native.py csr_minres_jacobi)."""
    return extension().csr_minres_jacobi(data, indices, indptr, b, x0, inv_diag, shape[0],
                                         shape[1], rtol, atol, maxiter, shift, plan=plan)


def csr_gmres(data, indices, indptr, b, x0, shape: Shape2D, *, rtol: float, atol: float,
              restart: int, maxiter: int, plan=None):
    """(x, info, residual, iterations) of restarted GMRES (reference:
    mlx_sparse/_native.py:1505-1530 csr_gmres)."""
    return extension().csr_gmres(data, indices, indptr, b, x0, shape[0], shape[1], rtol, atol,
                                 restart, maxiter, plan=plan)


def csr_gmres_jacobi(data, indices, indptr, b, x0, inv_diag, shape: Shape2D, *, rtol: float,
                     atol: float, restart: int, maxiter: int, plan=None):
    """(x, info, residual, iterations) of Jacobi-preconditioned restarted
    GMRES (reference: mlx_sparse/_native.py csr_gmres_jacobi)."""
    return extension().csr_gmres_jacobi(data, indices, indptr, b, x0, inv_diag, shape[0],
                                        shape[1], rtol, atol, restart, maxiter, plan=plan)


def csr_plan(indptr, n_rows: int, nnz: int, block_nnz: int = 0, *, data=None, indices=None,
             n_cols: int = -1, slice_mode: int = 0, defer: bool = False):
    """Row-block plan; with ``data``/``indices`` a plan bound to the matrix,
    which may hold a reordered copy for scattered gathers (slice_mode 0 auto,
    1 off, 2 XCD column slices, 3 LDS column panels; ``defer``: auto's panels
    wait where only many products repay their build)."""
    return extension().csr_plan(indptr, n_rows, nnz, block_nnz, data=data, indices=indices,
                                n_cols=n_cols, slice_mode=slice_mode, defer=defer)


def window_attention(q, k, v, lengths, window: int, sinks: int, scale: float, with_lse: bool):
    """(out, lse, low) of attention over a band and sink columns; the last two,
    with ``with_lse``, for the backward pass (``low``, of 16-bit outputs, what
    rounding left of them)."""
    return extension().window_attention(q, k, v, lengths, window, sinks, scale, with_lse)


def window_attention_backward(q, k, v, lengths, out, lse, low, grad, window: int, sinks: int,
                              scale: float):
    """(dq, dk, dv) of window_attention."""
    return extension().window_attention_backward(q, k, v, lengths, out, lse, low, grad, window,
                                                 sinks, scale)


def window_attention_step(q, k, v, cache_k, cache_v, lengths, window: int, sinks: int,
                          scale: float) -> torch.Tensor:
    """One token of every sequence against its ring cache (updated in place)."""
    return extension().window_attention_step(q, k, v, cache_k, cache_v, lengths, window, sinks,
                                             scale)


def window_cache_store(k, v, cache_k, cache_v, starts, lengths, sinks: int) -> None:
    """A prompt's keys and values into ring caches, in place."""
    extension().window_cache_store(k, v, cache_k, cache_v, starts, lengths, sinks)


def rotary(x, starts, positions, rotation, inverse: bool) -> torch.Tensor:
    """Heads rotated by their tokens' positions, or back; ``rotation``: (turns a
    position, dim, interleaved, magnitude)."""
    return extension().rotary(x, starts, positions, rotation, inverse)


def paged_cache_append(k, v, cache_k, cache_v, pages, starts, lengths, rotation, q):
    """Keys and values into a paged cache, in place; the rotated queries, or None."""
    return extension().paged_cache_append(k, v, cache_k, cache_v, pages, starts, lengths, rotation,
                                          q)


def paged_attention(q, cache_k, cache_v, pages, starts, lengths, window: int, sinks: int,
                    scale: float, shared_pages: int) -> torch.Tensor:
    """Attention of every sequence's last tokens over its pages."""
    return extension().paged_attention(q, cache_k, cache_v, pages, starts, lengths, window, sinks,
                                       scale, shared_pages)


def distill_loss(logits, data, indices, indptr, temperature: float, with_lse: bool):
    """(losses, lse or None) against a CSR teacher's kept logits."""
    return extension().distill_loss(logits, data, indices, indptr, temperature, with_lse)


def distill_grad(logits, data, indices, indptr, weights, lse, temperature: float) -> torch.Tensor:
    """Gradient of the weighted losses in the logits."""
    return extension().distill_grad(logits, data, indices, indptr, weights, lse, temperature)


def distill_loss_grad(logits, data, indices, indptr, weights, temperature: float):
    """(losses, gradient of the weighted losses)."""
    return extension().distill_loss_grad(logits, data, indices, indptr, weights, temperature)
