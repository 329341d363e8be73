"""mlx_sparse on MI355X: the CSR sparse x dense path of mlx-sparse
(``csr_array``, ``A @ x``, ``A @ X``), on PyTorch-ROCm tensors and
hand-written gfx950 HIP kernels behind the C ABI in ``include/msx_sparse.h``.
"""

from __future__ import annotations

from mlx_sparse import linalg, runtime
from mlx_sparse._attention import window_attention, window_attention_step, window_cache_store
from mlx_sparse._csr import CSRArray, csr_array
from mlx_sparse._device import default_torch_device, use_cpu, use_device, use_gpu
from mlx_sparse._distill import distill_loss, distill_value_and_grad
from mlx_sparse._io import from_scipy, mminfo, mmread
from mlx_sparse._ops import (
    csr_batched_matmul,
    csr_batched_matvec,
    csr_matmul,
    csr_matmul_transpose,
    csr_matvec,
    csr_matvec_transpose,
)
from mlx_sparse._paged import paged_attention, paged_cache_append
from mlx_sparse._rotary import Rotary, rotary
from mlx_sparse._typing import INDEX_DTYPES, VALUE_DTYPES, is_available


def capabilities() -> dict:
    """Compile-time facts of the native module (reference
    mlx_sparse/_capabilities.py:279-322 reports the same keys)."""
    from mlx_sparse._ext_loader import extension

    return dict(extension()._compiled_capabilities())


__all__ = [
    "CSRArray",
    "INDEX_DTYPES",
    "Rotary",
    "VALUE_DTYPES",
    "capabilities",
    "csr_array",
    "csr_batched_matmul",
    "csr_batched_matvec",
    "csr_matmul",
    "csr_matmul_transpose",
    "csr_matvec",
    "csr_matvec_transpose",
    "default_torch_device",
    "distill_loss",
    "distill_value_and_grad",
    "from_scipy",
    "is_available",
    "linalg",
    "mminfo",
    "mmread",
    "paged_attention",
    "paged_cache_append",
    "rotary",
    "runtime",
    "use_cpu",
    "use_device",
    "use_gpu",
    "window_attention",
    "window_attention_step",
    "window_cache_store",
]
