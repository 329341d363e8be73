// torch_view.h - torch tensors as the primitive layer sees them, for the files
// of the Python module.
#pragma once

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <pybind11/pybind11.h>

#include <string>

#include "common/array_view.h"

namespace msx {

namespace py = pybind11;

inline DType dtype_of(at::ScalarType t) {
  switch (t) {
  case at::kFloat: return DType::Float32;
  case at::kHalf: return DType::Float16;
  case at::kBFloat16: return DType::BFloat16;
  case at::kComplexFloat: return DType::Complex64;
  case at::kInt: return DType::Int32;
  case at::kLong: return DType::Int64;
  default: return DType::Other;
  }
}

// torch's spelling of a dtype, for error texts.
inline std::string dtype_name(at::ScalarType t) {
  switch (t) {
  case at::kFloat: return "float32";
  case at::kHalf: return "float16";
  case at::kBFloat16: return "bfloat16";
  case at::kComplexFloat: return "complex64";
  case at::kInt: return "int32";
  case at::kLong: return "int64";
  case at::kShort: return "int16";
  case at::kDouble: return "float64";
  case at::kComplexDouble: return "complex128";
  case at::kBool: return "bool";
  case at::kByte: return "uint8";
  case at::kChar: return "int8";
  default: return c10::toString(t);
  }
}

inline DType dtype_of(py::handle dtype) {
  if (!THPDtype_Check(dtype.ptr())) return DType::Other;
  return dtype_of(reinterpret_cast<THPDtype *>(dtype.ptr())->scalar_type);
}

inline const at::Tensor &tensor_of(py::handle t) {
  if (!THPVariable_Check(t.ptr())) throw py::type_error("mlx_sparse expects a torch tensor.");
  return THPVariable_Unpack(t.ptr());
}

inline int current_device() { return c10::hip::current_device(); }

inline int device_index(const at::Tensor &t) {
  const at::Device d = t.device();
  if (d.is_cpu()) return -1;
  if (!d.is_cuda())
    throw std::invalid_argument("mlx_sparse supports cpu and HIP (cuda) tensors only, got " +
                                c10::DeviceTypeName(d.type(), true) + ".");
  return d.has_index() ? d.index() : current_device();
}

inline ArrayView view_of(const at::Tensor &t) {
  ArrayView v;
  v.dtype_name = dtype_name(t.scalar_type());
  v.dtype = dtype_of(t.scalar_type());
  v.ndim = static_cast<int>(t.dim());
  if (v.ndim <= 4) {
    for (int i = 0; i < v.ndim; ++i) {
      v.shape[i] = t.size(i);
      v.strides[i] = t.stride(i);
    }
  }
  v.device = device_index(t);
  v.ptr = t.data_ptr();
  return v;
}

inline ArrayView view_of(py::handle t) { return view_of(tensor_of(t)); }

// The stream torch's current stream of `device` wraps.
inline void *stream_for(int device) {
  if (device < 0) return nullptr;
  const int current = current_device();
  if (current != device)
    throw std::invalid_argument("mlx_sparse: GPU operands must be on the current device (cuda:" +
                                std::to_string(current) + "), got cuda:" + std::to_string(device) + ".");
  return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream();
}

// Device scratch of one call from torch's caching allocator (the stream-ordered
// one of the C ABI gives its memory back at every synchronisation and maps it
// anew: 40 us a call), kept until the call's kernels are enqueued; torch
// orders its reuse on the current stream.
inline at::Tensor scratch_for(ExecContext &ctx, const at::Tensor &like, size_t bytes) {
  if (ctx.stream == nullptr && like.is_cpu()) return {};
  if (bytes == 0) return {};
  at::Tensor t = at::empty({static_cast<int64_t>(bytes)}, at::TensorOptions().dtype(at::kByte).device(like.device()));
  ctx.scratch = t.data_ptr();
  ctx.scratch_bytes = bytes;
  return t;
}

inline ExecContext context_for(const ArrayView &v, int n_threads) {
  ExecContext ctx;
  ctx.n_threads = n_threads;
  ctx.stream = v.device >= 0 ? stream_for(v.device) : nullptr;
  return ctx;
}

}  // namespace msx
