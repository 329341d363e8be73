// bindings_operands.h - operands of the module's operators: torch tensors read in
// place, and what is asked of them.
#pragma once

#include <ATen/ops/constant_pad_nd.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/custom_function.h>

#include <optional>
#include <string>

#include "common/torch_view.h"
#include "common/validate.h"

namespace msx {

namespace py = pybind11;
using at::Tensor;

// A view of a tensor that may be absent.
struct OptionalView {
  ArrayView view;
  const ArrayView *get = nullptr;
  explicit OptionalView(const Tensor &t) {
    if (!t.defined()) return;
    view = view_of(t);
    get = &view;
  }
  OptionalView(const OptionalView &) = delete;
  OptionalView &operator=(const OptionalView &) = delete;
};

inline Tensor optional_tensor(py::handle o) { return o.is_none() ? Tensor() : tensor_of(o); }

inline Tensor new_tensor(const Tensor &like, std::initializer_list<int64_t> shape, at::ScalarType dtype) {
  return at::empty(at::IntArrayRef(shape), at::TensorOptions().dtype(dtype).device(like.device()));
}

inline py::object wrap(const Tensor &t) {
  if (!t.defined()) return py::none();
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(t));
}

// What is written in place has a place for every value.
inline void require_writable(const Tensor &t, const char *name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0)
      throw std::invalid_argument(std::string(name) +
                                  " is written in place and cannot be an expanded tensor.");
}

// A write that torch did not make: a derivative that saved the tensor, or a view
// of it, raises as after torch's own in-place operations.
inline void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Runs `fn`; without the interpreter lock where it works on the host.
template <class Fn>
inline void run_op(const ArrayView &v, Fn &&fn) {
  std::optional<py::gil_scoped_release> nogil;
  if (v.device < 0 && PyGILState_Check()) nogil.emplace();
  fn();
}

// Adjacent values in the last dimension, no lazy sign.
inline bool direct(const Tensor &t) {
  return !t.is_neg() && (t.dim() == 0 || t.size(-1) < 2 || t.stride(-1) == 1);
}
inline Tensor made_direct(const Tensor &t) {
  if (direct(t)) return t;
  return (t.is_neg() ? t.resolve_neg() : t).contiguous();
}

// Rows at sixteen-byte addresses, as the matrix cores' kernels read them; a
// dimension of one has no stride.
inline bool aligned_rows(const Tensor &t) {
  const auto size = static_cast<int64_t>(t.element_size());
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) < 2 || t.stride(i) * size % 16 == 0);
  return ok;
}
// A device operand whose layout alone would keep its call from those kernels, at
// such addresses: copying it costs a pass over it, the kernels for any layout 80
// times the others' and more (a slice of what `cat` was given, as its backward
// pass hands on, is such an operand).
constexpr int64_t kTilesDim = 128, kStepDim = 256;
inline Tensor for_tiles(const Tensor &t, int64_t most_dim) {
  const int64_t dim = t.size(-1);
  if (!t.is_cuda() || dim > most_dim || dim * static_cast<int64_t>(t.element_size()) % 16 != 0 ||
      aligned_rows(t))
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}
inline std::optional<Tensor> present(const Tensor &t) {
  return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}

inline bool on_device(const Tensor &t, int64_t device) {
  return device < 0 ? t.is_cpu() : t.is_cuda() && t.device().index() == device;
}

inline bool usable(const Tensor &t, at::ScalarType type, int64_t device) {
  return t.scalar_type() == type && on_device(t, device) && direct(t);
}

inline bool real_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

inline bool usable_counts(const Tensor &t, int64_t batch, int64_t device) {
  return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 1 &&
         t.size(0) == batch && on_device(t, device) && t.is_contiguous() && !t.is_neg();
}

}  // namespace msx
