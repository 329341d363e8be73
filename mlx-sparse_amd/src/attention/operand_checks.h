// operand_checks.h - what the attention operators ask of their operands.
#pragma once

#include <string>

#include "common/validate.h"

namespace msx {

inline void require_real(const ArrayView &a, const std::string &name) {
  if (a.dtype != DType::Float32 && a.dtype != DType::Float16 && a.dtype != DType::BFloat16)
    throw std::invalid_argument(name + " must have dtype float32, float16 or bfloat16, got " +
                                a.dtype_name + ".");
}

inline void require_like(const ArrayView &a, const ArrayView &like, const std::string &name) {
  if (a.dtype != like.dtype)
    throw std::invalid_argument(name + " must have the queries' dtype " + like.dtype_name +
                                ", got " + a.dtype_name + ".");
}

inline void require_shape(const ArrayView &a, std::initializer_list<int64_t> shape,
                          const std::string &name) {
  require_rank(a, static_cast<int>(shape.size()), name.c_str());
  std::string want, got;
  bool ok = true;
  int i = 0;
  for (int64_t s : shape) {
    ok = ok && a.shape[i] == s;
    want += (i ? ", " : "") + std::to_string(s);
    got += (i ? ", " : "") + std::to_string(a.shape[i]);
    ++i;
  }
  if (!ok)
    throw std::invalid_argument(name + " must have shape (" + want + "), got (" + got + ").");
}

// Strides of the leading dimensions; one of a single place is never used, and
// whatever it is says nothing about alignment.
inline void copy_strides(const ArrayView &a, int64_t *to) {
  for (int i = 0; i + 1 < a.ndim; ++i) to[i] = a.shape[i] > 1 ? a.strides[i] : 0;
}

// The values of a head lie side by side (an expanded tensor without values, as
// the sum of nothing hands on, counts as contiguous and keeps its strides).
inline void require_packed(const ArrayView &a, const std::string &name) {
  const int last = a.ndim - 1;
  if (a.size() > 0 && a.shape[last] > 1 && a.strides[last] != 1)
    throw std::invalid_argument(name + " must have adjacent values in its last dimension.");
}

inline void require_counts(const ArrayView &a, int64_t batch, const std::string &name) {
  require_index_dtype(a, name.c_str());
  require_shape(a, {batch}, name);
  require_contiguous(a, name.c_str());
}

}  // namespace msx
