// window_attention.cpp - C++ primitive layer of window attention: checks the
// operands, then calls the C ABI (device operands: the HIP entry point on
// ctx.stream; host operands: the native CPU entry point).
#include "attention/window_attention.h"

#include <string>

#include "common/validate.h"

namespace msx {
namespace {

void require_real(const ArrayView &a, const std::string &name) {
  if (a.dtype != DType::Float32 && a.dtype != DType::Float16 && a.dtype != DType::BFloat16)
    throw std::invalid_argument(name + " must have dtype float32, float16 or bfloat16, got " +
                                a.dtype_name + ".");
}

void require_like(const ArrayView &a, const ArrayView &like, const std::string &name) {
  if (a.dtype != like.dtype)
    throw std::invalid_argument(name + " must have the queries' dtype " + like.dtype_name +
                                ", got " + a.dtype_name + ".");
}

void require_shape(const ArrayView &a, std::initializer_list<int64_t> shape,
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
void copy_strides(const ArrayView &a, int64_t *to) {
  for (int i = 0; i + 1 < a.ndim; ++i) to[i] = a.shape[i] > 1 ? a.strides[i] : 0;
}

// The values of a head lie side by side.
void require_packed(const ArrayView &a, const std::string &name) {
  const int last = a.ndim - 1;
  if (a.shape[last] > 1 && a.strides[last] != 1)
    throw std::invalid_argument(name + " must have adjacent values in its last dimension.");
}

void require_counts(const ArrayView &a, int64_t batch, const std::string &name) {
  require_index_dtype(a, name.c_str());
  require_shape(a, {batch}, name);
  require_contiguous(a, name.c_str());
}

}  // namespace

msx_window_attention_desc window_attention_desc(const ArrayView &q, const ArrayView &k,
                                                const ArrayView &v, const ArrayView *lengths,
                                                int64_t window, int64_t sinks, double scale) {
  const std::string op = "window_attention";
  require_rank(q, 4, "window_attention q");
  require_rank(k, 4, "window_attention k");
  require_real(q, op + " q");
  require_like(k, q, op + " k");
  require_like(v, q, op + " v");
  require_shape(k, {q.shape[0], k.shape[1], k.shape[2], q.shape[3]}, op + " k");
  require_shape(v, {k.shape[0], k.shape[1], k.shape[2], k.shape[3]}, op + " v");
  if (lengths != nullptr) {
    require_counts(*lengths, q.shape[0], op + " lengths");
    require_same_device({&q, &k, &v, lengths}, op.c_str());
  } else {
    require_same_device({&q, &k, &v}, op.c_str());
  }
  for (const ArrayView *a : {&q, &k, &v}) require_packed(*a, op + " operand");
  msx_window_attention_desc d{};
  d.vtype = to_vtype(q.dtype);
  d.lengths_itype = lengths != nullptr ? to_itype(lengths->dtype) : MSX_I32;
  d.batch = q.shape[0];
  d.lq = q.shape[1];
  d.lk = k.shape[1];
  d.heads = q.shape[2];
  d.kv_heads = k.shape[2];
  d.dim = q.shape[3];
  d.window = window;
  d.sinks = sinks;
  d.scale = scale;
  d.lengths = lengths != nullptr ? lengths->ptr : nullptr;
  d.q = q.ptr;
  d.k = k.ptr;
  d.v = v.ptr;
  copy_strides(q, d.q_strides);
  copy_strides(k, d.k_strides);
  copy_strides(v, d.v_strides);
  return d;
}

void window_attention(const msx_window_attention_desc &desc, const ArrayView &out, float *lse,
                      const ExecContext &ctx) {
  require_contiguous(out, "window_attention output");
  check_status(out.device >= 0 ? msx_window_attention(&desc, out.ptr, lse, ctx.scratch, ctx.scratch_bytes, ctx.stream)
                               : msx_window_attention_cpu(&desc, out.ptr, lse, ctx.n_threads),
               "window_attention");
}

void window_attention_backward(const msx_window_attention_desc &desc, const ArrayView &out,
                               const float *lse, const ArrayView &grad, const ArrayView &dq,
                               const ArrayView &dk, const ArrayView &dv, const ExecContext &ctx) {
  const std::string op = "window_attention_backward";
  require_shape(out, {desc.batch, desc.lq, desc.heads, desc.dim}, op + " out");
  require_shape(grad, {desc.batch, desc.lq, desc.heads, desc.dim}, op + " grad");
  require_like(grad, out, op + " grad");
  require_same_device({&out, &grad, &dq, &dk, &dv}, op.c_str());
  require_packed(grad, op + " grad");
  for (const ArrayView *a : {&out, &dq, &dk, &dv}) require_contiguous(*a, "window_attention_backward array");
  int64_t grad_strides[3];
  copy_strides(grad, grad_strides);
  check_status(out.device >= 0
                   ? msx_window_attention_backward(&desc, out.ptr, lse, grad.ptr, grad_strides,
                                                   dq.ptr, dk.ptr, dv.ptr, ctx.scratch,
                                                   ctx.scratch_bytes, ctx.stream)
                   : msx_window_attention_backward_cpu(&desc, out.ptr, lse, grad.ptr, grad_strides,
                                                       dq.ptr, dk.ptr, dv.ptr, ctx.n_threads),
               op.c_str());
}

msx_window_step_desc window_step_desc(const ArrayView &q, const ArrayView &k, const ArrayView &v,
                                      const ArrayView &cache_k, const ArrayView &cache_v,
                                      const ArrayView &lengths, int64_t window, int64_t sinks,
                                      double scale) {
  const std::string op = "window_attention_step";
  require_rank(q, 3, "window_attention_step q");
  require_rank(k, 3, "window_attention_step k");
  require_rank(cache_k, 4, "window_attention_step cache_k");
  require_real(q, op + " q");
  for (const ArrayView *a : {&k, &v, &cache_k, &cache_v}) require_like(*a, q, op + " operand");
  require_shape(k, {q.shape[0], k.shape[1], q.shape[2]}, op + " k");
  require_shape(v, {k.shape[0], k.shape[1], k.shape[2]}, op + " v");
  require_shape(cache_k, {k.shape[0], cache_k.shape[1], k.shape[1], k.shape[2]}, op + " cache_k");
  require_shape(cache_v, {k.shape[0], cache_k.shape[1], k.shape[1], k.shape[2]}, op + " cache_v");
  require_counts(lengths, q.shape[0], op + " lengths");
  require_same_device({&q, &k, &v, &cache_k, &cache_v, &lengths}, op.c_str());
  for (const ArrayView *a : {&q, &k, &v, &cache_k, &cache_v}) require_packed(*a, op + " operand");
  msx_window_step_desc d{};
  d.vtype = to_vtype(q.dtype);
  d.lengths_itype = to_itype(lengths.dtype);
  d.batch = q.shape[0];
  d.heads = q.shape[1];
  d.kv_heads = k.shape[1];
  d.dim = q.shape[2];
  d.slots = cache_k.shape[1];
  d.window = window;
  d.sinks = sinks;
  d.scale = scale;
  d.lengths = lengths.ptr;
  d.q = q.ptr;
  d.k = k.ptr;
  d.v = v.ptr;
  d.cache_k = cache_k.ptr;
  d.cache_v = cache_v.ptr;
  copy_strides(q, d.q_strides);
  copy_strides(k, d.k_strides);
  copy_strides(v, d.v_strides);
  copy_strides(cache_k, d.cache_k_strides);
  copy_strides(cache_v, d.cache_v_strides);
  return d;
}

void window_attention_step(const msx_window_step_desc &desc, const ArrayView &out,
                           const ExecContext &ctx) {
  require_contiguous(out, "window_attention_step output");
  check_status(out.device >= 0 ? msx_window_attention_step(&desc, out.ptr, ctx.scratch,
                                                           ctx.scratch_bytes, ctx.stream)
                               : msx_window_attention_step_cpu(&desc, out.ptr, ctx.n_threads),
               "window_attention_step");
}

void window_cache_store(const ArrayView &k, const ArrayView &v, const ArrayView &cache_k,
                        const ArrayView &cache_v, const ArrayView *starts,
                        const ArrayView *lengths, int64_t sinks, const ExecContext &ctx) {
  const std::string op = "window_cache_store";
  require_rank(k, 4, "window_cache_store k");
  require_rank(cache_k, 4, "window_cache_store cache_k");
  require_real(k, op + " k");
  for (const ArrayView *a : {&v, &cache_k, &cache_v}) require_like(*a, k, op + " operand");
  require_shape(v, {k.shape[0], k.shape[1], k.shape[2], k.shape[3]}, op + " v");
  require_shape(cache_k, {k.shape[0], cache_k.shape[1], k.shape[2], k.shape[3]}, op + " cache_k");
  require_shape(cache_v, {k.shape[0], cache_k.shape[1], k.shape[2], k.shape[3]}, op + " cache_v");
  for (const ArrayView *a : {&k, &v, &cache_k, &cache_v}) require_packed(*a, op + " operand");
  require_same_device({&k, &v, &cache_k, &cache_v}, op.c_str());
  const ArrayView *counts = starts != nullptr ? starts : lengths;
  for (const ArrayView *a : {starts, lengths})
    if (a != nullptr) {
      require_counts(*a, k.shape[0], op + (a == starts ? " starts" : " lengths"));
      require_same_device({&k, a}, op.c_str());
    }
  if (starts != nullptr && lengths != nullptr)
    require_same_index_dtype(*starts, *lengths, "window_cache_store starts",
                             "window_cache_store lengths");
  msx_window_step_desc d{};
  d.vtype = to_vtype(k.dtype);
  d.batch = k.shape[0];
  d.kv_heads = k.shape[2];
  d.dim = k.shape[3];
  d.slots = cache_k.shape[1];
  d.sinks = sinks;
  d.cache_k = cache_k.ptr;
  d.cache_v = cache_v.ptr;
  copy_strides(cache_k, d.cache_k_strides);
  copy_strides(cache_v, d.cache_v_strides);
  const msx_itype it = counts != nullptr ? to_itype(counts->dtype) : MSX_I32;
  const void *s = starts != nullptr ? starts->ptr : nullptr;
  const void *n = lengths != nullptr ? lengths->ptr : nullptr;
  check_status(k.device >= 0 ? msx_window_cache_store(&d, k.shape[1], k.ptr, k.strides, v.ptr,
                                                      v.strides, it, s, n, ctx.stream)
                             : msx_window_cache_store_cpu(&d, k.shape[1], k.ptr, k.strides, v.ptr,
                                                          v.strides, it, s, n),
               op.c_str());
}

}  // namespace msx
