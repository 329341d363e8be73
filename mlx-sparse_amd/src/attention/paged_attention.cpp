// paged_attention.cpp - C++ primitive layer of rotary positions, paged caches and
// the attention over them: checks the operands, then calls the C ABI (device
// operands: the HIP entry point on ctx.stream; host operands: the native CPU one).
#include "attention/paged_attention.h"

#include <string>

#include "attention/operand_checks.h"

namespace msx {
namespace {

msx_rotation rotation_of(const RotationView &r, const ArrayView &x, const std::string &op) {
  msx_rotation out{};
  out.dim = r.turns != nullptr ? r.dim : 0;
  out.interleaved = r.interleaved;
  out.inverse = r.inverse;
  out.magnitude = r.magnitude;
  if (r.turns == nullptr) return out;
  if (r.turns->dtype_name != "float64")
    throw std::invalid_argument(op + " turns must have dtype float64, got " + r.turns->dtype_name + ".");
  require_shape(*r.turns, {r.dim / 2}, op + " turns");
  require_contiguous(*r.turns, (op + " turns").c_str());
  require_same_device({&x, r.turns}, op.c_str());
  out.turns = static_cast<const double *>(r.turns->ptr);
  return out;
}

msx_paged_cache cache_of(const CacheView &c, const ArrayView &q, const std::string &op) {
  require_rank(c.k, 4, (op + " cache_k").c_str());
  require_rank(c.pages, 2, (op + " pages").c_str());
  require_like(c.k, q, op + " cache_k");
  require_like(c.v, q, op + " cache_v");
  require_shape(c.v, {c.k.shape[0], c.k.shape[1], c.k.shape[2], c.k.shape[3]}, op + " cache_v");
  require_shape(c.k, {c.k.shape[0], c.k.shape[1], c.k.shape[2], q.shape[3]}, op + " cache_k");
  require_index_dtype(c.pages, (op + " pages").c_str());
  require_shape(c.pages, {q.shape[0], c.pages.shape[1]}, op + " pages");
  for (const ArrayView *a : {&c.k, &c.v}) require_packed(*a, op + " cache");
  require_packed(c.pages, op + " pages");
  require_same_device({&q, &c.k, &c.v, &c.pages}, op.c_str());
  msx_paged_cache out{};
  out.n_pages = c.k.shape[0];
  out.page_size = c.k.shape[1];
  out.kv_heads = c.k.shape[2];
  out.dim = c.k.shape[3];
  out.k = c.k.ptr;
  out.v = c.v.ptr;
  copy_strides(c.k, out.k_strides);
  copy_strides(c.v, out.v_strides);
  out.pages = c.pages.ptr;
  copy_strides(c.pages, &out.pages_stride);
  out.width = c.pages.shape[1];
  out.pages_itype = to_itype(c.pages.dtype);
  return out;
}

// Starts and lengths share one index type.
int32_t counts_of(const ArrayView *starts, const ArrayView *lengths, const ArrayView &q,
                  const std::string &op) {
  for (const ArrayView *a : {starts, lengths})
    if (a != nullptr) {
      require_counts(*a, q.shape[0], op + (a == starts ? " starts" : " lengths"));
      require_same_device({&q, a}, op.c_str());
    }
  if (starts != nullptr && lengths != nullptr)
    require_same_index_dtype(*starts, *lengths, (op + " starts").c_str(), (op + " lengths").c_str());
  const ArrayView *counts = starts != nullptr ? starts : lengths;
  return counts != nullptr ? to_itype(counts->dtype) : MSX_I32;
}

}  // namespace

void rotary(const ArrayView &x, const ArrayView *starts, const ArrayView *positions,
            const RotationView &rotation, const ArrayView &out, const ExecContext &ctx) {
  const std::string op = "rotary";
  require_rank(x, 4, "rotary x");
  require_real(x, op + " x");
  require_packed(x, op + " x");
  require_contiguous(out, "rotary output");
  msx_rotary_desc d{};
  d.vtype = to_vtype(x.dtype);
  d.batch = x.shape[0];
  d.tokens = x.shape[1];
  d.heads = x.shape[2];
  d.dim = x.shape[3];
  d.x = x.ptr;
  copy_strides(x, d.x_strides);
  if (starts != nullptr && positions != nullptr)
    throw std::invalid_argument("rotary takes starts or positions, not both.");
  if (positions != nullptr) {
    require_index_dtype(*positions, "rotary positions");
    require_shape(*positions, {d.batch, d.tokens}, op + " positions");
    require_same_device({&x, positions}, "rotary");
    d.itype = to_itype(positions->dtype);
    d.positions = positions->ptr;
    d.position_strides[0] = positions->strides[0];
    d.position_strides[1] = positions->strides[1];
  } else {
    d.itype = counts_of(starts, nullptr, x, op);
    d.starts = starts != nullptr ? starts->ptr : nullptr;
  }
  d.rotation = rotation_of(rotation, x, op);
  check_status(out.device >= 0 ? msx_rotary(&d, out.ptr, ctx.stream)
                               : msx_rotary_cpu(&d, out.ptr, ctx.n_threads),
               "rotary");
}

void paged_cache_append(const ArrayView &k, const ArrayView &v, const CacheView &cache,
                        const ArrayView *starts, const ArrayView *lengths,
                        const RotationView &rotation, const ArrayView *q, const ArrayView *q_out,
                        const ExecContext &ctx) {
  const std::string op = "paged_cache_append";
  require_rank(k, 4, "paged_cache_append k");
  require_real(k, op + " k");
  require_like(v, k, op + " v");
  require_shape(v, {k.shape[0], k.shape[1], k.shape[2], k.shape[3]}, op + " v");
  msx_paged_append_desc d{};
  d.cache = cache_of(cache, k, op);
  require_shape(k, {k.shape[0], k.shape[1], d.cache.kv_heads, k.shape[3]}, op + " k");
  for (const ArrayView *a : {&k, &v}) require_packed(*a, op + " operand");
  require_same_device({&k, &v}, op.c_str());
  d.vtype = to_vtype(k.dtype);
  d.itype = counts_of(starts, lengths, k, op);
  d.batch = k.shape[0];
  d.tokens = k.shape[1];
  d.k = k.ptr;
  d.v = v.ptr;
  copy_strides(k, d.k_strides);
  copy_strides(v, d.v_strides);
  if (q != nullptr) {
    require_rank(*q, 4, "paged_cache_append q");
    require_like(*q, k, op + " q");
    require_shape(*q, {k.shape[0], k.shape[1], q->shape[2], k.shape[3]}, op + " q");
    require_packed(*q, op + " q");
    require_same_device({&k, q}, op.c_str());
    require_contiguous(*q_out, "paged_cache_append output");
    d.heads = q->shape[2];
    d.q = q->ptr;
    copy_strides(*q, d.q_strides);
  }
  d.starts = starts != nullptr ? starts->ptr : nullptr;
  d.lengths = lengths != nullptr ? lengths->ptr : nullptr;
  d.rotation = rotation_of(rotation, k, op);
  void *to = q_out != nullptr ? q_out->ptr : nullptr;
  check_status(k.device >= 0 ? msx_paged_cache_append(&d, to, ctx.stream)
                             : msx_paged_cache_append_cpu(&d, to, ctx.n_threads),
               op.c_str());
}

msx_paged_attention_desc paged_attention_desc(const ArrayView &q, const CacheView &cache,
                                              const ArrayView *starts, const ArrayView *lengths,
                                              int64_t window, int64_t sinks, double scale,
                                              int64_t shared_pages) {
  const std::string op = "paged_attention";
  require_rank(q, 4, "paged_attention q");
  require_real(q, op + " q");
  require_packed(q, op + " q");
  msx_paged_attention_desc d{};
  d.cache = cache_of(cache, q, op);
  d.vtype = to_vtype(q.dtype);
  d.itype = counts_of(starts, lengths, q, op);
  d.batch = q.shape[0];
  d.tokens = q.shape[1];
  d.heads = q.shape[2];
  d.window = window;
  d.sinks = sinks;
  d.shared_pages = shared_pages;
  d.scale = scale;
  d.q = q.ptr;
  copy_strides(q, d.q_strides);
  d.starts = starts != nullptr ? starts->ptr : nullptr;
  d.lengths = lengths != nullptr ? lengths->ptr : nullptr;
  return d;
}

void paged_attention(const msx_paged_attention_desc &desc, const ArrayView &out,
                     const ExecContext &ctx) {
  require_contiguous(out, "paged_attention output");
  check_status(out.device >= 0 ? msx_paged_attention(&desc, out.ptr, ctx.scratch,
                                                     ctx.scratch_bytes, ctx.stream)
                               : msx_paged_attention_cpu(&desc, out.ptr, ctx.n_threads),
               "paged_attention");
}

}  // namespace msx
