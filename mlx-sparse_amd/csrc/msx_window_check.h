// msx_window_check.h - argument checks of the window attention and
// distillation entry points, shared by the HIP and the host implementations.
#pragma once

#include <stdint.h>

#include <cmath>
#include <string>

#include "msx_sparse.h"

namespace msx {

msx_status fail(msx_status code, const std::string &msg);
void clear_error();

inline bool real_vtype(int vt) { return vt == MSX_F32 || vt == MSX_F16 || vt == MSX_BF16; }

constexpr int64_t kWindowMaxDim = 256;
constexpr int64_t kWindowIntMax = 2147483647;

inline msx_status check_window_heads(const char *op, int vt, int it, int64_t batch, int64_t heads,
                                     int64_t kv_heads, int64_t dim, int64_t window, int64_t sinks,
                                     double scale) {
  const std::string name(op);
  if (!real_vtype(vt))
    return fail(MSX_ETYPE, name + " requires float32, float16 or bfloat16 values.");
  if (it != MSX_I32 && it != MSX_I64)
    return fail(MSX_ETYPE, name + " requires int32 or int64 lengths.");
  if (batch < 0 || batch > kWindowIntMax)
    return fail(MSX_EINVAL, name + " batch must be non-negative and fit in int32.");
  if (heads < 1 || kv_heads < 1 || heads > 65535 || heads % kv_heads != 0)
    return fail(MSX_EINVAL, name + " heads must be a multiple of kv_heads (both at least 1).");
  if (dim < 1 || dim > kWindowMaxDim)
    return fail(MSX_EINVAL, name + " head dimension must be between 1 and 256.");
  if (window < 1) return fail(MSX_EINVAL, name + " window must be at least 1.");
  if (sinks < 0) return fail(MSX_EINVAL, name + " sinks must be non-negative.");
  // scores are float32, in base 2
  if (!std::isfinite(static_cast<float>(scale * 1.44269504088896340736)))
    return fail(MSX_EINVAL, name + " scale must be finite in float32.");
  return MSX_OK;
}

inline msx_status check_window_attention(const char *op, const msx_window_attention_desc *d) {
  const std::string name(op);
  if (d == nullptr) return fail(MSX_EINVAL, name + " descriptor is NULL.");
  if (msx_status st = check_window_heads(op, d->vtype, d->lengths_itype, d->batch, d->heads,
                                         d->kv_heads, d->dim, d->window, d->sinks, d->scale);
      st != MSX_OK)
    return st;
  if (d->lq < 0 || d->lk < 0 || d->lq > kWindowIntMax / 2 || d->lk > kWindowIntMax / 2)
    return fail(MSX_EINVAL, name + " token counts must be non-negative and below 2^30.");
  if (d->batch > 0 && d->lq > 0 && d->q == nullptr) return fail(MSX_EINVAL, name + " q is NULL.");
  if (d->batch > 0 && d->lk > 0 && (d->k == nullptr || d->v == nullptr))
    return fail(MSX_EINVAL, name + " k and v must be non-NULL.");
  return MSX_OK;
}

inline msx_status check_window_cache(const char *op, const msx_window_step_desc *d) {
  const std::string name(op);
  if (d->slots < 1 || d->slots > kWindowIntMax / 2)
    return fail(MSX_EINVAL, name + " cache slots must be at least 1 and below 2^30.");
  if (d->sinks > d->slots || d->window > d->slots - d->sinks)
    return fail(MSX_EINVAL, name + " cache needs at least sinks + window slots.");
  if (d->batch > 0 && (d->cache_k == nullptr || d->cache_v == nullptr))
    return fail(MSX_EINVAL, name + " caches must be non-NULL.");
  return MSX_OK;
}

inline msx_status check_window_step(const char *op, const msx_window_step_desc *d) {
  const std::string name(op);
  if (d == nullptr) return fail(MSX_EINVAL, name + " descriptor is NULL.");
  if (msx_status st = check_window_heads(op, d->vtype, d->lengths_itype, d->batch, d->heads,
                                         d->kv_heads, d->dim, d->window, d->sinks, d->scale);
      st != MSX_OK)
    return st;
  if (msx_status st = check_window_cache(op, d); st != MSX_OK) return st;
  if (d->batch > 0 && (d->q == nullptr || d->k == nullptr || d->v == nullptr))
    return fail(MSX_EINVAL, name + " q, k and v must be non-NULL.");
  if (d->batch > 0 && d->lengths == nullptr)
    return fail(MSX_EINVAL, name + " lengths is NULL.");
  return MSX_OK;
}

inline msx_status check_window_store(const char *op, const msx_window_step_desc *d, int64_t tokens,
                                     const void *k, const int64_t *k_strides, const void *v,
                                     const int64_t *v_strides, int it) {
  const std::string name(op);
  if (d == nullptr) return fail(MSX_EINVAL, name + " descriptor is NULL.");
  if (msx_status st = check_window_heads(op, d->vtype, it, d->batch, d->kv_heads, d->kv_heads,
                                         d->dim, 1, d->sinks, 1.0);
      st != MSX_OK)
    return st;
  if (d->slots < 1 || d->slots > kWindowIntMax / 2 || d->sinks >= d->slots)
    return fail(MSX_EINVAL, name + " cache needs at least sinks + 1 slots (and below 2^30).");
  if (tokens < 0 || tokens > kWindowIntMax / 2)
    return fail(MSX_EINVAL, name + " token count must be non-negative and below 2^30.");
  if (d->batch > 0 && tokens > 0 &&
      (k == nullptr || v == nullptr || k_strides == nullptr || v_strides == nullptr ||
       d->cache_k == nullptr || d->cache_v == nullptr))
    return fail(MSX_EINVAL, name + " buffers must be non-NULL.");
  return MSX_OK;
}

inline msx_status check_distill(const char *op, const msx_distill_desc *d) {
  const std::string name(op);
  if (d == nullptr) return fail(MSX_EINVAL, name + " descriptor is NULL.");
  if (!real_vtype(d->vtype) || !real_vtype(d->teacher_vtype))
    return fail(MSX_ETYPE, name + " requires float32, float16 or bfloat16 values.");
  if (d->itype != MSX_I32 && d->itype != MSX_I64)
    return fail(MSX_ETYPE, name + " requires int32 or int64 indices.");
  if (d->n_rows < 0 || d->n_cols < 0 || d->nnz < 0)
    return fail(MSX_EINVAL, name + " shape dimensions must be non-negative.");
  if (d->n_rows >= kWindowIntMax || d->n_cols > kWindowIntMax)
    return fail(MSX_EINVAL, name + " shape dimensions must fit in int32.");
  if (d->ld < d->n_cols)
    return fail(MSX_EINVAL, name + " leading dimension must be at least the column count.");
  if (!(d->temperature > 0.0) || !std::isfinite(d->temperature))
    return fail(MSX_EINVAL, name + " temperature must be positive and finite.");
  // losses take its square, and logits are divided by it, in float32
  if (!std::isnormal(static_cast<float>(d->temperature * d->temperature)))
    return fail(MSX_EINVAL, name + " temperature must have a square that float32 holds.");
  if (d->indptr == nullptr) return fail(MSX_EINVAL, name + " indptr is NULL.");
  if (d->nnz > 0 && (d->data == nullptr || d->indices == nullptr))
    return fail(MSX_EINVAL, name + " data and indices must be non-NULL when nnz > 0.");
  if (d->n_rows > 0 && d->n_cols > 0 && d->logits == nullptr)
    return fail(MSX_EINVAL, name + " logits is NULL.");
  return MSX_OK;
}

}  // namespace msx
