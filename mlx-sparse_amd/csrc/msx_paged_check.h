// msx_paged_check.h - argument checks of rotary positions and of paged
// caches, shared by the HIP and the host implementations.
#pragma once

#include <stdint.h>

#include <cmath>
#include <string>

#include "msx_sparse.h"
#include "msx_window_check.h"

namespace msx {

inline msx_status check_rotation(const std::string &name, const msx_rotation &r, int64_t dim) {
  if (r.dim < 0 || r.dim > dim || r.dim % 2 != 0)
    return fail(MSX_EINVAL, name + " rotates an even number of values, at most the head's.");
  if (!std::isfinite(static_cast<float>(r.magnitude)))
    return fail(MSX_EINVAL, name + " magnitude must be finite in float32.");
  if (r.dim > 0 && r.turns == nullptr) return fail(MSX_EINVAL, name + " turns is NULL.");
  return MSX_OK;
}

inline msx_status check_tokens(const std::string &name, int vt, int it, int64_t batch,
                               int64_t tokens, int64_t heads, int64_t least_heads, int64_t dim) {
  if (!real_vtype(vt))
    return fail(MSX_ETYPE, name + " requires float32, float16 or bfloat16 values.");
  if (it != MSX_I32 && it != MSX_I64)
    return fail(MSX_ETYPE, name + " requires int32 or int64 positions.");
  if (batch < 0 || batch > kWindowIntMax)
    return fail(MSX_EINVAL, name + " batch must be non-negative and fit in int32.");
  if (tokens < 0 || tokens > kWindowIntMax / 2)
    return fail(MSX_EINVAL, name + " token count must be non-negative and below 2^30.");
  if (heads < least_heads || heads > 65535)
    return fail(MSX_EINVAL, name + " heads must be between " + std::to_string(least_heads) +
                                " and 65535.");
  if (dim < 1 || dim > kWindowMaxDim)
    return fail(MSX_EINVAL, name + " head dimension must be between 1 and 256.");
  return MSX_OK;
}

inline msx_status check_cache(const std::string &name, const msx_paged_cache &c, int64_t batch) {
  if (c.pages_itype != MSX_I32 && c.pages_itype != MSX_I64)
    return fail(MSX_ETYPE, name + " requires int32 or int64 pages.");
  if (c.kv_heads < 1 || c.kv_heads > 65535)
    return fail(MSX_EINVAL, name + " kv_heads must be between 1 and 65535.");
  if (c.n_pages < 0 || c.n_pages > kWindowIntMax)
    return fail(MSX_EINVAL, name + " page count must be non-negative and fit in int32.");
  if (c.page_size < 1 || c.width < 0 || c.page_size > kWindowIntMax / 2 ||
      c.width > kWindowIntMax / 2 / c.page_size)
    return fail(MSX_EINVAL, name + " pages must hold at least one token each, and a sequence's "
                                   "pages together less than 2^30.");
  if (batch > 0 && c.width > 0 && c.pages == nullptr)
    return fail(MSX_EINVAL, name + " pages is NULL.");
  if (c.n_pages > 0 && (c.k == nullptr || c.v == nullptr))
    return fail(MSX_EINVAL, name + " caches must be non-NULL.");
  return MSX_OK;
}

inline msx_status check_rotary(const char *op, const msx_rotary_desc *d) {
  const std::string name(op);
  if (d == nullptr) return fail(MSX_EINVAL, name + " descriptor is NULL.");
  if (msx_status st = check_tokens(name, d->vtype, d->itype, d->batch, d->tokens, d->heads, 0, d->dim);
      st != MSX_OK)
    return st;
  if (d->batch > 0 && d->tokens > 0 && d->heads > 0 && d->x == nullptr)
    return fail(MSX_EINVAL, name + " x is NULL.");
  return check_rotation(name, d->rotation, d->dim);
}

inline msx_status check_paged_append(const char *op, const msx_paged_append_desc *d) {
  const std::string name(op);
  if (d == nullptr) return fail(MSX_EINVAL, name + " descriptor is NULL.");
  if (msx_status st = check_tokens(name, d->vtype, d->itype, d->batch, d->tokens, d->heads, 0,
                                   d->cache.dim);
      st != MSX_OK)
    return st;
  if (msx_status st = check_cache(name, d->cache, d->batch); st != MSX_OK) return st;
  if (d->batch > 0 && d->tokens > 0 &&
      (d->k == nullptr || d->v == nullptr || (d->heads > 0 && d->q == nullptr)))
    return fail(MSX_EINVAL, name + " q, k and v must be non-NULL.");
  return check_rotation(name, d->rotation, d->cache.dim);
}

inline msx_status check_paged_attention(const char *op, const msx_paged_attention_desc *d) {
  const std::string name(op);
  if (d == nullptr) return fail(MSX_EINVAL, name + " descriptor is NULL.");
  if (msx_status st = check_tokens(name, d->vtype, d->itype, d->batch, d->tokens, d->heads, 1,
                                   d->cache.dim);
      st != MSX_OK)
    return st;
  if (msx_status st = check_window_heads(op, d->vtype, d->itype, d->batch, d->heads,
                                         d->cache.kv_heads, d->cache.dim, d->window, d->sinks,
                                         d->scale);
      st != MSX_OK)
    return st;
  if (msx_status st = check_cache(name, d->cache, d->batch); st != MSX_OK) return st;
  if (d->shared_pages < 0 || d->shared_pages > d->cache.width)
    return fail(MSX_EINVAL, name + " shared_pages must be between 0 and the table's width.");
  if (d->batch > 0 && d->tokens > 0 && d->q == nullptr)
    return fail(MSX_EINVAL, name + " q is NULL.");
  return MSX_OK;
}

}  // namespace msx
