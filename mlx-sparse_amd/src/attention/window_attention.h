// window_attention.h - C++ primitive layer of window attention with sinks.
#pragma once

#include "common/array_view.h"
#include "msx_sparse.h"

namespace msx {

// q (batch, lq, heads, dim), k and v (batch, lk, kv_heads, dim), lengths
// (batch) or null.  Checks ranks, dtypes, shapes and devices.
msx_window_attention_desc window_attention_desc(const ArrayView &q, const ArrayView &k,
                                                const ArrayView &v, const ArrayView *lengths,
                                                int64_t window, int64_t sinks, double scale);

// out as q, contiguous; lse (batch, heads, lq) float32, or null.
void window_attention(const msx_window_attention_desc &desc, const ArrayView &out, float *lse,
                      const ExecContext &ctx);

// grad as q with strides of its own; dq, dk, dv contiguous.
void window_attention_backward(const msx_window_attention_desc &desc, const ArrayView &out,
                               const float *lse, const ArrayView &grad, const ArrayView &dq,
                               const ArrayView &dk, const ArrayView &dv, const ExecContext &ctx);

// q (batch, heads, dim), k and v (batch, kv_heads, dim), caches (batch,
// slots, kv_heads, dim), lengths (batch).
msx_window_step_desc window_step_desc(const ArrayView &q, const ArrayView &k, const ArrayView &v,
                                      const ArrayView &cache_k, const ArrayView &cache_v,
                                      const ArrayView &lengths, int64_t window, int64_t sinks,
                                      double scale);
void window_attention_step(const msx_window_step_desc &desc, const ArrayView &out,
                           const ExecContext &ctx);

// k and v (batch, tokens, kv_heads, dim); starts and lengths (batch) or null.
void window_cache_store(const ArrayView &k, const ArrayView &v, const ArrayView &cache_k,
                        const ArrayView &cache_v, const ArrayView *starts,
                        const ArrayView *lengths, int64_t sinks, const ExecContext &ctx);

}  // namespace msx
