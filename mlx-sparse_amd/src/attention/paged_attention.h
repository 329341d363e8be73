// paged_attention.h - C++ primitive layer of rotary positions, paged caches and the
// attention over them.
#pragma once

#include "common/array_view.h"
#include "msx_sparse.h"

namespace msx {

// How heads are rotated; `turns` (dim / 2) float64.
struct RotationView {
  int64_t dim = 0;
  bool interleaved = false, inverse = false;
  double magnitude = 1.0;
  const ArrayView *turns = nullptr;
};

// x (batch, tokens, heads, dim), starts (batch) or null, positions (batch, tokens)
// or null; out as x, contiguous.
void rotary(const ArrayView &x, const ArrayView *starts, const ArrayView *positions,
            const RotationView &rotation, const ArrayView &out, const ExecContext &ctx);

// The parts of a paged cache: caches (pages, slots, kv_heads, dim), pages (batch,
// width).
struct CacheView {
  const ArrayView &k, &v, &pages;
};

// k and v (batch, tokens, kv_heads, dim); starts and lengths (batch) or null; q
// (batch, tokens, heads, dim) and q_out as q, contiguous, or null; `rotation`
// without turns: none.
void paged_cache_append(const ArrayView &k, const ArrayView &v, const CacheView &cache,
                        const ArrayView *starts, const ArrayView *lengths,
                        const RotationView &rotation, const ArrayView *q, const ArrayView *q_out,
                        const ExecContext &ctx);

// q (batch, tokens, heads, dim); starts and lengths (batch) or null.
msx_paged_attention_desc paged_attention_desc(const ArrayView &q, const CacheView &cache,
                                              const ArrayView *starts, const ArrayView *lengths,
                                              int64_t window, int64_t sinks, double scale,
                                              int64_t shared_pages);
// out as q, contiguous.
void paged_attention(const msx_paged_attention_desc &desc, const ArrayView &out,
                     const ExecContext &ctx);

}  // namespace msx
