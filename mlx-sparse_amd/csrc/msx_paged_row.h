// msx_paged_row.h - a query of paged attention by its definition, one wave: what
// the row kernel runs, and the tiles' kernels where a product of theirs is not
// finite, which a masked key's own infinity or NaN does too.
//
//   s_j = scale q.k_j,  out = sum_j exp(s_j) v_j / sum_j exp(s_j)
//
// in one pass over the keys with the running maximum m and sum l: a larger maximum m'
// rescales what is there by exp(m - m').
#pragma once

#include "msx_paged.h"
#include "msx_window_check.h"

#pragma clang fp contract(fast)

namespace msx {

// Query t, head h of sequence b; `q_lds`: room for a.dim floats of the wave's own.
// A lane takes a key of each 64 for the scores and head values lane, lane + 64, ...
// for the sum over them.
template <class V>
__device__ void paged_row(const PagedArgs &a, int64_t b, int32_t t, int32_t h, float *q_lds,
                          typename V::Storage *out) {
  using S = typename V::Storage;
  constexpr int kMaxPer = kWindowMaxDim / kWave;
  const int lane = threadIdx.x % kWave;
  float m = -INFINITY, l = 0.0f, o[kMaxPer] = {};
  if (t < a.length(b)) {
    const S *q = static_cast<const S *>(a.q) + b * a.qs[0] + t * a.qs[1] + h * a.qs[2];
    const S *k = static_cast<const S *>(a.k) + (h / a.group) * a.ks[2];
    const S *v = static_cast<const S *>(a.v) + (h / a.group) * a.vs[2];
    __builtin_amdgcn_wave_barrier();
    for (int d = lane; d < a.dim; d += kWave) q_lds[d] = V::widen(q[d]);
    __builtin_amdgcn_wave_barrier();
    const Keys seen = a.keys(a.start(b), t, t);
    const int32_t n = seen.count();
    for (int32_t c0 = 0; c0 < n; c0 += kWave) {
      const int32_t j = seen.key(min(c0 + lane, n - 1));
      const int32_t page = c0 + lane < n ? a.table.page(b, j) : -1, slot = a.table.slot(j);
      float s = -INFINITY;
      if (page >= 0) {
        const S *from = k + page * a.ks[0] + slot * a.ks[1];
        s = 0.0f;
        for (int d = 0; d < a.dim; ++d) s += q_lds[d] * V::widen(from[d]);
        s *= a.scale;
      }
      const float top = fmaxf(m, wave_max(s));
      const float base = top == -INFINITY ? 0.0f : top;
      const float e = page >= 0 ? exp2_fast(s - base) : 0.0f, keep = exp2_fast(m - base);
      l = l * keep + wave_sum(e);
      m = top;
#pragma unroll
      for (int r = 0; r < kMaxPer; ++r) o[r] *= keep;
      const int32_t here = min(kWave, n - c0);
      for (int32_t i = 0; i < here; ++i) {
        const int32_t from_page = __shfl(page, i);
        if (from_page < 0) continue;
        const float w = __shfl(e, i);
        const S *from = v + from_page * a.vs[0] + __shfl(slot, i) * a.vs[1];
#pragma unroll
        for (int r = 0; r < kMaxPer; ++r)
          if (lane + kWave * r < a.dim) o[r] += w * V::widen(from[lane + kWave * r]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t row = (b * a.tokens + t) * a.heads + h;
#pragma unroll
  for (int r = 0; r < kMaxPer; ++r)
    if (lane + kWave * r < a.dim) out[row * a.dim + lane + kWave * r] = V::narrow(o[r] * inv);
}

}  // namespace msx
