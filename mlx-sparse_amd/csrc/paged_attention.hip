// paged_attention.hip - attention over paged caches: the entry points, and the row
// kernel that takes every type, head dimension, alignment and page size.
//
// For a query at position p (sees keys [p - window + 1, p] and [0, sinks)):
//   s_j = scale q.k_j,  out = sum_j exp(s_j) v_j / sum_j exp(s_j)
// in one pass over the keys with the running maximum m and sum l: a larger
// maximum m' rescales what is there by exp(m - m').
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_device.h"
#include "msx_internal.h"
#include "msx_paged.h"
#include "msx_paged_check.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kRowWaves = 4;
constexpr int kMaxPer = 4;  // head values a lane holds: dim <= 256

// One wave a (sequence, query, head).
template <class V>
__global__ __launch_bounds__(kRowWaves * kWave) void paged_rows(PagedArgs a, int64_t first, int64_t rows,
                                                                typename V::Storage *out) {
  using S = typename V::Storage;
  __shared__ float q_lds[kRowWaves][kWindowMaxDim];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row = first + static_cast<int64_t>(blockIdx.x) * kRowWaves + wave;
  if (row >= rows) return;  // whole waves leave; there is no barrier below
  const int32_t h = static_cast<int32_t>(row % a.heads);
  const int32_t t = static_cast<int32_t>(row / a.heads % a.tokens);
  const int64_t b = row / a.heads / a.tokens;
  float m = -INFINITY, l = 0.0f, o[kMaxPer] = {};
  if (t < a.length(b)) {
    const S *q = static_cast<const S *>(a.q) + b * a.qs[0] + t * a.qs[1] + h * a.qs[2];
    const S *k = static_cast<const S *>(a.k) + (h / a.group) * a.ks[2];
    const S *v = static_cast<const S *>(a.v) + (h / a.group) * a.vs[2];
    float *ql = q_lds[wave];
    for (int d = lane; d < a.dim; d += kWave) ql[d] = V::widen(q[d]);
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
        for (int d = 0; d < a.dim; ++d) s += ql[d] * V::widen(from[d]);
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
#pragma unroll
  for (int r = 0; r < kMaxPer; ++r)
    if (lane + kWave * r < a.dim) out[row * a.dim + lane + kWave * r] = V::narrow(o[r] * inv);
}

PagedArgs args_of(const msx_paged_attention_desc &d) {
  PagedArgs a{};
  a.batch = d.batch;
  a.tokens = static_cast<int32_t>(d.tokens);
  a.heads = static_cast<int32_t>(d.heads);
  a.kv_heads = static_cast<int32_t>(d.cache.kv_heads);
  a.group = a.heads / a.kv_heads;
  a.dim = static_cast<int32_t>(d.cache.dim);
  a.table = table_of(d.cache);
  a.window = std::min(d.window, int64_t{1} << 40);  // no sequence is as long
  a.sinks = static_cast<int32_t>(std::min<int64_t>(d.sinks, a.table.capacity));
  a.scale = static_cast<float>(d.scale * 1.44269504088896340736);
  a.starts = d.starts;
  a.lengths = d.lengths;
  a.counts64 = d.itype == MSX_I64;
  a.q = d.q;
  a.k = d.cache.k;
  a.v = d.cache.v;
  std::copy(d.q_strides, d.q_strides + 3, a.qs);
  std::copy(d.cache.k_strides, d.cache.k_strides + 3, a.ks);
  std::copy(d.cache.v_strides, d.cache.v_strides + 3, a.vs);
  return a;
}

template <class Fn>
msx_status by_vtype(int vt, Fn &&fn) {
  switch (vt) {
  case MSX_F32: return fn(F32{});
  case MSX_F16: return fn(F16{});
  default: return fn(BF16{});
  }
}

}  // namespace
}  // namespace msx

using namespace msx;

extern "C" size_t msx_paged_attention_scratch(const msx_paged_attention_desc *desc) {
  if (check_paged_attention("paged_attention", desc) != MSX_OK) return 0;
  return 0;
}

extern "C" msx_status msx_paged_attention(const msx_paged_attention_desc *desc, void *out,
                                          void *scratch, size_t scratch_bytes, void *stream) {
  clear_error();
  (void)scratch;
  (void)scratch_bytes;
  if (msx_status st = check_paged_attention("paged_attention", desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->tokens == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "paged_attention out is NULL.");
  const PagedArgs a = args_of(*desc);
  const int64_t rows = a.batch * a.tokens * a.heads;
  return by_vtype(desc->vtype, [&](auto v) {
    using V = decltype(v);
    constexpr int64_t kMost = max_blocks(kRowWaves * kWave) * kRowWaves;
    for (int64_t first = 0; first < rows; first += kMost)
      paged_rows<V><<<static_cast<unsigned>((std::min(rows - first, kMost) + kRowWaves - 1) / kRowWaves),
                      kRowWaves * kWave, 0, static_cast<hipStream_t>(stream)>>>(
          a, first, rows, static_cast<typename V::Storage *>(out));
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
  });
}
