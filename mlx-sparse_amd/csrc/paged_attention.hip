// paged_attention.hip - attention over paged caches: the entry points, and the row
// kernel that takes every type, head dimension, alignment and page size.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_device.h"
#include "msx_internal.h"
#include "msx_paged.h"
#include "msx_paged_check.h"
#include "msx_paged_row.h"
#include "msx_paged_tiles.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kRowWaves = 4;
// One wave a (sequence, query, head).
template <class V>
__global__ __launch_bounds__(kRowWaves * kWave) void paged_rows(PagedArgs a, int64_t first, int64_t rows,
                                                                typename V::Storage *out) {
  __shared__ float q_lds[kRowWaves][kWindowMaxDim];
  const int wave = threadIdx.x / kWave;
  const int64_t row = first + static_cast<int64_t>(blockIdx.x) * kRowWaves + wave;
  if (row >= rows) return;  // whole waves leave; there is no barrier below
  paged_row<V>(a, row / a.heads / a.tokens, static_cast<int32_t>(row / a.heads % a.tokens),
               static_cast<int32_t>(row % a.heads), q_lds[wave], out);
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

// Whether the tiles' kernels can read the operands: sixteen-byte rows at sixteen-byte
// strides, and queries that share a kv head that 32 bits count.
bool takes_tiles(const msx_paged_attention_desc &d) {
  const auto size = static_cast<int64_t>(value_bytes(static_cast<msx_vtype>(d.vtype)));
  const auto aligned = [&](const void *p, const int64_t *strides) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && strides[0] * size % 16 == 0 &&
           strides[1] * size % 16 == 0 && strides[2] * size % 16 == 0;
  };
  return d.cache.dim * size % 16 == 0 &&
         d.tokens * (d.heads / d.cache.kv_heads) <= kWindowIntMax - 256 && aligned(d.q, d.q_strides) &&
         aligned(d.cache.k, d.cache.k_strides) && aligned(d.cache.v, d.cache.v_strides);
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
  if (check_paged_attention("paged_attention", desc) != MSX_OK || desc->batch == 0 ||
      desc->tokens == 0 || !takes_tiles(*desc))
    return 0;
  return paged_step_scratch(args_of(*desc));
}

extern "C" msx_status msx_paged_attention(const msx_paged_attention_desc *desc, void *out,
                                          void *scratch, size_t scratch_bytes, void *stream) {
  clear_error();
  if (msx_status st = check_paged_attention("paged_attention", desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->tokens == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "paged_attention out is NULL.");
  const PagedArgs a = args_of(*desc);
  if (takes_tiles(*desc)) {
    if (scratch == nullptr || scratch_bytes < paged_step_scratch(a) ||
        reinterpret_cast<uintptr_t>(scratch) % 16 != 0)
      return fail(MSX_EINVAL, "paged_attention scratch is too small or not aligned.");
    return launch_paged_step(static_cast<msx_vtype>(desc->vtype), a, out, scratch,
                             static_cast<hipStream_t>(stream));
  }
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
