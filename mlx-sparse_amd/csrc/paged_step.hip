// paged_step.hip - a few queries of every sequence against its pages; see
// msx_paged_step.h.
#include <hip/hip_runtime.h>

#include "msx_internal.h"
#include "msx_paged_step.h"

namespace msx {
namespace {

template <class V, int DP, int kWaves, bool kPast>
__global__ __launch_bounds__(kWaves * kWave, DP > 128 || kWaves > 4 ? 1 : 2) void paged_step(PagedArgs a, StepGrid grid,
                                                                                            TileParts to) {
  __shared__ __attribute__((aligned(16))) char lds[step_lds<V, DP, kWaves>()];
  __shared__ StretchLds own;
  step_stretch<V, DP, kWaves, kPast>(a, grid, blockIdx.x, to, lds, own);
}

template <class V, int DP>
msx_status run(const PagedArgs &a, const StepGrid &grid, const TileParts &to, hipStream_t stream) {
  if constexpr (DP <= 128) {
    if (grid.waves == 8) {
      paged_step<V, DP, 8, false><<<grid.groups, 8 * kWave, 0, stream>>>(a, grid, to);
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
    }
  }
  // (of other rows this is slower: 16-bit heads of 64 4 to 9 %, float32 of 64 5 to 9, of 256 4 to 10)
  if constexpr (DP * sizeof(typename V::Storage) <= 512 &&
                StepShape<V, DP>::kKeys * DP * sizeof(typename V::Storage) >= 8192) {
    if (grid.past) {
      paged_step<V, DP, kStepWaves, true><<<grid.groups, kStepWaves * kWave, 0, stream>>>(a, grid, to);
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
    }
  }
  paged_step<V, DP, kStepWaves, false><<<grid.groups, kStepWaves * kWave, 0, stream>>>(a, grid, to);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
}

template <class V>
msx_status by_dim(const PagedArgs &a, const StepGrid &grid, const TileParts &to, hipStream_t stream) {
  if (a.dim <= 32) return run<V, 32>(a, grid, to, stream);
  if (a.dim <= 64) return run<V, 64>(a, grid, to, stream);
  if (a.dim <= 96) return run<V, 96>(a, grid, to, stream);
  if (a.dim <= 128) return run<V, 128>(a, grid, to, stream);
  return run<V, 256>(a, grid, to, stream);
}

}  // namespace

msx_status launch_paged_step(msx_vtype vt, const PagedArgs &a, const StepGrid &grid,
                             const TileParts &to, hipStream_t stream) {
  switch (vt) {
  case MSX_F32: return by_dim<F32>(a, grid, to, stream);
  case MSX_F16: return by_dim<F16>(a, grid, to, stream);
  default: return by_dim<BF16>(a, grid, to, stream);
  }
}

}  // namespace msx
