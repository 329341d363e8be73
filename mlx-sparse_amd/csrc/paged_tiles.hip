// paged_tiles.hip - many queries against the same pages (msx_paged_block.h), for a
// batch that shares its first pages together with the sequences' own
// (msx_paged_step.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_internal.h"
#include "msx_paged_block.h"
#include "msx_paged_step.h"

namespace msx {
namespace {

template <class V, int DP>
__global__ __launch_bounds__(kTileThreads, (PagedShape<V, DP>::kBlocks)) void paged_tiles(PagedArgs a, StepGrid grid,
                                                                                          TileParts to) {
  __shared__ __attribute__((aligned(1024))) char lds[PagedShape<V, DP>::kLds];
  __shared__ StretchLds own;
  tiles_stretch<V, DP, false>(a, grid, blockIdx.x, to, lds, own);
}

// The shared pages by the first workgroups, the sequences' own by the others: either
// alone leaves the chip waiting for its loads (64 sequences of up to 1,000 tokens behind 8,192:
// 29 and 20 us one after the other).
template <class V, int DP>
__global__ __launch_bounds__(kTileThreads, (PagedShape<V, DP>::kBlocks)) void paged_shared(
    PagedArgs a, StepGrid tiles, TileParts tiles_to, StepGrid step, TileParts step_to) {
  static_assert(kTileThreads == kStepWaves * kWave, "one launch");
  __shared__ __attribute__((aligned(1024))) char
      lds[std::max(PagedShape<V, DP>::kLds, step_lds<V, DP, kStepWaves>())];
  __shared__ StretchLds own;
  if (blockIdx.x < static_cast<uint32_t>(tiles.groups))
    tiles_stretch<V, DP, true>(a, tiles, blockIdx.x, tiles_to, lds, own);
  else
    step_stretch<V, DP>(a, step, blockIdx.x - tiles.groups, step_to, lds, own);
}

template <class V, int DP>
msx_status run(const PagedArgs &a, const StepGrid &tiles, const TileParts &tiles_to, const StepGrid *step,
               const TileParts *step_to, hipStream_t stream) {
  if (step == nullptr)
    paged_tiles<V, DP><<<tiles.groups, kTileThreads, 0, stream>>>(a, tiles, tiles_to);
  else
    paged_shared<V, DP><<<tiles.groups + step->groups, kTileThreads, 0, stream>>>(a, tiles, tiles_to, *step, *step_to);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
}

template <class V>
msx_status by_dim(const PagedArgs &a, const StepGrid &tiles, const TileParts &tiles_to, const StepGrid *step,
                  const TileParts *step_to, hipStream_t stream) {
  if (a.dim <= 32) return run<V, 32>(a, tiles, tiles_to, step, step_to, stream);
  if (a.dim <= 64) return run<V, 64>(a, tiles, tiles_to, step, step_to, stream);
  if (a.dim <= 96) return run<V, 96>(a, tiles, tiles_to, step, step_to, stream);
  if (a.dim <= 128) return run<V, 128>(a, tiles, tiles_to, step, step_to, stream);
  if constexpr (sizeof(typename V::Storage) == 2) return run<V, 256>(a, tiles, tiles_to, step, step_to, stream);
  return fail(MSX_EINVAL, "paged_attention tiles take float32 heads of 128 at most.");
}

msx_status by_type(msx_vtype vt, const PagedArgs &a, const StepGrid &tiles, const TileParts &tiles_to,
                   const StepGrid *step, const TileParts *step_to, hipStream_t stream) {
  switch (vt) {
  case MSX_F32: return by_dim<F32>(a, tiles, tiles_to, step, step_to, stream);
  case MSX_F16: return by_dim<F16>(a, tiles, tiles_to, step, step_to, stream);
  default: return by_dim<BF16>(a, tiles, tiles_to, step, step_to, stream);
  }
}

}  // namespace

msx_status launch_paged_tiles(msx_vtype vt, const PagedArgs &a, const StepGrid &grid, const TileParts &to,
                              hipStream_t stream) {
  return by_type(vt, a, grid, to, nullptr, nullptr, stream);
}

msx_status launch_paged_shared(msx_vtype vt, const PagedArgs &a, const StepGrid &tiles, const TileParts &tiles_to,
                               const StepGrid &step, const TileParts &step_to, hipStream_t stream) {
  return by_type(vt, a, tiles, tiles_to, &step, &step_to, stream);
}

}  // namespace msx
