// msx_paged_tiles.h - how the matrix cores' kernels of paged attention share their
// work, and their launches.
#pragma once

#include "msx_paged.h"

namespace msx {

struct StepGrid {
  int32_t tiles;   // of sixteen queries: of a sequence and kv head
  int32_t groups;  // workgroups launched, as many as run at once
};

// 64-bit quotients take a workgroup some microseconds, those of 32 bits are free.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t by) {
  if (((x | by) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(by);
  return x / by;
}

// Equal stretches of `work`: workgroup g takes [first(g), first(g + 1)).
struct StepShare {
  int64_t groups, each, more;  // the first `more` take one more
  __device__ __forceinline__ StepShare(int64_t work, int32_t launched) {
    groups = max(min(work / kLeast, static_cast<int64_t>(launched)), int64_t{1});
    each = quotient(work, groups);
    more = work - each * groups;
  }
  __device__ __forceinline__ int64_t first(int64_t g) const { return each * g + min(g, more); }
  // The workgroup that takes x.
  __device__ __forceinline__ int64_t owner(int64_t x) const {
    const int64_t longer = more * (each + 1);
    return x < longer ? quotient(x, each + 1) : more + quotient(x - longer, each);
  }
  // a step a wave at least
  static constexpr int64_t kLeast = 4;
};

// The workgroups that a tile of queries was cut over; none (last < first) where one
// took all of it and wrote its results.
struct StepSpan {
  int32_t first, last;
};

// paged_step.hip: rows and caches at sixteen-byte addresses and strides, scratch of
// paged_step_scratch bytes.
size_t paged_step_scratch(const PagedArgs &a);
msx_status launch_paged_step(msx_vtype vt, const PagedArgs &a, void *out, void *scratch,
                             hipStream_t stream);

}  // namespace msx
