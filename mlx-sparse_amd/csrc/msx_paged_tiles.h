// msx_paged_tiles.h - how the matrix cores' kernels of paged attention share their
// work, and their launches.
#pragma once

#include "msx_paged.h"

namespace msx {

struct StepGrid {
  int32_t tiles;   // of sixteen queries: of a sequence and kv head
  int32_t groups;  // workgroups launched, as many as run at once
};

// Equal stretches of `work` steps: workgroup g takes [first(g), first(g + 1)).
struct StepShare {
  int64_t work, groups;
  __device__ __forceinline__ StepShare(int64_t w, int32_t launched) : work(w) {
    // two steps a wave at least: shorter stretches cost more in joining than they gain
    constexpr int64_t kLeast = 8;
    groups = max(min(w / kLeast, static_cast<int64_t>(launched)), int64_t{1});
  }
  __device__ __forceinline__ int64_t first(int64_t g) const { return work * g / groups; }
  // The workgroup that takes step x: the last whose first step is not past it.
  __device__ __forceinline__ int64_t owner(int64_t x) const { return ((x + 1) * groups - 1) / work; }
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
