// msx_paged_tiles.h - how the matrix cores' kernels of paged attention share their
// work, and their launches.
#pragma once

#include "msx_paged.h"
#include "msx_step_mfma.h"

namespace msx {

struct StepGrid {
  int32_t tiles;   // of queries: of a sequence and kv head
  int32_t groups;  // workgroups launched, as many as run at once
  int32_t from;    // the first key
  int32_t whole;   // a workgroup a tile of queries and kv head, all of its keys
  int32_t waves;   // of a workgroup: eight where whole and few, else four
  int32_t past;    // steps that are cut: past the caches, where that pays
};

// The steps of `kKeys` keys that a tile of queries takes: those over the sinks, then
// those over the window's keys.  Steps start at whole multiples of kKeys.
struct Steps {
  Keys keys;      // that any of the queries sees
  int32_t last;   // the last query that is there, -1 if none is
  int32_t sinks, window, count;  // steps over the sinks, the window's first, all (one at least)

  template <int kKeys>
  __device__ __forceinline__ int32_t key(int32_t s) const {
    return kKeys * (s < sinks ? keys.from / kKeys + s : window + s - sinks);
  }
};

// What a tile of queries costs beside its steps, in steps (64 sequences of up to 16,384 keys,
// 32 heads of 128 on 8: 204 us with 0, 63 with 4).
constexpr int32_t kStart = 4;

// Of `kRows` queries and heads that share a kv head, the tile'th such of sequence
// b, keys from `from` on.
template <int kKeys, int kRows>
__device__ __forceinline__ Steps steps_of(const PagedArgs &a, int64_t b, int32_t tile, int32_t from) {
  Steps s;
  const int32_t rows = a.length(b) * a.group, first = tile * kRows / a.group;
  s.last = rows == 0 ? -1 : min(tile * kRows + kRows, rows) - 1;
  s.last = s.last < tile * kRows ? -1 : s.last / a.group;
  s.keys = Keys{0, 0, -1, from};
  s.sinks = s.window = 0;
  s.count = 1;
  if (s.last < 0) return s;
  s.keys = a.keys(a.start(b), first, s.last);
  s.keys.from = from;
  const int32_t origin = from / kKeys, low = max(s.keys.lo, from);
  s.sinks = max((s.keys.far + kKeys - 1) / kKeys - origin, 0);
  s.window = max(low / kKeys, s.sinks > 0 ? origin + s.sinks : 0);
  const int32_t end = s.keys.hi < low ? 0 : s.keys.hi / kKeys + 1;
  s.count = max(s.sinks + max(end - s.window, 0), 1);
  return s;
}

// The same of every lane, for scalar registers.
__device__ __forceinline__ Steps uniform(const Steps &s) {
  const auto one = [](int32_t x) { return __builtin_amdgcn_readfirstlane(x); };
  return {{one(s.keys.far), one(s.keys.lo), one(s.keys.hi), one(s.keys.from)}, one(s.last),
          one(s.sinks), one(s.window), one(s.count)};
}

__device__ __forceinline__ int64_t uniform(int64_t x) {
  const auto low = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int32_t>(x)));
  return static_cast<int64_t>(__builtin_amdgcn_readfirstlane(static_cast<int32_t>(x >> 32))) << 32 | low;
}

// Inclusive sums over a workgroup of kWaves waves; `total` the last one's.
template <int kWaves>
__device__ __forceinline__ int64_t running_sums(int64_t x, int64_t *lds, int64_t &total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t below = __shfl_up(x, d);
    if (lane >= d) x += below;
  }
  __syncthreads();
  if (lane == kWave - 1) lds[wave] = x;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) x += lds[w];
    total += lds[w];
  }
  total = uniform(total);
  return x;
}

// 64-bit quotients take a workgroup some microseconds, those of 32 bits are free.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t by) {
  if (((x | by) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(by);
  return x / by;
}

// Equal stretches of `work`: workgroup g takes [first(g), first(g + 1)).
struct StepShare {
  int64_t groups, each, more;  // the first `more` take one more
  __device__ __forceinline__ StepShare(int64_t work, int32_t launched)
      : StepShare(work, max(min(work / kLeast, static_cast<int64_t>(launched)), int64_t{1})) {}
  __device__ __forceinline__ StepShare(int64_t work, int64_t n) : groups(n) {
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
// took all of it.
struct StepSpan {
  int32_t first, last;
};

// Where a kernel's results go: those of a tile that it has all keys of to `out`, or
// where `whole` is there, as sums, m and l to the query's place of it; those of a cut tile to
// the workgroup's places of `parts`, the first of two if its stretch begins with them.
struct TileParts {
  void *out;
  StepSpan *spans;
  float *whole, *parts;
};

// What a workgroup has in LDS beside its tiles.
struct StretchLds {
  int64_t sums[8], found_first;
  int32_t most[4], least[4];
  int32_t found;
  uint32_t odd;  // rows whose results are not finite
};

constexpr int32_t kTileRows = 128;  // queries a workgroup, where they are many

// paged_step.hip, paged_tiles.hip: rows and caches at sixteen-byte addresses and strides.
// Grids of tiles of kStepRows and kTileRows queries; the latter take float32 heads of 128 at most,
// 16-bit heads of 256.
// launch_paged_shared: `tiles` those of the batch against the keys before tiles.from, of the
// pages that it shares, `step` those of each sequence against the keys from there on.
msx_status launch_paged_step(msx_vtype vt, const PagedArgs &a, const StepGrid &grid,
                             const TileParts &to, hipStream_t stream);
msx_status launch_paged_tiles(msx_vtype vt, const PagedArgs &a, const StepGrid &grid,
                              const TileParts &to, hipStream_t stream);
msx_status launch_paged_shared(msx_vtype vt, const PagedArgs &a, const StepGrid &tiles,
                               const TileParts &tiles_to, const StepGrid &step,
                               const TileParts &step_to, hipStream_t stream);

// Parts of one kernel, as paged_join reads them.
struct PartSource {
  const StepSpan *spans;
  const float *whole, *parts;
  int32_t rows;    // of a tile; 0: there is no such source
  int32_t tiles;   // of a sequence and kv head; of the batch where `batched`
  int32_t batched; // tiles go through all sequences
};

// paged_join.hip: the results that are in parts, of one source or of two.
msx_status launch_paged_join(msx_vtype vt, const PagedArgs &a, const PartSource &first,
                             const PartSource &second, void *out, hipStream_t stream);

}  // namespace msx
