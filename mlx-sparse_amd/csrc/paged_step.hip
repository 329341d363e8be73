// paged_step.hip - a few queries of every sequence against its pages.
//
// Bound by memory: every visible key and value is read once, 2 flops a byte, query
// and head.  The queries and heads that share a kv head (sixteen at a time) share
// each read, as the sixteen columns of matrix products; a wave takes 32 keys (16 in
// float32) after the other, with the next ones in flight and their pages' numbers
// a step ahead of them, and keeps running maximum, sum and output of its own.
//
// Sequences differ in length, and the host knows none of them.  The steps of all
// (sequence, sixteen queries, kv head) are numbered through, and each workgroup takes
// an equal stretch of them, whatever it begins and ends in: every workgroup adds
// up the batch's lengths to find its own.  Of a stretch only the first and the last tile
// of queries can be another's as well; what it has of them goes to two places
// of scratch, and paged_join adds those up in the order of the keys.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_internal.h"
#include "msx_paged.h"
#include "msx_paged_row.h"
#include "msx_paged_tiles.h"
#include "msx_step_mfma.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kThreads = kStepWaves * kWave;

// The steps of `kKeys` keys that sixteen queries take: those over the sinks,
// then those over the window's keys.
struct Steps {
  Keys keys;      // that any of the queries sees
  int32_t first;  // queries [first, last] are there, none where last < first
  int32_t last;
  int32_t sinks, window, count;  // steps over the sinks, the window's first, all (one at least)
};

// What a tile of queries costs beside its steps, in steps.
constexpr int32_t kStart = 4;

template <int kKeys>
__device__ __forceinline__ Steps steps_of(const PagedArgs &a, int64_t b, int32_t tile) {
  Steps s;
  const int32_t rows = a.tokens * a.group;
  const int64_t start = a.start(b);
  s.first = tile * kStepRows / a.group;
  s.last = min(min(tile * kStepRows + kStepRows, rows) - 1, a.length(b) * a.group - 1) / a.group;
  if (a.length(b) == 0 || s.last < s.first) {
    s.last = s.first - 1;
    s.keys = Keys{0, 0, -1};
    s.sinks = s.window = 0;
    s.count = 1;
    return s;
  }
  s.keys = a.keys(start, s.first, s.last);
  s.sinks = (s.keys.far + kKeys - 1) / kKeys;
  s.window = max(s.keys.lo / kKeys, s.sinks);
  const int32_t end = s.keys.hi < s.keys.lo ? 0 : s.keys.hi / kKeys + 1;
  s.count = max(s.sinks + max(end - s.window, 0), 1);
  return s;
}

// The same of every lane, for scalar registers.
__device__ __forceinline__ Steps uniform(const Steps &s) {
  const auto one = [](int32_t x) { return __builtin_amdgcn_readfirstlane(x); };
  return {{one(s.keys.far), one(s.keys.lo), one(s.keys.hi)}, one(s.first), one(s.last),
          one(s.sinks), one(s.window), one(s.count)};
}

// Inclusive sums over the workgroup's threads; `total` the last one's.
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
  for (int w = 0; w < kStepWaves; ++w) {
    if (w < wave) x += lds[w];
    total += lds[w];
  }
  return x;
}

template <class V, int DP>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void paged_step(PagedArgs a, StepGrid grid,
                                                                         typename V::Storage *out,
                                                                         StepSpan *spans,
                                                                         float *parts) {
  using S = typename V::Storage;
  using F = StepShape<V, DP>;
  __shared__ __attribute__((aligned(16))) char lds[F::kLds];
  __shared__ int64_t sums[kStepWaves], found_first;
  __shared__ int32_t found;
  __shared__ uint32_t odd;

  const int lane = threadIdx.x % kWave, quad = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int bytes = a.dim * F::kSize;

  // this workgroup's stretch of all steps
  const int64_t entries = a.batch * grid.tiles;  // (sequence, sixteen queries)
  const auto cost_at = [&](int64_t e) -> int64_t {
    if (e >= entries) return 0;
    const int64_t b = grid.tiles == 1 ? e : e / grid.tiles;
    return kStart + steps_of<F::kKeys>(a, b, static_cast<int32_t>(e - b * grid.tiles)).count;
  };
  int64_t total = 0, cost = cost_at(threadIdx.x), upto = running_sums(cost, sums, total);
  if (entries > kThreads) {
    int64_t mine = cost;
    for (int64_t e = threadIdx.x + kThreads; e < entries; e += kThreads) mine += cost_at(e);
    running_sums(mine, sums, total);
  }
  const StepShare share(total * a.kv_heads, grid.groups);
  const int64_t g = blockIdx.x;
  if (g >= share.groups) return;  // whole workgroups leave
  const int64_t begin = share.first(g), end = share.first(g + 1);
  int64_t before = 0;
  for (int64_t e0 = 0;; e0 += kThreads) {  // (all that is to be done is some entry's)
    int64_t here = total;
    if (entries > kThreads) {
      if (e0 > 0) cost = cost_at(e0 + threadIdx.x);
      upto = running_sums(cost, sums, here);
    }
    const int64_t low = (before + upto - cost) * a.kv_heads, high = (before + upto) * a.kv_heads;
    if (low <= begin && begin < high) {
      found = static_cast<int32_t>(e0 + threadIdx.x);
      found_first = low;
    }
    before += here;
    if (begin < before * a.kv_heads || e0 + kThreads >= entries) break;
  }
  __syncthreads();
  int32_t entry = __builtin_amdgcn_readfirstlane(found), kvh = -1;
  int64_t x = found_first;  // where the next (entry, kv head) begins

  while (x < end) {
    const int64_t b = grid.tiles == 1 ? entry : entry / grid.tiles;
    const int32_t row_tile = entry - static_cast<int32_t>(b) * grid.tiles;
    const Steps steps = uniform(steps_of<F::kKeys>(a, b, row_tile));
    if (kvh < 0) {
      kvh = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(quotient(begin - x, steps.count + kStart)));
      x += static_cast<int64_t>(kvh) * (steps.count + kStart);
    }
    const int64_t first_step = x + kStart;
    x = first_step + steps.count;
    const int32_t s_begin = __builtin_amdgcn_readfirstlane(
        static_cast<int32_t>(min(max(begin - first_step, int64_t{0}), static_cast<int64_t>(steps.count))));
    const int32_t s_end = __builtin_amdgcn_readfirstlane(
        static_cast<int32_t>(max(min(end - first_step, static_cast<int64_t>(steps.count)), int64_t{0})));
    const int32_t head = kvh, mine_entry = entry;
    if (++kvh == a.kv_heads) {
      kvh = 0;
      ++entry;
    }
    if (s_begin >= s_end) continue;  // what this workgroup has of it is no step
    const auto key_of = [&](int32_t s) { return F::kKeys * (s < steps.sinks ? s : steps.window + s - steps.sinks); };

    // this lane's query, and what it sees
    const int32_t row = row_tile * kStepRows + lane % 16, t = row / a.group;
    const int32_t h = head * a.group + row % a.group;
    const bool live = t <= steps.last && row < a.tokens * a.group;
    Keys mine{0, 0, -1};
    if (live) mine = a.keys(a.start(b), t, t);

    v4u qf[F::kSteps];
    {
      const char *q = reinterpret_cast<const char *>(static_cast<const S *>(a.q) + b * a.qs[0] +
                                                     t * a.qs[1] + h * a.qs[2]);
#pragma unroll
      for (int s = 0; s < F::kSteps; ++s) {
        const int c = 4 * s + quad;
        qf[s] = v4u{0, 0, 0, 0};
        if (live && c * 16 < bytes) qf[s] = *reinterpret_cast<const v4u *>(q + c * 16);
      }
    }
    const char *ck = reinterpret_cast<const char *>(static_cast<const S *>(a.k) + head * a.ks[2]);
    const char *cv = reinterpret_cast<const char *>(static_cast<const S *>(a.v) + head * a.vs[2]);

    // the page of key `lane` of a step, -1 where nobody sees it
    const auto pages_of = [&](int32_t s) {
      const int32_t j = key_of(s) + lane;
      return s < s_end && lane < F::kKeys && steps.keys.sees(j) ? a.table.page(b, j) : -1;
    };
    v4u kf[F::kTiles][F::kSteps], vf[F::kVPer];
    const auto fetch_k = [&](int32_t s, int32_t pages) {
#pragma unroll
      for (int i = 0; i < F::kTiles; ++i) {
        const int place = 16 * i + lane % 16;
        const int64_t page = __shfl(pages, place);
        const char *from = ck + (page * a.ks[0] + a.table.slot(key_of(s) + place) * a.ks[1]) * F::kSize;
#pragma unroll
        for (int c = 0; c < F::kSteps; ++c) {
          const int chunk = 4 * c + quad;
          kf[i][c] = v4u{0, 0, 0, 0};
          if (page >= 0 && chunk * 16 < bytes) kf[i][c] = *reinterpret_cast<const v4u *>(from + chunk * 16);
        }
      }
    };
    const auto fetch_v = [&](int32_t s, int32_t pages) {
#pragma unroll
      for (int r = 0; r < F::kVPer; ++r) {
        const int at = lane + r * kWave, chunk = at % F::kChunks, place = at / F::kChunks;
        const int64_t page = __shfl(pages, place);
        const char *from = cv + (page * a.vs[0] + a.table.slot(key_of(s) + place) * a.vs[1]) * F::kSize;
        vf[r] = v4u{0, 0, 0, 0};
        if (page >= 0 && chunk * 16 < bytes) vf[r] = *reinterpret_cast<const v4u *>(from + chunk * 16);
      }
    };

    char *tile = lds + wave * F::kTile;
    v4f o[DP / 16];
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[d] = v4f{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;  // l: this lane's keys only

    int32_t step = s_begin + wave;
    int32_t pages = pages_of(step), ahead = pages_of(step + kStepWaves);
    if (step < s_end) {
      fetch_k(step, pages);
      fetch_v(step, pages);
    }
    for (; step < s_end; step += kStepWaves) {
      v4f s[F::kTiles];
#pragma unroll
      for (int i = 0; i < F::kTiles; ++i) {
        s[i] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < F::kSteps; ++c) s[i] = Mfma16<V>::mul(kf[i][c], qf[c], s[i]);
      }
      const uint32_t there = static_cast<uint32_t>(__ballot(pages >= 0));
      const bool more = step + kStepWaves < s_end;
      pages = ahead;
      ahead = pages_of(step + 2 * kStepWaves);
      if (more) fetch_k(step + kStepWaves, pages);
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r = 0; r < F::kVPer; ++r) {
        const int at = lane + r * kWave;
        *reinterpret_cast<v4u *>(tile + F::at(at / F::kChunks, at % F::kChunks)) = vf[r];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (more) fetch_v(step + kStepWaves, pages);

      float x[F::kTiles * 4], top = -INFINITY;
      const int32_t j0 = key_of(step) + 4 * quad;
#pragma unroll
      for (int i = 0; i < F::kTiles; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int place = 16 * i + k;
          const bool seen = (there >> (place + 4 * quad) & 1) && mine.sees(j0 + place);
          x[4 * i + k] = seen ? s[i][k] * a.scale : -INFINITY;
          top = fmaxf(top, x[4 * i + k]);
        }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float grown = fmaxf(m, top);
      const float base = grown == -INFINITY ? 0.0f : grown;
      if (__any(grown > m)) {
        const float shrink = exp2_fast(m - base);
        l *= shrink;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[d] *= shrink;
      }
      m = grown;
#pragma unroll
      for (int k = 0; k < F::kTiles * 4; ++k) {
        x[k] = exp2_fast(x[k] - base);
        l += x[k];
      }
      if constexpr (F::kSize == 2) {
        v4u p, low;  // rounded, and what that leaves: the output has its own rounding alone
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t pair = Mfma<V>::pack(x[2 * k], x[2 * k + 1]);
          p[k] = pair;
          low[k] = Mfma<V>::pack(x[2 * k] - V::widen(static_cast<uint16_t>(pair)),
                                 x[2 * k + 1] - V::widen(static_cast<uint16_t>(pair >> 16)));
        }
        const int i = lane % 16;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          v4s part[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int place = 16 * k + 4 * quad + i / 4, column = d * 16 + (i % 4) * 4;
            part[k] = read_transposed(tile + F::at(place, column / 8) + (column % 8) * 2);
          }
          const auto lo = __builtin_bit_cast(v2u, part[0]), hi = __builtin_bit_cast(v2u, part[1]);
          const v4u values{lo[0], lo[1], hi[0], hi[1]};
          o[d] = Mfma16<V>::mul(values, p, o[d]);
          o[d] = Mfma16<V>::mul(values, low, o[d]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) {
            const int place = 4 * quad + i, column = d * 16 + lane % 16;
            const float v = *reinterpret_cast<const float *>(tile + F::at(place, column / 4) + (column % 4) * 4);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[i], o[d], 0, 0, 0);
          }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' parts, joined: a row of DP sums, m and l a query and wave
    __syncthreads();
    float *own = reinterpret_cast<float *>(lds) + (wave * kStepRows + lane % 16) * (DP + 4);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) *reinterpret_cast<v4f *>(own + 16 * d + 4 * quad) = o[d];
    if (quad == 0) {
      own[DP] = m;
      own[DP + 1] = l;
    }
    if (threadIdx.x == 0) odd = 0;
    __syncthreads();
    const bool whole = s_begin == 0 && s_end == steps.count;
    const int64_t unit = static_cast<int64_t>(mine_entry) * a.kv_heads + head;
    if (threadIdx.x == 0 && s_begin == 0)
      spans[unit] = whole ? StepSpan{0, -1}
                          : StepSpan{static_cast<int32_t>(g),
                                     static_cast<int32_t>(share.owner(first_step + steps.count - 1))};
    const float *all = reinterpret_cast<const float *>(lds);
    const int32_t rows = min(kStepRows, a.tokens * a.group - row_tile * kStepRows);
    for (int at = threadIdx.x; at < rows * DP; at += kThreads) {
      const int i = at / DP, d = at % DP;
      if (d >= a.dim) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kStepWaves; ++w) top = fmaxf(top, all[(w * kStepRows + i) * (DP + 4) + DP]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, norm = 0.0f;
#pragma unroll
      for (int w = 0; w < kStepWaves; ++w) {
        const float *from = all + (w * kStepRows + i) * (DP + 4);
        const float f = exp2_fast(from[DP] - base);
        sum += from[d] * f;
        norm += from[DP + 1] * f;
      }
      const int32_t r = row_tile * kStepRows + i;
      if (whole) {
        const float value = norm == 0.0f ? 0.0f : sum / norm;
        if (!(fabsf(value) < INFINITY)) atomicOr(&odd, 1u << i);
        out[((b * a.tokens + r / a.group) * a.heads + head * a.group + r % a.group) * a.dim + d] =
            V::narrow(value);
      } else {
        float *part = parts + ((2 * g + (s_begin == 0 ? 1 : 0)) * kStepRows + i) * part_stride(a.dim);
        part[d] = sum;
        if (d == 0) {
          part[a.dim] = top;
          part[a.dim + 1] = norm;
        }
      }
    }
    __syncthreads();
    for (uint32_t anew = odd; anew != 0; anew &= anew - 1) {
      const int i = __builtin_ctz(anew);
      if (i % kStepWaves != wave) continue;
      const int32_t r = row_tile * kStepRows + i;
      paged_row<V>(a, b, r / a.group, head * a.group + r % a.group,
                   reinterpret_cast<float *>(lds) + wave * DP, out);
    }
    __syncthreads();
  }
}

// A workgroup a (sequence, query, head) whose keys were cut over workgroups: their sums
// in the order of the keys, four values a thread, every eighth part (dim 128) of
// them; then those of the threads that have the same values, through LDS.
template <class V, int DP>
__global__ __launch_bounds__(kThreads) void paged_join(PagedArgs a, StepGrid grid,
                                                       const StepSpan *spans, const float *parts,
                                                       typename V::Storage *out) {
  constexpr int kLanes = DP / 4, kBeside = kThreads / kLanes;
  __shared__ __attribute__((aligned(16))) float lds[kBeside][DP + 4];
  const int64_t row = blockIdx.x;
  const int32_t h = static_cast<int32_t>(row % a.heads);
  const int32_t t = static_cast<int32_t>(row / a.heads % a.tokens);
  const int64_t b = row / a.heads / a.tokens;
  const int32_t r = t * a.group + h % a.group, i = r % kStepRows;
  const StepSpan span = spans[(b * grid.tiles + r / kStepRows) * a.kv_heads + h / a.group];
  if (span.last < span.first) return;
  const int64_t stride = part_stride(a.dim);
  const int32_t n = span.last - span.first + 1;
  const int beside = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  float m = -INFINITY, l = 0.0f;
  v4f o{0, 0, 0, 0};
#pragma unroll 4
  for (int32_t s = beside; s < n; s += kBeside) {
    // the first workgroup's last place, the others' first
    const float *part = parts + ((2 * static_cast<int64_t>(span.first + s) + (s == 0 ? 1 : 0)) * kStepRows + i) * stride;
    const float part_m = part[a.dim], part_l = part[a.dim + 1];
    v4f x{0, 0, 0, 0};
    if (d < a.dim) x = *reinterpret_cast<const v4f *>(part + d);
    const float top = fmaxf(m, part_m), base = top == -INFINITY ? 0.0f : top;
    const float keep = exp2_fast(m - base), f = exp2_fast(part_m - base);
    l = l * keep + part_l * f;
    o = o * keep + x * f;
    m = top;
  }
  *reinterpret_cast<v4f *>(&lds[beside][d]) = o;
  if (d == 0) {
    lds[beside][DP] = m;
    lds[beside][DP + 1] = l;
  }
  __syncthreads();
  bool bad = false;
  if (threadIdx.x < a.dim) {
    float top = -INFINITY, sum = 0.0f, norm = 0.0f;
#pragma unroll
    for (int s = 0; s < kBeside; ++s) top = fmaxf(top, lds[s][DP]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int s = 0; s < kBeside; ++s) {
      const float f = exp2_fast(lds[s][DP] - base);
      sum += lds[s][threadIdx.x] * f;
      norm += lds[s][DP + 1] * f;
    }
    const float value = norm == 0.0f ? 0.0f : sum / norm;
    bad = !(fabsf(value) < INFINITY);
    out[row * a.dim + threadIdx.x] = V::narrow(value);
  }
  if (__syncthreads_or(bad) && threadIdx.x < kWave) paged_row<V>(a, b, t, h, &lds[0][0], out);
}

StepGrid grid_of(const PagedArgs &a) {
  StepGrid g;
  g.tiles = static_cast<int32_t>((static_cast<int64_t>(a.tokens) * a.group + kStepRows - 1) / kStepRows);
  g.groups = a.dim > 128 ? 256 : 512;  // what runs at once: registers allow one a CU, or two
  return g;
}

size_t spans_bytes(const PagedArgs &a) {
  return (sizeof(StepSpan) * static_cast<size_t>(a.batch) * grid_of(a).tiles * a.kv_heads + 255) / 256 * 256;
}

template <class V, int DP>
msx_status run(const PagedArgs &a, void *out, void *scratch, hipStream_t stream) {
  using S = typename V::Storage;
  const StepGrid grid = grid_of(a);
  const int64_t rows = a.batch * a.tokens * a.heads;
  if (a.batch * grid.tiles > kWindowIntMax || rows > max_blocks(kThreads))
    return fail(MSX_EINVAL, "paged_attention has more rows than a grid holds.");
  auto *spans = static_cast<StepSpan *>(scratch);
  auto *parts = reinterpret_cast<float *>(static_cast<char *>(scratch) + spans_bytes(a));
  paged_step<V, DP><<<grid.groups, kThreads, 0, stream>>>(a, grid, static_cast<S *>(out), spans, parts);
  paged_join<V, DP><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(a, grid, spans, parts,
                                                                         static_cast<S *>(out));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
}

template <class V>
msx_status by_dim(const PagedArgs &a, void *out, void *scratch, hipStream_t stream) {
  if (a.dim <= 64) return run<V, 64>(a, out, scratch, stream);
  if (a.dim <= 128) return run<V, 128>(a, out, scratch, stream);
  return run<V, 256>(a, out, scratch, stream);
}

}  // namespace

size_t paged_step_scratch(const PagedArgs &a) {
  return spans_bytes(a) +
         sizeof(float) * 2 * grid_of(a).groups * kStepRows * static_cast<size_t>(part_stride(a.dim));
}

msx_status launch_paged_step(msx_vtype vt, const PagedArgs &a, void *out, void *scratch,
                             hipStream_t stream) {
  switch (vt) {
  case MSX_F32: return by_dim<F32>(a, out, scratch, stream);
  case MSX_F16: return by_dim<F16>(a, out, scratch, stream);
  default: return by_dim<BF16>(a, out, scratch, stream);
  }
}

}  // namespace msx
