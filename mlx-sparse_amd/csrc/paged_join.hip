// paged_join.hip - results of paged attention that are in parts, joined by exp(m - max m).
//
// A workgroup a (sequence, query, head): its parts in the order of the keys, four
// values a thread, of heads of 128 every eighth part; then those of the threads that
// have the same values, through LDS.  64 parts of 32 rows: 5 us (a wave a row, 13.5).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_internal.h"
#include "msx_paged.h"
#include "msx_paged_row.h"
#include "msx_paged_tiles.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kThreads = 256;

// The parts of one query and head from one source.
struct Parts {
  const float *whole, *first, *next;  // the first one lies apart
  int64_t step;
  int32_t count;
  __device__ __forceinline__ Parts(const PagedArgs &a, const PartSource &s, int64_t b, int32_t t, int32_t h)
      : whole(nullptr), first(nullptr), next(nullptr), step(0), count(0) {
    if (s.rows == 0) return;
    const int64_t stride = part_stride(a.dim);
    const int64_t r = (s.batched ? b * a.tokens + t : t) * a.group + h % a.group;
    const int64_t entries = s.batched ? s.tiles : a.batch * s.tiles;
    const int64_t entry = (s.batched ? 0 : b * s.tiles) + r / s.rows;
    const StepSpan span = s.spans[(h / a.group) * entries + entry];
    if (span.last < span.first) {
      whole = s.whole == nullptr ? nullptr : s.whole + ((b * a.tokens + t) * a.heads + h) * stride;
      first = whole;
      count = whole == nullptr ? 0 : 1;
      return;
    }
    // the first workgroup's second place, the others' first
    const float *place = s.parts + (2 * static_cast<int64_t>(span.first) * s.rows + r % s.rows) * stride;
    first = place + s.rows * stride;
    step = 2 * s.rows * stride;
    next = place;
    count = span.last - span.first + 1;
  }
  __device__ __forceinline__ const float *at(int32_t s) const { return s == 0 ? first : next + s * step; }
};

template <class V, int DP>
__global__ __launch_bounds__(kThreads) void paged_join(PagedArgs a, PartSource one, PartSource two,
                                                       typename V::Storage *out) {
  constexpr int kLanes = DP / 4, kBeside = kThreads / kLanes;
  __shared__ __attribute__((aligned(16))) float lds[kBeside][DP + 4];
  const int64_t row = blockIdx.x;
  const int32_t h = static_cast<int32_t>(row % a.heads);
  const int32_t t = static_cast<int32_t>(row / a.heads % a.tokens);
  const int64_t b = row / a.heads / a.tokens;
  const Parts p(a, one, b, t, h), q(a, two, b, t, h);
  const int32_t n = p.count + q.count;
  if (n == 0) return;  // written where it was worked out
  const int beside = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
  float m = -INFINITY, l = 0.0f;
  v4f o{0, 0, 0, 0};
#pragma unroll 4
  for (int32_t s = beside; s < n; s += kBeside) {
    const float *part = s < p.count ? p.at(s) : q.at(s - p.count);
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
  // a value that is not finite may be a key's that this query does not see
  if (__syncthreads_or(bad) && threadIdx.x < kWave) paged_row<V>(a, b, t, h, &lds[0][0], out);
}

// The same for many rows of few parts each: a row's parts one after the other, four
// values a thread, kBeside rows a workgroup.
template <class V, int DP>
__global__ __launch_bounds__(kThreads) void paged_join_rows(PagedArgs a, PartSource one, PartSource two,
                                                            int64_t first, int64_t rows,
                                                            typename V::Storage *out) {
  constexpr int kLanes = DP / 4, kBeside = kThreads / kLanes;
  __shared__ float q_lds[kThreads / kWave][kWindowMaxDim];
  const int64_t row = first + static_cast<int64_t>(blockIdx.x) * kBeside + threadIdx.x / kLanes;
  const int d = threadIdx.x % kLanes * 4;
  const int32_t h = static_cast<int32_t>(row % a.heads);
  const int32_t t = static_cast<int32_t>(row / a.heads % a.tokens);
  const int64_t b = row / a.heads / a.tokens;
  bool bad = false;
  if (row < rows) {
    const Parts p(a, one, b, t, h), q(a, two, b, t, h);
    const int32_t n = p.count + q.count;
    float m = -INFINITY, l = 0.0f;
    v4f o{0, 0, 0, 0};
#pragma unroll 4
    for (int32_t s = 0; s < n; ++s) {
      const float *part = s < p.count ? p.at(s) : q.at(s - p.count);
      const float part_m = part[a.dim], part_l = part[a.dim + 1];
      v4f x{0, 0, 0, 0};
      if (d < a.dim) x = *reinterpret_cast<const v4f *>(part + d);
      const float top = fmaxf(m, part_m), base = top == -INFINITY ? 0.0f : top;
      const float keep = exp2_fast(m - base), f = exp2_fast(part_m - base);
      l = l * keep + part_l * f;
      o = o * keep + x * f;
      m = top;
    }
    if (n > 0 && d < a.dim) {  // (else written where it was worked out)
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = l == 0.0f ? 0.0f : o[j] / l;
        bad = bad || !(fabsf(x[j]) < INFINITY);
      }
      store_four<V>(x, x, out + row * a.dim + d, nullptr);
    }
  }
  uint64_t anew = __ballot(bad);
  while (anew != 0) {
    const int at = __builtin_ctzll(anew) / kLanes * kLanes;  // the first lane of the row's
    anew &= ~((kLanes == kWave ? ~uint64_t{0} : (uint64_t{1} << kLanes) - 1) << at);
    paged_row<V>(a, __shfl(b, at), __shfl(t, at), __shfl(h, at), q_lds[threadIdx.x / kWave], out);
  }
}

// Above so many rows a row has few parts: they share 512 workgroups' stretches.  2,048 queries
// of 16 heads in three parts each take 12 us so, 63 a workgroup a row.
constexpr int64_t kManyRows = 4096;

template <class V, int DP>
msx_status run(const PagedArgs &a, const PartSource &first, const PartSource &second, void *out,
               hipStream_t stream) {
  constexpr int64_t kBeside = kThreads / (DP / 4);
  const int64_t rows = a.batch * a.tokens * a.heads;
  auto *to = static_cast<typename V::Storage *>(out);
  if (rows > kManyRows) {
    const int64_t most = max_blocks(kThreads) * kBeside;
    for (int64_t row = 0; row < rows; row += most)
      paged_join_rows<V, DP><<<static_cast<unsigned>((std::min(rows - row, most) + kBeside - 1) / kBeside),
                               kThreads, 0, stream>>>(a, first, second, row, rows, to);
  } else {
    paged_join<V, DP><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(a, first, second, to);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
}

template <class V>
msx_status by_dim(const PagedArgs &a, const PartSource &first, const PartSource &second, void *out,
                  hipStream_t stream) {
  if (a.dim <= 64) return run<V, 64>(a, first, second, out, stream);
  if (a.dim <= 128) return run<V, 128>(a, first, second, out, stream);
  return run<V, 256>(a, first, second, out, stream);
}

}  // namespace

msx_status launch_paged_join(msx_vtype vt, const PagedArgs &a, const PartSource &first,
                             const PartSource &second, void *out, hipStream_t stream) {
  switch (vt) {
  case MSX_F32: return by_dim<F32>(a, first, second, out, stream);
  case MSX_F16: return by_dim<F16>(a, first, second, out, stream);
  default: return by_dim<BF16>(a, first, second, out, stream);
  }
}

}  // namespace msx
