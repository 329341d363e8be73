// window_step.hip - one token of every sequence against its ring cache.
//
// Bound by memory: every visible key and value is read once, 2 flops a byte
// and query head.  The heads of a kv head (sixteen at a time) share each
// read, as the sixteen columns of matrix products; a wave takes 32 keys (16 in
// float32) after the other, with the next ones in flight, and keeps running
// maximum, sum and output of its own.  Keys are cut over the waves of a
// workgroup, and over workgroups where sequences and heads are too few to fill
// the chip; what they have is joined by exp(m - max m).
//
// 64 sequences of 4,100 keys, 32 heads of 128 on 8, bfloat16: 1.08 GB in 198
// us, 5.4 TB/s, over one pair of caches as over six in turn (a copy moves 5.1, reading
// and writing; float32 365 us, 5.9 TB/s); 37 of up to 1,001 keys, 24 heads of 96 on
// 8: 25 to 27 us, 3.1 TB/s, of which a third is the launch.
//
// A probability enters its products as two 16-bit values, rounded and what that
// leaves: 16 bits would add half as much again to the error of rounding the
// output, and the second product takes no time beside the memory.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_internal.h"
#include "msx_window.h"
#include "msx_step_mfma.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kWaves = kStepWaves;
constexpr int kThreads = kWaves * kWave;
constexpr int kHeads = kStepRows;  // query heads a workgroup

// The visible slots of a sequence, numbered: sinks, then the window's.
struct Slots {
  int64_t p;
  int32_t far, count;  // keys: far sinks, then the window up to p
  int32_t below;       // of the window's, those at positions below `sinks`
  int32_t near, ring, first;  // ring index of the first position past the sinks
  int32_t sinks;
  __device__ inline Slots(const StepArgs &a, int64_t position)
      : p(position), ring(a.slots - a.sinks), sinks(a.sinks) {
    const int64_t lo = p >= a.window ? p - a.window + 1 : 0;
    far = static_cast<int32_t>(lo < a.sinks ? lo : a.sinks);
    count = p < 0 ? 0 : far + static_cast<int32_t>(p - lo) + 1;
    near = static_cast<int32_t>(lo < a.sinks ? lo : 0);
    below = lo < a.sinks ? a.sinks - static_cast<int32_t>(lo) : 0;
    const int64_t past = lo < a.sinks ? 0 : lo - a.sinks;
    first = static_cast<int32_t>(past % ring);
  }
  __device__ inline int32_t slot(int32_t c) const {
    if (c < far) return c;
    const int32_t w = c - far;
    if (w < below) return near + w;
    const int32_t r = first + (w - below);
    return sinks + (r >= ring ? r - ring : r);
  }
};

template <class V, int DP>
__global__ __launch_bounds__(kThreads, DP > 128 ? 1 : 2) void step_tiles(StepArgs a, int32_t head_tiles,
                                                          int32_t splits,
                                                          typename V::Storage *out,
                                                          float *parts) {
  using S = typename V::Storage;
  using F = StepShape<V, DP>;
  __shared__ __attribute__((aligned(16))) char lds[F::kLds];

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, quad = lane / 16;
  int64_t id = blockIdx.x;
  const int32_t split = static_cast<int32_t>(id % splits);
  id /= splits;
  const int32_t head_tile = static_cast<int32_t>(id % head_tiles);
  id /= head_tiles;
  const int32_t kvh = static_cast<int32_t>(id % a.kv_heads);
  const int64_t b = id / a.kv_heads;
  const int32_t heads = min(kHeads, a.group - head_tile * kHeads);
  const int32_t h0 = kvh * a.group + head_tile * kHeads;
  const int bytes = a.dim * F::kSize;

  const Slots slots(a, a.length(b));
  // whole steps to a split, and to a wave every fourth of them
  const int32_t steps = (slots.count + F::kKeys - 1) / F::kKeys;
  const int32_t begin = static_cast<int32_t>(static_cast<int64_t>(steps) * split / splits);
  const int32_t end = static_cast<int32_t>(static_cast<int64_t>(steps) * (split + 1) / splits);

  const char *ck = reinterpret_cast<const char *>(static_cast<S *>(a.ck) + b * a.cks[0] + kvh * a.cks[2]);
  const char *cv = reinterpret_cast<const char *>(static_cast<S *>(a.cv) + b * a.cvs[0] + kvh * a.cvs[2]);
  const char *new_k = reinterpret_cast<const char *>(static_cast<const S *>(a.k) + b * a.ks[0] + kvh * a.ks[1]);
  const char *new_v = reinterpret_cast<const char *>(static_cast<const S *>(a.v) + b * a.vs[0] + kvh * a.vs[1]);
  const int64_t k_step = a.cks[1] * F::kSize, v_step = a.cvs[1] * F::kSize;

  // The token itself is read from where the caller has it; the workgroup
  // whose keys end with it puts it into the cache, where nobody reads it now.
  if (slots.count > 0 && split == splits - 1 && head_tile == 0) {
    const int64_t at = slots.slot(slots.count - 1);
    for (int c = threadIdx.x; c * 16 < bytes; c += kThreads) {
      *reinterpret_cast<v4u *>(const_cast<char *>(ck) + at * k_step + c * 16) =
          *reinterpret_cast<const v4u *>(new_k + c * 16);
      *reinterpret_cast<v4u *>(const_cast<char *>(cv) + at * v_step + c * 16) =
          *reinterpret_cast<const v4u *>(new_v + c * 16);
    }
  }

  v4u qf[F::kSteps];
  {
    const char *q = reinterpret_cast<const char *>(static_cast<const S *>(a.q) + b * a.qs[0] +
                                                   (h0 + lane % 16) * a.qs[1]);
#pragma unroll
    for (int s = 0; s < F::kSteps; ++s) {
      const int c = 4 * s + quad;
      qf[s] = v4u{0, 0, 0, 0};
      if (lane % 16 < heads && c * 16 < bytes) qf[s] = *reinterpret_cast<const v4u *>(q + c * 16);
    }
  }

  v4u kf[F::kTiles][F::kSteps], vf[F::kVPer];
  const auto fetch_k = [&](int32_t step) {
#pragma unroll
    for (int t = 0; t < F::kTiles; ++t) {
      const int32_t c = step * F::kKeys + 16 * t + lane % 16;
      const char *row = c == slots.count - 1 ? new_k : ck + slots.slot(c) * k_step;
#pragma unroll
      for (int s = 0; s < F::kSteps; ++s) {
        const int chunk = 4 * s + quad;
        kf[t][s] = v4u{0, 0, 0, 0};
        if (c < slots.count && chunk * 16 < bytes)
          kf[t][s] = *reinterpret_cast<const v4u *>(row + chunk * 16);
      }
    }
  };
  const auto fetch_v = [&](int32_t step) {
#pragma unroll
    for (int r = 0; r < F::kVPer; ++r) {
      const int at = lane + r * kWave, chunk = at % F::kChunks;
      const int32_t c = step * F::kKeys + at / F::kChunks;
      const char *row = c == slots.count - 1 ? new_v : cv + slots.slot(c) * v_step;
      vf[r] = v4u{0, 0, 0, 0};
      if (c < slots.count && chunk * 16 < bytes)
        vf[r] = *reinterpret_cast<const v4u *>(row + chunk * 16);
    }
  };

  char *tile = lds + wave * F::kTile;
  v4f o[DP / 16];
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) o[d] = v4f{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;  // l: this lane's keys only

  int32_t step = begin + wave;
  if (step < end) {
    fetch_k(step);
    fetch_v(step);
  }
  for (; step < end; step += kWaves) {
    v4f s[F::kTiles];
#pragma unroll
    for (int t = 0; t < F::kTiles; ++t) {
      s[t] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < F::kSteps; ++k) s[t] = Mfma16<V>::mul(kf[t][k], qf[k], s[t]);
    }
    const bool more = step + kWaves < end;
    if (more) fetch_k(step + kWaves);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < F::kVPer; ++r) {
      const int at = lane + r * kWave;
      *reinterpret_cast<v4u *>(tile + F::at(at / F::kChunks, at % F::kChunks)) = vf[r];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (more) fetch_v(step + kWaves);

    float x[F::kTiles * 4], top = -INFINITY;
#pragma unroll
    for (int t = 0; t < F::kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t c = step * F::kKeys + 16 * t + 4 * quad + i;
        x[4 * t + i] = c < slots.count ? s[t][i] * a.scale : -INFINITY;
        top = fmaxf(top, x[4 * t + i]);
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
    for (int j = 0; j < F::kTiles * 4; ++j) {
      x[j] = exp2_fast(x[j] - base);
      l += x[j];
    }
    if constexpr (F::kSize == 2) {
      v4u p, low;  // rounded, and what that leaves
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = Mfma<V>::pack(x[2 * j], x[2 * j + 1]);
        p[j] = pair;
        low[j] = Mfma<V>::pack(x[2 * j] - V::widen(static_cast<uint16_t>(pair)),
                               x[2 * j + 1] - V::widen(static_cast<uint16_t>(pair >> 16)));
      }
      const int i = lane % 16;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        v4s part[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int row = 16 * t + 4 * quad + i / 4, column = d * 16 + (i % 4) * 4;
          part[t] = read_transposed(tile + F::at(row, column / 8) + (column % 8) * 2);
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
          const int row = 4 * quad + i, column = d * 16 + lane % 16;
          const float v = *reinterpret_cast<const float *>(tile + F::at(row, column / 4) + (column % 4) * 4);
          o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[i], o[d], 0, 0, 0);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);

  // the waves' parts, joined: a row of DP sums, m and l a head and wave
  __syncthreads();
  float *mine = reinterpret_cast<float *>(lds) + (wave * kHeads + lane % 16) * (DP + 4);
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) *reinterpret_cast<v4f *>(mine + 16 * d + 4 * quad) = o[d];
  if (quad == 0) {
    mine[DP] = m;
    mine[DP + 1] = l;
  }
  __syncthreads();
  const float *all = reinterpret_cast<const float *>(lds);
  for (int at = threadIdx.x; at < heads * DP; at += kThreads) {
    const int head = at / DP, d = at % DP;
    if (d >= a.dim) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, all[(w * kHeads + head) * (DP + 4) + DP]);
    const float base = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float *row = all + (w * kHeads + head) * (DP + 4);
      const float f = exp2_fast(row[DP] - base);
      sum += row[d] * f;
      total += row[DP + 1] * f;
    }
    const int64_t row = b * a.heads + h0 + head;
    if (splits == 1) {
      out[row * a.dim + d] = V::narrow(total == 0.0f ? 0.0f : sum / total);
    } else {
      float *part = parts + (row * splits + split) * part_stride(a.dim);
      part[d] = sum;
      if (d == 0) {
        part[a.dim] = top;
        part[a.dim + 1] = total;
      }
    }
  }
}

// A wave a head: the splits' parts in order.
template <class V>
__global__ __launch_bounds__(kThreads) void step_join(int64_t rows, int32_t dim, int32_t splits,
                                                      const float *parts,
                                                      typename V::Storage *out) {
  const int lane = threadIdx.x % kWave;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave;
  if (row >= rows) return;
  const int64_t stride = part_stride(dim);
  const float *first = parts + row * splits * stride;
  float top = -INFINITY;
  for (int32_t s = lane; s < splits; s += kWave) top = fmaxf(top, first[s * stride + dim]);
  top = wave_max(top);
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  for (int32_t s = lane; s < splits; s += kWave)
    total += first[s * stride + dim + 1] * exp2_fast(first[s * stride + dim] - base);
  total = wave_sum(total);
  for (int32_t d = lane; d < dim; d += kWave) {
    float sum = 0.0f;
    for (int32_t s = 0; s < splits; ++s)
      sum += first[s * stride + d] * exp2_fast(first[s * stride + dim] - base);
    out[row * dim + d] = V::narrow(total == 0.0f ? 0.0f : sum / total);
  }
}

int32_t head_tiles(const StepArgs &a) { return (a.group + kHeads - 1) / kHeads; }

// Workgroups until each CU has two (what the registers allow), of four steps
// a wave at least: shorter parts cost more in joining than they gain.
int32_t splits_for(const StepArgs &a, int32_t keys_a_step) {
  constexpr int64_t kFull = 2 * 256;
  const int64_t groups = a.batch * a.kv_heads * head_tiles(a);
  const int64_t held = std::min<int64_t>(static_cast<int64_t>(a.window) + a.sinks, a.slots);
  const int64_t most = std::max<int64_t>(1, held / (4 * kWaves * keys_a_step));
  return static_cast<int32_t>(std::min(most, std::max<int64_t>(1, kFull / groups)));
}

template <class V, int DP>
msx_status run(const StepArgs &a, void *out, float *parts, hipStream_t stream) {
  using S = typename V::Storage;
  const int32_t splits = splits_for(a, StepShape<V, DP>::kKeys);
  const int64_t blocks = a.batch * a.kv_heads * head_tiles(a) * splits;
  if (std::max(blocks, (a.batch * a.heads + kWaves - 1) / kWaves) > max_blocks(kThreads))
    return fail(MSX_EINVAL, "window_attention_step has more rows than a grid holds.");
  step_tiles<V, DP><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
      a, head_tiles(a), splits, static_cast<S *>(out), parts);
  if (splits > 1) {
    const int64_t rows = a.batch * a.heads;
    step_join<V><<<static_cast<unsigned>((rows + kWaves - 1) / kWaves), kThreads, 0, stream>>>(
        rows, a.dim, splits, parts, static_cast<S *>(out));
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "window_attention_step");
}

template <class V>
msx_status by_dim(const StepArgs &a, void *out, float *parts, hipStream_t stream) {
  if (a.dim <= 64) return run<V, 64>(a, out, parts, stream);
  if (a.dim <= 128) return run<V, 128>(a, out, parts, stream);
  return run<V, 256>(a, out, parts, stream);
}

}  // namespace

size_t window_step_scratch(msx_vtype vt, const StepArgs &a) {
  const int32_t splits = splits_for(a, vt == MSX_F32 ? 16 : 32);
  if (splits == 1) return 0;
  return sizeof(float) * static_cast<size_t>(a.batch) * a.heads * splits * ((a.dim + 5) / 4 * 4);
}

msx_status launch_window_step(msx_vtype vt, const StepArgs &a, void *out, void *scratch,
                              hipStream_t stream) {
  float *parts = static_cast<float *>(scratch);
  switch (vt) {
  case MSX_F32: return by_dim<F32>(a, out, parts, stream);
  case MSX_F16: return by_dim<F16>(a, out, parts, stream);
  default: return by_dim<BF16>(a, out, parts, stream);
  }
}

}  // namespace msx
