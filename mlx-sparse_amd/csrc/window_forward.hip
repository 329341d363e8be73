// window_forward.hip - window attention's forward product on the matrix
// cores: float32, float16 and bfloat16, head dimensions up to 128 whose rows
// are sixteen-byte aligned.
//
// A wave takes 32 queries of one head, a workgroup kWaves such units that
// follow each other over (32 positions, head of the group): with four heads a
// kv head, its waves share one span of keys.  Keys are numbered through: the
// sinks before the span, then the span, so that a few sinks cost no tile of
// their own.  Per tile of keys: S^T = K Q^T from LDS, the running maximum and
// sum, O^T += V^T P^T; the next tile's rows are on their way to LDS meanwhile.
//
// Probabilities are rounded to the operands' 16 bits for the second product,
// unnormalised and at most 2^8, as the matrix instruction takes them: their errors are
// independent and no larger than the output's own rounding.  The residue that a
// call with gradients keeps is of the output divided by the sum of the rounded
// ones: where two keys share a query 85 to 1 the rounding of one would be a factor of
// delta, and dq 21 % off in bfloat16 (0.7 so).  Scores, maximum, sums and output stay
// float32.
//
// Bound by how a wave's matrix instructions, exponentials and LDS reads take
// turns: a tile of 64 keys costs a wave 1,024 cycles of products, some 950 of
// vector instructions and 2 x 16 KB of LDS, and with two waves a SIMD the
// products are under way 30 % of the time, without a bank conflict.  A call of 8,192
// tokens of 32 heads of 128 on 8, a window of 1,024: 177 us, 730 TFLOP/s of
// the work that the window needs (a large matrix product reaches 1,199); 4,099
// on 20,001 keys, 16 heads on 8, a window of 4,096, float16: 165 us, 840, of which
// 6 are the join's.  float32, 8,192 tokens as above: 1,270 us, 102 (a large product 153).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_internal.h"
#include "msx_window.h"
#include "msx_window_mfma.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kRows = 32;  // queries a wave

template <class V, int DP>
struct ForwardShape {
  using T = TileShape<V, DP>;
  static constexpr int kSub = T::kSize == 2 ? 2 : 1;  // 32-key parts of a tile
  static constexpr int kKeys = 32 * kSub;
  static constexpr int kTile = kKeys * T::kPitch;
  static constexpr int kLds = 4 * kTile;  // K and V, twice
  // workgroups a CU: two hide each other's waits; wide float32 heads need the
  // registers of one (76 spilled with two at 128)
  static constexpr int kBlocks = T::kRowBytes > 256 ? 1 : 2;
  static constexpr int kStride = DP + 4;  // of a row's sums, m, l and taken in scratch
};

// A query row by its definition, one wave: keys over the lanes for the
// scores, head values over the lanes for the sum.  Taken where a tile's
// product is not finite, which a masked key's own infinity or NaN does too.
template <class V>
__device__ void forward_row(const WindowArgs &a, int64_t b, int32_t i, int32_t h, int32_t p,
                            float *q_lds, typename V::Storage *out) {
  using S = typename V::Storage;
  const int lane = threadIdx.x % kWave;
  const S *q = static_cast<const S *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const S *k = static_cast<const S *>(a.k) + b * a.ks[0] + (h / a.group) * a.ks[2];
  const S *v = static_cast<const S *>(a.v) + b * a.vs[0] + (h / a.group) * a.vs[2];
  __builtin_amdgcn_wave_barrier();
  for (int d = lane; d < a.dim; d += kWave) q_lds[d] = V::widen(q[d]);
  __builtin_amdgcn_wave_barrier();
  const Seen seen(p, a.window, a.sinks);
  const int32_t n = seen.count(p);
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  for (int32_t c0 = 0; c0 < n; c0 += kWave) {
    const S *row = k + seen.key(min(c0 + lane, n - 1)) * a.ks[1];
    float s = 0.0f;
    for (int d = 0; d < a.dim; ++d) s += q_lds[d] * V::widen(row[d]);
    s = c0 + lane < n ? s * a.scale : -INFINITY;
    const float top = fmaxf(m, wave_max(s)), base = top == -INFINITY ? 0.0f : top;
    const float e = exp2_fast(s - base), keep = exp2_fast(m - base);
    l = l * keep + wave_sum(e);
    m = top;
    o0 *= keep;
    o1 *= keep;
    const int32_t here = min(kWave, n - c0);
    for (int32_t t = 0; t < here; ++t) {
      const float w = __shfl(e, t);
      const S *from = v + seen.key(c0 + t) * a.vs[1];
      if (lane < a.dim) o0 += w * V::widen(from[lane]);
      if (lane + kWave < a.dim) o1 += w * V::widen(from[lane + kWave]);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t at = ((b * a.lq + i) * a.heads + h) * a.dim;
  const auto store = [&](int d, float x) {
    if (d >= a.dim) return;
    const S kept = V::narrow(x);
    out[at + d] = kept;
    if constexpr (sizeof(S) == 2)
      if (a.low != nullptr) static_cast<S *>(a.low)[a.low_at(b, i, h, d)] = Residue<V>::of(x, kept);
  };
  store(lane, o0 * inv);
  store(lane + kWave, o1 * inv);
}

template <class V, int DP>
__global__ __launch_bounds__(kThreads, (ForwardShape<V, DP>::kBlocks)) void forward_tiles(WindowArgs a, int32_t units_per_bh,
                                                             int64_t blocks_per_bh, TailCut cut,
                                                             typename V::Storage *out, float *lse,
                                                             float *sums) {
  using S = typename V::Storage;
  using T = TileShape<V, DP>;
  using F = ForwardShape<V, DP>;
  using Frag = typename Mfma<V>::Frag;
  constexpr int kSteps = DP / Mfma<V>::kDepth;
  __shared__ __attribute__((aligned(1024))) char lds[F::kLds];
  const TileLanes<V, DP> lanes(lds);

  const int lane = threadIdx.x % kWave, half = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const CutItem item(cut, blockIdx.x);
  const uint32_t per_bh = static_cast<uint32_t>(blocks_per_bh), bh = item.block / per_bh;
  const int32_t first_unit = static_cast<int32_t>(item.block % per_bh) * kWaves;
  const int64_t b = bh / a.kv_heads;
  const int32_t kvh = static_cast<int32_t>(bh % a.kv_heads);
  const int32_t n = __builtin_amdgcn_readfirstlane(a.length(b)), offset = a.lk - a.lq;

  // this wave's queries
  const int32_t unit = first_unit + wave;
  const bool live = unit < units_per_bh;
  const int32_t i0 = live ? unit / a.group * kRows : 0;
  const int32_t h = kvh * a.group + (live ? unit % a.group : 0);
  const int32_t i = i0 + lane % 32;
  int32_t p = i + offset;
  if (!live || i >= a.lq || p < 0 || p >= n) p = -1;
  // positions of the wave's queries that see anything: [p_first, p_last]
  const int32_t p_first = max(i0 + offset, 0);
  const int32_t p_last = live ? min(min(i0 + kRows, a.lq) + offset, n) - 1 : -1;

  // the workgroup's keys: sinks [0, far), then [near, end)
  const int32_t last_unit = min(first_unit + kWaves, units_per_bh) - 1;
  const int32_t g_first = max(first_unit / a.group * kRows + offset, 0);
  const int32_t end = min(min((last_unit / a.group + 1) * kRows, a.lq) + offset, n);
  const int32_t near = max(g_first - a.window + 1, 0);
  const Numbering number(a, near);
  const int32_t far = number.far, skip = number.skip;
  const int32_t count = end > g_first ? far + end - near : 0;

  const S *k_base = static_cast<const S *>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const S *v_base = static_cast<const S *>(a.v) + b * a.vs[0] + kvh * a.vs[2];

  // queries stay in registers; a negative scale moves its sign here, so that
  // the largest product is the largest score
  const float scale = fabsf(a.scale);
  Frag qf[kSteps];
  {
    const S *q = static_cast<const S *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      v4u w = {0, 0, 0, 0};
      const int chunk = 2 * s + half;
      if (p >= 0 && chunk * 16 < a.dim * T::kSize)
        w = *reinterpret_cast<const v4u *>(reinterpret_cast<const char *>(q) + chunk * 16);
      if (a.scale < 0.0f) w ^= Mfma<V>::kSign;
      qf[s] = __builtin_bit_cast(Frag, w);
    }
  }

  RowLoader<V, DP, F::kKeys, kThreads> k_rows, v_rows;
  k_rows.start(a.ks[1], a.dim);
  v_rows.start(a.vs[1], a.dim);
  // one operand's rows of the tile at c0, to LDS
  const auto fetch = [&](const S *base, int64_t stride, const auto &rows, int32_t c0,
                         uint32_t to) {
    if (rows.plain && c0 >= far && c0 + F::kKeys <= count)
      rows.direct(base + (c0 + skip) * stride, lds + to);
    else
      rows.each([&](int row) -> const void * {
        const int32_t c = c0 + row;
        return c < count ? base + number.key(c) * stride : nullptr;
      }, a.dim, lds + to);
  };
  const auto k_tile = [](int parity) { return static_cast<uint32_t>(parity * F::kTile); };
  const auto v_tile = [](int parity) { return static_cast<uint32_t>((2 + parity) * F::kTile); };

  // whether the wave sees any key of the tile at c0: sinks, and [first, last]
  // of the span
  const auto sees = [&](int32_t c0) {
    const int32_t first = max(c0, far) + skip, last = min(c0 + F::kKeys, count) - 1 + skip;
    return c0 < count && p_last >= p_first &&
           (c0 < far || (first <= p_last && (p_first - last < a.window || first < a.sinks)));
  };

  v16f o[DP / 32];
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
  // l: the sum of exponentials; taken: that of what the products take of them, for
  // the residues; of this lane's keys only
  float m = -INFINITY, base = 0.0f, l = 0.0f, taken = 0.0f;

  const auto scores = [&](uint32_t tile, int t, v16f &to) {
#pragma unroll
    for (int r = 0; r < 16; ++r) to[r] = 0.0f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
      to = Mfma<V>::mul(read_rows<V>(lanes, tile, 32 * t, st), qf[st], to);
  };
  const auto exponentials = [&](const v16f &from) {
    float e[16], sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      e[r] = exp2_fast(from[r] * scale - base);
      sum[r % 2] += e[r];
    }
    const Column<V> column(e);
    l += sum[0] + sum[1];
    if constexpr (T::kSize == 2)
      if (a.low != nullptr) taken += rounded_sum(column);
    return column;
  };
  // masks the scores of the tile at c0 and moves the maximum.  It is moved
  // only where it has grown by more than 2^8: until then exponentials up to
  // 2^8 stand beside sums of their own scale.
  const auto settle = [&](int32_t c0, v16f (&x)[F::kSub]) {
    // all of the tile's keys seen by all of the wave's queries: no mask
    const int32_t first = max(c0, far) + skip, last = min(c0 + F::kKeys, count) - 1 + skip;
    const bool whole = c0 + F::kKeys <= count && last <= p_first &&
                       (p_last - first < a.window || last < a.sinks) && p_last - p_first == kRows - 1;
    if (__builtin_amdgcn_readfirstlane(!whole)) {
      const SeenFrom seen(number, p, c0 + 4 * half);
#pragma unroll
      for (int t = 0; t < F::kSub; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          x[t][r] = seen(32 * t + 8 * (r / 4) + r % 4) ? x[t][r] : -INFINITY;
    }
    float tops[2] = {x[0][0], x[0][1]};
#pragma unroll
    for (int t = 0; t < F::kSub; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) tops[r % 2] = fmaxf(tops[r % 2], x[t][r]);
    float top = fmaxf(tops[0], tops[1]);
    top = fmaxf(top, other_half(top)) * scale;
    if (__any(top > m + 8.0f)) {
      const float grown = fmaxf(m, top);
      const float shrink = grown == -INFINITY ? 1.0f : exp2_fast(m - grown);
      m = grown;
      base = m == -INFINITY ? 0.0f : m;
      l *= shrink;
      taken *= shrink;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= shrink;
    }
  };

  const int32_t tiles = (count + F::kKeys - 1) / F::kKeys;
  const int32_t c_begin = item.first(tiles) * F::kKeys, c_end = item.first(tiles, 1) * F::kKeys;
  fetch(k_base, a.ks[1], k_rows, c_begin, k_tile(0));
  fetch(v_base, a.vs[1], v_rows, c_begin, v_tile(0));
  sync_tiles();
  const auto tile = [&](int32_t c0, int parity) __attribute__((always_inline)) {
    if (c0 + F::kKeys < c_end) {  // into the other tiles, which all waves are past
      fetch(k_base, a.ks[1], k_rows, c0 + F::kKeys, k_tile(parity ^ 1));
      fetch(v_base, a.vs[1], v_rows, c0 + F::kKeys, v_tile(parity ^ 1));
    }
    if (sees(c0)) {
      v16f s[F::kSub];
#pragma unroll
      for (int t = 0; t < F::kSub; ++t) scores(k_tile(parity), t, s[t]);
      settle(c0, s);
#pragma unroll
      for (int t = 0; t < F::kSub; ++t)
        mul_transposed<V>(lanes, v_tile(parity), 32 * t, exponentials(s[t]), o);
    }
    sync_tiles();
  };
  for (int32_t c0 = c_begin; c0 < c_end; c0 += 2 * F::kKeys) {
    tile(c0, 0);
    if (c0 + F::kKeys < c_end) tile(c0 + F::kKeys, 1);
  }

  l += other_half(l);
  taken += other_half(taken);
  if (item.slot >= 0) {  // a part: its sums as they are, joined by forward_join
    float *to = sums + ((item.slot * kWaves + wave) * kRows + lane % 32) * F::kStride;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 4)
        *reinterpret_cast<v4f *>(to + dt * 32 + 2 * r + 4 * half) =
            v4f{o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]};
    if (half == 0) {
      to[DP] = m;
      to[DP + 1] = l;
      to[DP + 2] = taken;
    }
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l, better = taken == 0.0f ? 0.0f : 1.0f / taken;
  bool odd = false;  // something is not finite: the row is computed anew
  if (live && i < a.lq) {
    const int64_t at = ((b * a.lq + i) * a.heads + h) * a.dim;
    S *low = a.low != nullptr ? static_cast<S *>(a.low) + a.low_at(b, i, h, 4 * half) : nullptr;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = dt * 32 + 2 * r + 4 * half;
        float x[4], y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = o[dt][r + j] * inv;
          y[j] = o[dt][r + j] * better;
          odd = odd || !(fabsf(x[j]) < INFINITY);
        }
        if (d < a.dim) store_four<V>(x, y, out + at + d, low == nullptr ? nullptr : low + d / 8 * 256);
      }
    if (lse != nullptr && half == 0)
      lse[(b * a.heads + h) * a.lq + i] = l == 0.0f ? INFINITY : m + log2_fast(l);
  }
  uint64_t anew = __ballot(odd && p >= 0);
  anew = (anew | anew >> 32) & 0xffffffffu;
  while (anew != 0) {  // the tiles in LDS are done with: all waves left the loop
    const int r = __builtin_ctzll(anew);
    anew &= anew - 1;
    forward_row<V>(a, b, i0 + r, h, i0 + r + offset, reinterpret_cast<float *>(lds) + wave * DP, out);
  }
}

// The blocks that ran in parts: four values of a row a lane.
template <class V, int DP>
struct JoinShape {
  static constexpr int kLanes = DP <= 32 ? 8 : DP <= 64 ? 16 : 32;  // of a row
  static constexpr int kRows = kThreads / kLanes;                   // of a workgroup
};
template <class V, int DP>
__global__ __launch_bounds__(kThreads) void forward_join(WindowArgs a, int32_t units_per_bh,
                                                         int64_t blocks_per_bh, TailCut cut,
                                                         const float *sums,
                                                         typename V::Storage *out, float *lse) {
  using J = JoinShape<V, DP>;
  constexpr int kStride = ForwardShape<V, DP>::kStride, kPerBlock = kWaves * kRows / J::kRows;
  constexpr int64_t kPart = static_cast<int64_t>(kWaves) * kRows * kStride;
  __shared__ float q_lds[kWaves][DP];
  const int64_t rest = blockIdx.x / kPerBlock, block = cut.whole + rest, bh = block / blocks_per_bh;
  const int32_t in_block = static_cast<int32_t>(blockIdx.x % kPerBlock) * J::kRows + threadIdx.x / J::kLanes;
  const int32_t unit = static_cast<int32_t>(block % blocks_per_bh) * kWaves + in_block / kRows;
  const int64_t b = bh / a.kv_heads;
  const int32_t i = unit / a.group * kRows + in_block % kRows;
  const int32_t h = static_cast<int32_t>(bh % a.kv_heads) * a.group + unit % a.group;
  const int32_t p = i + a.lk - a.lq, d = threadIdx.x % J::kLanes * 4;
  const bool live = unit < units_per_bh && i < a.lq;
  bool odd = false;
  if (live) {
    const float *first = sums + rest * cut.parts * kPart + in_block * kStride;
    float m = -INFINITY, l = 0.0f, taken = 0.0f, o[4] = {}, better[4];
#pragma unroll 4
    for (int32_t part = 0; part < cut.parts; ++part) m = fmaxf(m, first[part * kPart + DP]);
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll 4
    for (int32_t part = 0; part < cut.parts; ++part) {
      const float *from = first + part * kPart;
      const float f = exp2_fast(from[DP] - base);
      l += from[DP + 1] * f;
      taken += from[DP + 2] * f;
      const v4f x = *reinterpret_cast<const v4f *>(from + min(d, DP - 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += x[j] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      better[j] = taken == 0.0f ? 0.0f : o[j] / taken;
      o[j] *= inv;
      odd = odd || (d < a.dim && !(fabsf(o[j]) < INFINITY));
    }
    if (d < a.dim) {
      const int64_t at = ((b * a.lq + i) * a.heads + h) * a.dim + d;
      store_four<V>(o, better, out + at, a.low == nullptr ? nullptr : static_cast<typename V::Storage *>(a.low) + a.low_at(b, i, h, d));
    }
    if (lse != nullptr && d == 0)
      lse[(b * a.heads + h) * a.lq + i] = l == 0.0f ? INFINITY : m + log2_fast(l);
  }
  uint64_t anew = __ballot(odd && p >= 0 && p < a.length(b));
  while (anew != 0) {
    const int row = __builtin_ctzll(anew) / J::kLanes;  // of the wave's
    anew &= ~(((uint64_t{1} << J::kLanes) - 1) << (row * J::kLanes));
    const int at = row * J::kLanes;
    forward_row<V>(a, b, __shfl(i, at), __shfl(h, at), __shfl(p, at), q_lds[threadIdx.x / kWave], out);
  }
}

// Blocks of queries and how they are cut.
struct Grid {
  int64_t units, per_bh;
  TailCut cut;
};

template <class V, int DP>
Grid grid_of(const WindowArgs &a) {
  using F = ForwardShape<V, DP>;
  Grid g;
  g.units = (static_cast<int64_t>(a.lq) + kRows - 1) / kRows * a.group;
  g.per_bh = (g.units + kWaves - 1) / kWaves;
  const int64_t keys = std::min<int64_t>(a.lk, static_cast<int64_t>(a.window) + a.sinks + kRows);
  g.cut = cut_tail(g.per_bh * a.batch * a.kv_heads, 256 * F::kBlocks, (keys + F::kKeys - 1) / F::kKeys,
                   join_cost(F::T::kSize == 4));
  return g;
}

template <class V, int DP>
msx_status run(const WindowArgs &a, void *out, float *lse, float *sums, size_t *bytes,
               hipStream_t stream) {
  const Grid g = grid_of<V, DP>(a);
  const int64_t rows = g.cut.rest * kWaves * kRows;
  if (bytes != nullptr) {
    *bytes = sizeof(float) * static_cast<size_t>(rows * g.cut.parts) * ForwardShape<V, DP>::kStride;
    return MSX_OK;
  }
  if (g.units > 0x7fffffff || std::max(g.cut.items(), rows / JoinShape<V, DP>::kRows) > max_blocks(kThreads))
    return fail(MSX_EINVAL, "window_attention has more rows than a grid holds.");
  auto *to = static_cast<typename V::Storage *>(out);
  forward_tiles<V, DP><<<static_cast<unsigned>(g.cut.items()), kThreads, 0, stream>>>(
      a, static_cast<int32_t>(g.units), g.per_bh, g.cut, to, lse, sums);
  if (rows > 0)
    forward_join<V, DP><<<static_cast<unsigned>(rows / JoinShape<V, DP>::kRows), kThreads, 0, stream>>>(
        a, static_cast<int32_t>(g.units), g.per_bh, g.cut, sums, to, lse);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "window_attention");
}

template <class V>
msx_status by_dim(const WindowArgs &a, void *out, float *lse, float *sums, size_t *bytes,
                  hipStream_t stream) {
  if (a.dim <= 32) return run<V, 32>(a, out, lse, sums, bytes, stream);
  if (a.dim <= 64) return run<V, 64>(a, out, lse, sums, bytes, stream);
  if (a.dim <= 96) return run<V, 96>(a, out, lse, sums, bytes, stream);
  return run<V, 128>(a, out, lse, sums, bytes, stream);
}

msx_status by_type(msx_vtype vt, const WindowArgs &a, void *out, float *lse, float *sums,
                   size_t *bytes, hipStream_t stream) {
  switch (vt) {
  case MSX_F32: return by_dim<F32>(a, out, lse, sums, bytes, stream);
  case MSX_F16: return by_dim<F16>(a, out, lse, sums, bytes, stream);
  default: return by_dim<BF16>(a, out, lse, sums, bytes, stream);
  }
}

}  // namespace

size_t window_forward_scratch(msx_vtype vt, const WindowArgs &a) {
  size_t bytes = 0;
  by_type(vt, a, nullptr, nullptr, nullptr, &bytes, nullptr);
  return bytes;
}

msx_status launch_window_forward(msx_vtype vt, const WindowArgs &a, void *out, float *lse,
                                 void *scratch, hipStream_t stream) {
  return by_type(vt, a, out, lse, static_cast<float *>(scratch), nullptr, stream);
}

}  // namespace msx
