// window_backward.hip - window attention's gradients on the matrix cores, for
// the operands the forward tiles take.
//
// Two sums over the same products, each in a fixed order and without atomics:
//
//   queries (dq): a wave takes 32 queries, as in the forward pass, and goes
//     through their keys: S^T = K Q^T, dP^T = V dO^T, dQ^T += K^T dS^T;
//   keys (dk, dv): a wave takes 32 keys, its workgroup 128, and goes through
//     the queries that see them, of every head of the group: S = Q K^T,
//     dP = dO V^T (rows are queries now), dV^T += dO^T P, dK^T += Q^T dS.
//
// The products of scores are made twice, seven in all where five would do with
// dq added atomically in float32; the rounding order would then change from
// run to run, and dq would pass through memory in 32 bits.
//
// Sinks are seen by all later queries, L of them where another key has
// `window`: the queries beyond a key block's own span are a pass of their own
// (the far pass), whose four waves take different queries for the same 32
// keys; its parts and the blocks' own sums are joined in order.
//
// P and dS are rounded to the operands' 16 bits for their products, as matrix
// instructions take them; each sum over them stays float32, and gradients are
// rounded once.  dS = P (dP - delta) is small beside dP and delta where P is
// nearly one, so delta = grad.out takes out with its residue, 32 bits in all
// (with out as rounded alone, dq of a head that keeps 98 % of its attention on
// one key was 39 % off in bfloat16, 5 % in float16; now 0.24 and 0.03 %).  Residues
// cost a step of 4 x 2,048 tokens 6 %, one of 16,384 5 %.
//
// Bound like the forward pass by products, exponentials and LDS reads taking
// turns; the products are under way a third of the time.  16,384 tokens of 16
// heads of 128 on 8, a window of 1,024: queries 277 us, keys 327 (790 and 840
// TFLOP/s of what they multiply), sinks 29, joining 9.
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
constexpr int kBlockKeys = 32 * kWaves;

struct Upstream {
  const void *grad;
  int64_t gs[3];
  const void *out;
  const float *lse;
  float *delta;
};

template <class V, int DP>
struct BackwardShape {
  using T = TileShape<V, DP>;
  static constexpr int kSub = T::kSize == 2 ? 2 : 1;
  static constexpr int kTokens = 32 * kSub;  // tokens of a tile
  static constexpr int kTile = kTokens * T::kPitch;
};

// float16 holds 2^-24 to 65504, gradients of scores much more: dS = P (dP -
// delta) is a thousandth of the upstream gradient where a thousand keys share
// a query, and a product of 128 terms of it where loss scaling is at work.  So the
// products take dS 2^exponent larger, a column of sums (a query of dq, a key of
// dk) with an exponent of its own: high at first, and lowered, with the sums so
// far, where the column's largest value would pass 2^15.  What is lost then is
// below 2^-31 of that.  P of the keys' pass, one at most, is taken 2^14 larger.
// The other types have float32's range: nothing is done there.
// (Unlifted, dq of 1,500 tokens was 1.0 % off at upstream gradients of 2^-14 and
// 7.9 % at 2^-17, where rounding it once costs 0.3 and 2.5.  The maxima cost 5 %
// of a backward pass at heads of 128, 11 at 64, 18 at 32.)
template <class V>
struct Lift {
  static constexpr bool kOn = V::kType == MSX_F16;
  static constexpr int kP = kOn ? 14 : 0, kStart = kOn ? 40 : 0;
  float up = kOn ? 0x1p40f : 1.0f;  // 2^exponent

  // Of a lane's part of a column of dS (the other is the lane's 32 away);
  // returns by how much the exponent fell.
  template <int kBlocks>
  __device__ __forceinline__ float fit(float (&ds)[16], v16f (&acc)[kBlocks]) {
    float fell = 0.0f;
    if constexpr (kOn) {
      float top[2] = {0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < 16; ++r) top[r % 2] = fmaxf(top[r % 2], fabsf(ds[r]));
      top[0] = fmaxf(top[0], top[1]);
      if (__any(top[0] > 0x1p15f)) {
        // to [2^7, 2^8), so that it seldom passes again; an infinity stays one
        top[0] = fmaxf(top[0], other_half(top[0]));
        const int over =
            top[0] > 0x1p15f ? static_cast<int>(__builtin_bit_cast(uint32_t, top[0]) >> 23) - 127 - 7 : 0;
        fell = static_cast<float>(over);
        const float shrink = __builtin_ldexpf(1.0f, -over);
        up *= shrink;
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] *= shrink;
#pragma unroll
        for (int dt = 0; dt < kBlocks; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[dt][r] *= shrink;
      }
    }
    return fell;
  }
};

template <int kBlocks>
__device__ __forceinline__ void multiply(v16f (&acc)[kBlocks], float factor) {
#pragma unroll
  for (int dt = 0; dt < kBlocks; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] *= factor;
}

// Sixteen bytes of a row, zeros beyond the head.
template <class V>
__device__ __forceinline__ v4u load_chunk(const typename V::Storage *row, int chunk, int dim) {
  if (chunk * 16 >= dim * static_cast<int>(sizeof(typename V::Storage))) return v4u{0, 0, 0, 0};
  return *reinterpret_cast<const v4u *>(reinterpret_cast<const char *>(row) + chunk * 16);
}

// Sum of products of two sixteen-byte pieces.
template <class V>
__device__ __forceinline__ float dot_chunk(v4u x, v4u y) {
  float acc = 0.0f;
  if constexpr (sizeof(typename V::Storage) == 4) {
    const auto a = __builtin_bit_cast(v4f, x), b = __builtin_bit_cast(v4f, y);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc += a[j] * b[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc += V::widen(static_cast<uint16_t>(x[j])) * V::widen(static_cast<uint16_t>(y[j]));
      acc += V::widen(static_cast<uint16_t>(x[j] >> 16)) * V::widen(static_cast<uint16_t>(y[j] >> 16));
    }
  }
  return acc;
}

// A lane's column of a transposed result: row `to` gets acc * factor.
template <class V, int DP>
__device__ __forceinline__ void store_column(const v16f (&acc)[DP / 32], float factor, int dim,
                                    typename V::Storage *to) {
  const int half = (threadIdx.x % kWave) / 32;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = dt * 32 + 2 * r + 4 * half;
      if (d >= dim) continue;
      const float x0 = acc[dt][r] * factor, x1 = acc[dt][r + 1] * factor;
      const float x2 = acc[dt][r + 2] * factor, x3 = acc[dt][r + 3] * factor;
      if constexpr (sizeof(typename V::Storage) == 2)
        *reinterpret_cast<v2u *>(to + d) = v2u{Mfma<V>::pack(x0, x1), Mfma<V>::pack(x2, x3)};
      else
        *reinterpret_cast<v4f *>(to + d) = v4f{x0, x1, x2, x3};
    }
}

template <int DP>
__device__ __forceinline__ void zero(v16f (&acc)[DP / 32]) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[dt][r] = 0.0f;
}

// The same as sums in scratch.
template <int DP>
__device__ __forceinline__ void store_sums(const v16f (&acc)[DP / 32], int dim, float *to) {
  const int half = (threadIdx.x % kWave) / 32;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = dt * 32 + 2 * r + 4 * half;
      if (d < dim)
        *reinterpret_cast<v4f *>(to + d) = v4f{acc[dt][r], acc[dt][r + 1], acc[dt][r + 2], acc[dt][r + 3]};
    }
}

// ---------------------------------------------------------------------------
// dq, and delta for the keys' pass.

// Blocks of 4 x 32 query rows of one key-value head, and how they are cut.
struct QueryPlan {
  int64_t units, per_bh;
  TailCut cut;
  float *sums;  // of the parts
};

template <class V, int DP>
__global__ __launch_bounds__(kThreads, (sizeof(typename V::Storage) == 4 && DP > 64 ? 1 : 2)) void
backward_queries(WindowArgs a, Upstream up, QueryPlan plan, typename V::Storage *dq) {
  using S = typename V::Storage;
  using T = TileShape<V, DP>;
  using F = BackwardShape<V, DP>;
  using Frag = typename Mfma<V>::Frag;
  constexpr int kSteps = DP / Mfma<V>::kDepth;
  __shared__ __attribute__((aligned(1024))) char lds[4 * F::kTile];
  const TileLanes<V, DP> lanes(lds);

  const int lane = threadIdx.x % kWave, half = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const CutItem item(plan.cut, blockIdx.x);
  const int32_t units_per_bh = static_cast<int32_t>(plan.units);
  const uint32_t per_bh = static_cast<uint32_t>(plan.per_bh), bh = item.block / per_bh;
  const int32_t first_unit = static_cast<int32_t>(item.block % per_bh) * kWaves;
  const int64_t b = bh / a.kv_heads;
  const int32_t kvh = static_cast<int32_t>(bh % a.kv_heads);
  const int32_t n = __builtin_amdgcn_readfirstlane(a.length(b)), offset = a.lk - a.lq;

  // units, spans and numbering of keys as in the forward pass
  const int32_t unit = first_unit + wave;
  const bool live = unit < units_per_bh;
  const int32_t i0 = live ? unit / a.group * 32 : 0;
  const int32_t h = kvh * a.group + (live ? unit % a.group : 0);
  const int32_t i = i0 + lane % 32;
  int32_t p = i + offset;
  if (!live || i >= a.lq || p < 0 || p >= n) p = -1;
  const int32_t p_first = max(i0 + offset, 0);
  const int32_t p_last = live ? min(min(i0 + 32, a.lq) + offset, n) - 1 : -1;
  const int32_t last_unit = min(first_unit + kWaves, units_per_bh) - 1;
  const int32_t g_first = max(first_unit / a.group * 32 + offset, 0);
  const int32_t end = min(min((last_unit / a.group + 1) * 32, a.lq) + offset, n);
  const int32_t near = max(g_first - a.window + 1, 0);
  const Numbering number(a, near);
  const int32_t far = number.far, skip = number.skip;
  const int32_t count = end > g_first ? far + end - near : 0;

  const S *k_base = static_cast<const S *>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const S *v_base = static_cast<const S *>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  Frag qf[kSteps], gf[kSteps];
  float delta = 0.0f, lse = INFINITY;
  {
    const S *q = static_cast<const S *>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
    const S *g = static_cast<const S *>(up.grad) + b * up.gs[0] + i * up.gs[1] + h * up.gs[2];
    const int64_t at = ((b * a.lq + i) * a.heads + h) * a.dim;
    const S *o = static_cast<const S *>(up.out) + at;
    const S *low = a.low == nullptr ? nullptr : static_cast<const S *>(a.low) + a.low_at(b, i, h, 0);
    float residue = 0.0f;
    if (p >= 0) lse = up.lse[(b * a.heads + h) * a.lq + i];
    if (lse == INFINITY) p = -1;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      v4u qw = {0, 0, 0, 0}, gw = {0, 0, 0, 0};
      if (p >= 0) {
        qw = load_chunk<V>(q, 2 * s + half, a.dim);
        gw = load_chunk<V>(g, 2 * s + half, a.dim);
        delta += dot_chunk<V>(gw, load_chunk<V>(o, 2 * s + half, a.dim));
        if constexpr (T::kSize == 2)
          if (low != nullptr) {
            const int chunk = 2 * s + half;
            if (chunk * 8 < a.dim)
              residue += dot_chunk<V>(gw, *reinterpret_cast<const v4u *>(low + chunk * 256));
          }
      }
      qf[s] = __builtin_bit_cast(Frag, qw);
      gf[s] = __builtin_bit_cast(Frag, gw);
    }
    delta += residue * (1.0f / Residue<V>::kUp);
    delta += other_half(delta);
  }

  RowLoader<V, DP, F::kTokens, kThreads> k_rows, v_rows;
  k_rows.start(a.ks[1], a.dim);
  v_rows.start(a.vs[1], a.dim);
  const auto fetch = [&](const S *base, int64_t stride, const auto &rows, int32_t c0, uint32_t to) {
    if (rows.plain && c0 >= far && c0 + F::kTokens <= count)
      rows.direct(base + (c0 + skip) * stride, lds + to);
    else
      rows.each([&](int row) -> const void * {
        const int32_t c = c0 + row;
        return c < count ? base + number.key(c) * stride : nullptr;
      }, a.dim, lds + to);
  };
  const auto k_tile = [](int parity) { return static_cast<uint32_t>(parity * F::kTile); };
  const auto v_tile = [](int parity) { return static_cast<uint32_t>((2 + parity) * F::kTile); };

  v16f acc[DP / 32];
  zero<DP>(acc);
  Lift<V> lift;
  float base = lse - Lift<V>::kStart;  // of lifted probabilities
  const int32_t tiles = (count + F::kTokens - 1) / F::kTokens;
  const int32_t c_begin = item.first(tiles) * F::kTokens, c_end = item.first(tiles, 1) * F::kTokens;
  // whether the wave sees any key of the tile at c0, and whether all of its
  // queries see all of them
  const auto sees = [&](int32_t c0, bool &whole) {
    const int32_t first = max(c0, far) + skip, last = min(c0 + F::kTokens, count) - 1 + skip;
    whole = c0 + F::kTokens <= count && last <= p_first &&
            (p_last - first < a.window || last < a.sinks) && p_last - p_first == 31;
    return p_last >= p_first &&
           (c0 < far || (first <= p_last && (p_first - last < a.window || first < a.sinks)));
  };
  const auto products = [&](int parity, int t, v16f &s, v16f &dp) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      s = Mfma<V>::mul(read_rows<V>(lanes, k_tile(parity), 32 * t, st), qf[st], s);
      dp = Mfma<V>::mul(read_rows<V>(lanes, v_tile(parity), 32 * t, st), gf[st], dp);
    }
  };
  // delta so far is of outputs whose sums took rounded probabilities.  A span of
  // one or two tiles is in LDS as a whole, and delta the sum of P dP over it
  // with P in 32 bits: up to 3 % less error there, for 0.5 % of a pass.
  int32_t held = -1;  // the tile in the first buffer
  if (T::kSize == 2 && count <= 2 * F::kTokens) {
    held = 0;
    fetch(k_base, a.ks[1], k_rows, 0, k_tile(0));
    fetch(v_base, a.vs[1], v_rows, 0, v_tile(0));
    if (count > F::kTokens) {
      fetch(k_base, a.ks[1], k_rows, F::kTokens, k_tile(1));
      fetch(v_base, a.vs[1], v_rows, F::kTokens, v_tile(1));
    }
    sync_tiles();
    delta = 0.0f;
#pragma unroll 1
    for (int at = 0; at * F::kTokens < count; ++at) {
      bool whole;
      if (!sees(at * F::kTokens, whole)) continue;
#pragma unroll 1
      for (int t = 0; t < F::kSub; ++t) {
        v16f s, dp;
        products(at, t, s, dp);
        const SeenFrom seen(number, p, at * F::kTokens + 32 * t + 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          delta += seen(8 * (r / 4) + r % 4) ? exp2_fast(s[r] * a.scale - lse) * dp[r] : 0.0f;
      }
    }
    delta += other_half(delta);
    sync_tiles();
  }
  if (held != c_begin) {
    fetch(k_base, a.ks[1], k_rows, c_begin, k_tile(0));
    fetch(v_base, a.vs[1], v_rows, c_begin, v_tile(0));
    sync_tiles();
  }
  if (live && i < a.lq && half == 0 && item.part == 0) up.delta[(b * a.heads + h) * a.lq + i] = delta;
  const auto tile = [&](int32_t c0, int parity) __attribute__((always_inline)) {
    if (c0 + F::kTokens < c_end) {  // into the other tiles, which all waves are past
      fetch(k_base, a.ks[1], k_rows, c0 + F::kTokens, k_tile(parity ^ 1));
      fetch(v_base, a.vs[1], v_rows, c0 + F::kTokens, v_tile(parity ^ 1));
    }
    bool whole;
    if (sees(c0, whole)) {
#pragma unroll
      for (int t = 0; t < F::kSub; ++t) {
        v16f s, dp;
        products(parity, t, s, dp);
        float ds[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = exp2_fast(s[r] * a.scale - base) * (dp[r] - delta);
        if (__builtin_amdgcn_readfirstlane(!whole)) {
          const SeenFrom seen(number, p, c0 + 32 * t + 4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] = seen(8 * (r / 4) + r % 4) ? ds[r] : 0.0f;
        }
        if constexpr (Lift<V>::kOn) {
          base += lift.fit(ds, acc);
        }
        mul_transposed<V>(lanes, k_tile(parity), 32 * t, Column<V>(ds), acc);
      }
    }
    sync_tiles();
  };
  for (int32_t c0 = c_begin; c0 < c_end; c0 += 2 * F::kTokens) {
    tile(c0, 0);
    if (c0 + F::kTokens < c_end) tile(c0 + F::kTokens, 1);
  }
  if (!live || i >= a.lq) return;
  if constexpr (Lift<V>::kOn) multiply(acc, 1.0f / lift.up);
  if (item.slot >= 0)  // a part: its sums as they are, joined by join_sums
    store_sums<DP>(acc, a.dim, plan.sums + ((item.slot * kWaves + wave) * 32 + lane % 32) * a.dim);
  else
    store_column<V, DP>(acc, a.grad_scale, a.dim, dq + ((b * a.lq + i) * a.heads + h) * a.dim);
}

// ---------------------------------------------------------------------------
// dk and dv.

// The sums of one wave's 32 keys.  Its keys and values stay in registers, or
// (kInLds) in LDS at the tiles' layout, where registers are short.
template <class V, int DP, bool kInLds>
struct KeyWave {
  using Frag = typename Mfma<V>::Frag;
  static constexpr int kSteps = DP / Mfma<V>::kDepth;
  Frag kf[kInLds ? 1 : kSteps], vf[kInLds ? 1 : kSteps];
  uint32_t k_tile, v_tile;  // with kInLds
  int key_row;               // of the tiles, the wave's first
  v16f dk[DP / 32], dv[DP / 32];
  Lift<V> lift;  // of dk's column

  __device__ __forceinline__ void start(const WindowArgs &a, int64_t b, int32_t kvh, int32_t key, bool live) {
    using S = typename V::Storage;
    const int half = (threadIdx.x % kWave) / 32;
    zero<DP>(dk);
    zero<DP>(dv);
    if constexpr (!kInLds) {
      const S *k = static_cast<const S *>(a.k) + b * a.ks[0] + key * a.ks[1] + kvh * a.ks[2];
      const S *v = static_cast<const S *>(a.v) + b * a.vs[0] + key * a.vs[1] + kvh * a.vs[2];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        v4u kw = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
        if (live) {
          kw = load_chunk<V>(k, 2 * s + half, a.dim);
          vw = load_chunk<V>(v, 2 * s + half, a.dim);
        }
        kf[s] = __builtin_bit_cast(Frag, kw);
        vf[s] = __builtin_bit_cast(Frag, vw);
      }
    }
  }
  __device__ __forceinline__ Frag key_frag(const TilePlaces<V, DP> &lanes, int s) const {
    if constexpr (kInLds) return read_rows<V>(lanes, k_tile, key_row, s);
    else return kf[s];
  }
  __device__ __forceinline__ Frag value_frag(const TilePlaces<V, DP> &lanes, int s) const {
    if constexpr (kInLds) return read_rows<V>(lanes, v_tile, key_row, s);
    else return vf[s];
  }

  // 32 queries from row `row0` of the tiles, at positions p0 .. p0 + 31;
  // `masked`: the lane's key is not seen by all of them.
  __device__ __forceinline__ void add(const WindowArgs &a, const TilePlaces<V, DP> &lanes, uint32_t q_tile,
                             uint32_t g_tile, const float *lse, const float *delta, int row0,
                             int32_t p0, int32_t key, bool masked) {
    const int lane = threadIdx.x % kWave, half = lane / 32;
    v16f s, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      s = Mfma<V>::mul(read_rows<V>(lanes, q_tile, row0, st), key_frag(lanes, st), s);
      dp = Mfma<V>::mul(read_rows<V>(lanes, g_tile, row0, st), value_frag(lanes, st), dp);
    }
    float p[16], ds[16];
    [[maybe_unused]] const float up = lift.up * __builtin_ldexpf(1.0f, -Lift<V>::kP);
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int row = row0 + 2 * r + 4 * half;
      const v4f l = *reinterpret_cast<const v4f *>(lse + row);
      const v4f d = *reinterpret_cast<const v4f *>(delta + row);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[r + j] = exp2_fast(s[r + j] * a.scale - l[j]);
        if constexpr (Lift<V>::kOn)
          ds[r + j] = p[r + j] * __builtin_fmaf(dp[r + j], up, -(d[j] * up));
        else
          ds[r + j] = p[r + j] * (dp[r + j] - d[j]);
      }
    }
    if (masked) {
      const uint32_t limit = key < a.sinks ? 0x7fffffff : a.window;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t back = static_cast<uint32_t>(p0 + 8 * (r / 4) + 4 * half + r % 4 - key);
        p[r] = back < limit ? p[r] : 0.0f;
        ds[r] = back < limit ? ds[r] : 0.0f;
      }
    }
    lift.fit(ds, dk);
    mul_transposed<V>(lanes, g_tile, row0, Column<V>(p), dv);
    mul_transposed<V>(lanes, q_tile, row0, Column<V>(ds), dk);
  }
  // The sums as they are.
  __device__ __forceinline__ void finish() {
    if constexpr (Lift<V>::kOn) {
      multiply(dk, 1.0f / lift.up);
      multiply(dv, __builtin_ldexpf(1.0f, -Lift<V>::kP));
    }
  }
};

// Queries of the walk in LDS: q, the upstream gradient, lse and delta.  A query
// beyond the sequence is zeros with lse = +inf: its P is zero.  lse is held as
// the lifted P takes it.
template <class V, int DP, int kTokens, int kThreads>
struct QueryTile {
  using T = TileShape<V, DP>;
  static constexpr int kTile = kTokens * T::kPitch;
  static constexpr int kBytes = 2 * kTile + 2 * kTokens * 4;
  float stat;
  RowLoader<V, DP, kTokens, kThreads> q_rows, g_rows;

  __device__ __forceinline__ void start(const WindowArgs &a, const Upstream &up) {
    q_rows.start(a.qs[1], a.dim);
    g_rows.start(up.gs[1], a.dim);
  }
  // The rows are on their way to `to`; the statistics wait for keep.
  __device__ __forceinline__ void fetch(const WindowArgs &a, const Upstream &up, int64_t b, int32_t h,
                               int32_t p0, int32_t last, int32_t offset, char *to) {
    using S = typename V::Storage;
    const S *q = static_cast<const S *>(a.q) + b * a.qs[0] + h * a.qs[2];
    const S *g = static_cast<const S *>(up.grad) + b * up.gs[0] + h * up.gs[2];
    const int64_t first = p0 - offset;
    if (q_rows.plain && g_rows.plain && p0 + kTokens - 1 <= last) {
      q_rows.direct(q + first * a.qs[1], to);
      g_rows.direct(g + first * up.gs[1], to + kTile);
    } else {
      q_rows.each([&](int row) -> const void * {
        return p0 + row <= last ? q + (first + row) * a.qs[1] : nullptr;
      }, a.dim, to);
      g_rows.each([&](int row) -> const void * {
        return p0 + row <= last ? g + (first + row) * up.gs[1] : nullptr;
      }, a.dim, to + kTile);
    }
    // the first kTokens threads take lse, the next as many delta
    static_assert(2 * kTokens <= kThreads, "a thread a statistic");
    const int row = threadIdx.x % kTokens;
    const bool is_lse = threadIdx.x < kTokens;
    stat = is_lse ? INFINITY : 0.0f;
    if (threadIdx.x < 2 * kTokens && p0 + row <= last) {
      const int64_t at = (b * a.heads + h) * a.lq + first + row;
      stat = is_lse ? up.lse[at] - Lift<V>::kP : up.delta[at];
    }
  }
  __device__ __forceinline__ void keep(char *to) const {
    if (threadIdx.x < 2 * kTokens)
      reinterpret_cast<float *>(to + 2 * kTile)[threadIdx.x] = stat;
  }
};

// How the keys' work is cut: blocks of kBlockKeys keys as in the forward pass,
// and the far units, 32 sink keys each, in `far_parts`.  The sums of blocks in
// parts and those of far units go through scratch.
struct KeyPlan {
  int32_t blocks;  // of a key-value head
  TailCut cut;
  int32_t far_units, far_parts;
  float *part_sums, *unit_sums, *far_sums;  // parts, far units of whole blocks, the far pass
};

// Queries within reach of a block's window: positions first .. last; the rest
// of a sink's queries are the far pass's.
__device__ __forceinline__ int32_t near_last(const WindowArgs &a, int32_t block, int32_t n) {
  const int64_t last = static_cast<int64_t>(block) * kBlockKeys + kBlockKeys + a.window - 2;
  return last < n - 1 ? static_cast<int32_t>(last) : n - 1;
}

// The near pass's workgroup.  Sums of 128 values a key leave room for one wave
// a SIMD if keys and values stay in registers too, which waits on LDS and
// products in turn: 16-bit heads above 64 keep them in LDS, and eight waves,
// two for the same keys, take alternate halves of a tile (16,384 tokens of 16
// heads of 128, a window of 1,024: 476 us with one wave a SIMD, 384 with two;
// 421 with TileLanes' addresses, which leave fewer registers to reads).
template <class V, int DP>
struct NearShape {
  using T = TileShape<V, DP>;
  static constexpr bool kInLds = T::kSize == 2 && DP > 64;
  static constexpr int kGroups = kInLds ? 2 : 1;  // waves of the same keys
  static constexpr int kThreads = kGroups * kWaves * kWave;
  // all but wide float32 heads fit twice (at 64: 3 to 7 % of a backward pass;
  // a third wave spills, 145 us become 204).  float32 heads of 128 do not fit once:
  // 17 registers spill here and 42 in the far pass (4,096 tokens, 8 heads on 2,
  // window 1,024: a training step 891 us, 178 in bfloat16)
  static constexpr int kWavesASimd = kInLds || DP <= 64 ? 2 : 1;
  static constexpr int kSub = T::kSize == 2 ? 2 : 1, kTokens = 32 * kSub;
  using Tile = QueryTile<V, DP, kTokens, kThreads>;
  static constexpr int kKeyBytes = kInLds ? 2 * kBlockKeys * T::kPitch : 0;
  static constexpr int kSums = kInLds ? kWaves * kWave * DP / 2 * 4 : 0;  // of four waves, dk or dv
  static constexpr int kLds = std::max(kKeyBytes + 2 * Tile::kBytes, kSums);
};

template <class V, int DP>
__global__ __launch_bounds__((NearShape<V, DP>::kThreads), (NearShape<V, DP>::kWavesASimd)) void
backward_keys_near(WindowArgs a, Upstream up, KeyPlan plan, typename V::Storage *dk,
                   typename V::Storage *dv) {
  using S = typename V::Storage;
  using N = NearShape<V, DP>;
  using T = TileShape<V, DP>;
  using Tile = typename N::Tile;
  constexpr int kSub = N::kSub, kTokens = N::kTokens;
  __shared__ __attribute__((aligned(1024))) char lds[N::kLds];
  const TilePlaces<V, DP> lanes(lds);

  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int keys_of = wave % kWaves, group = wave / kWaves;
  const CutItem item(plan.cut, blockIdx.x);
  const int32_t block = static_cast<int32_t>(item.block % plan.blocks);
  const uint32_t head = item.block / plan.blocks;
  const int64_t bh = head, b = head / a.kv_heads;
  const int32_t kvh = static_cast<int32_t>(head % a.kv_heads);
  const int32_t n = __builtin_amdgcn_readfirstlane(a.length(b)), offset = a.lk - a.lq;
  const int32_t w_first = block * kBlockKeys + keys_of * 32, w_last = w_first + 31;
  const int32_t key = w_first + lane % 32;

  KeyWave<V, DP, N::kInLds> keys;
  keys.start(a, b, kvh, key, key < n);
  if constexpr (N::kInLds) {
    keys.k_tile = 0;
    keys.v_tile = kBlockKeys * T::kPitch;
    keys.key_row = keys_of * 32;
    const S *k = static_cast<const S *>(a.k) + b * a.ks[0] + kvh * a.ks[2];
    const S *v = static_cast<const S *>(a.v) + b * a.vs[0] + kvh * a.vs[2];
    for (int at = threadIdx.x; at < kBlockKeys * T::kUsed; at += N::kThreads) {
      const int row = at / T::kUsed, chunk = at % T::kUsed;
      const int64_t j = block * kBlockKeys + row;
      v4u kw = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
      if (j < n) {
        kw = load_chunk<V>(k + j * a.ks[1], chunk, a.dim);
        vw = load_chunk<V>(v + j * a.vs[1], chunk, a.dim);
      }
      *reinterpret_cast<v4u *>(lds + T::along(row, chunk)) = kw;
      *reinterpret_cast<v4u *>(lds + kBlockKeys * T::kPitch + T::along(row, chunk)) = vw;
    }
  }

  const int32_t first = max(block * kBlockKeys, offset), last = near_last(a, block, n);
  const int32_t tiles = last >= first ? (last - first) / kTokens + 1 : 0;
  const int64_t total = static_cast<int64_t>(tiles) * a.group;
  const int32_t begin = static_cast<int32_t>(item.parts == 1 ? 0 : total * item.part / item.parts);
  const int32_t end = static_cast<int32_t>(item.parts == 1 ? total : total * (item.part + 1) / item.parts);

  Tile next;
  next.start(a, up);
  const auto tile_at = [](int parity) { return static_cast<uint32_t>(N::kKeyBytes + parity * Tile::kBytes); };
  const auto fetch = [&](int32_t step, int parity) {
    next.fetch(a, up, b, kvh * a.group + step / tiles, first + step % tiles * kTokens, last, offset,
               lds + tile_at(parity));
  };
  if (begin < end) {
    fetch(begin, 0);
    next.keep(lds + tile_at(0));
  }
  sync_tiles();
  const auto walk = [&](int32_t step, int parity) __attribute__((always_inline)) {
    const bool more = step + 1 < end;
    if (more) fetch(step + 1, parity ^ 1);  // into the other tile, which all waves are past
    const uint32_t tile = tile_at(parity);
    const float *stat = reinterpret_cast<const float *>(lds + tile + 2 * Tile::kTile);
#pragma unroll
    for (int t0 = 0; t0 < kSub; t0 += N::kGroups) {
      const int t = t0 + group;
      const int32_t p0 = first + step % tiles * kTokens + 32 * t, p1 = p0 + 31;
      const bool any = p1 >= w_first && p0 <= last && (p0 - w_last < a.window || w_first < a.sinks);
      const bool whole = p0 >= w_last && (p1 - w_first < a.window || w_last < a.sinks);
      if (any)
        keys.add(a, lanes, tile, tile + Tile::kTile, stat, stat + kTokens, 32 * t, p0, key,
                 __builtin_amdgcn_readfirstlane(!whole));
    }
    if (more) next.keep(lds + tile_at(parity ^ 1));
    sync_tiles();
  };
#pragma unroll 1
  for (int32_t step = begin; step < end; ++step) walk(step, (step - begin) & 1);
  keys.finish();

  if constexpr (N::kGroups == 2) {  // the second wave's sums to the first: dk, then dv
    float *sums = reinterpret_cast<float *>(lds) + (keys_of * kWave + lane) * 4;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      v16f(&mine)[DP / 32] = which == 0 ? keys.dk : keys.dv;
      if (which == 1) sync_tiles();
      if (group == 1) {
#pragma unroll
        for (int r = 0; r < DP / 2; r += 4)
          *reinterpret_cast<v4f *>(sums + r * kWaves * kWave) =
              v4f{mine[r / 16][r % 16], mine[r / 16][r % 16 + 1], mine[r / 16][r % 16 + 2],
                  mine[r / 16][r % 16 + 3]};
      }
      sync_tiles();
      if (group == 0) {
#pragma unroll
        for (int r = 0; r < DP / 2; r += 4) {
          const v4f other = *reinterpret_cast<const v4f *>(sums + r * kWaves * kWave);
#pragma unroll
          for (int j = 0; j < 4; ++j) mine[r / 16][r % 16 + j] += other[j];
        }
      }
    }
    if (group == 1) return;
  }

  if (key >= a.lk) return;
  const int32_t unit = block * kWaves + keys_of;
  if (item.slot >= 0 || unit < plan.far_units) {
    const int64_t slot = item.slot >= 0 ? item.slot * kWaves + keys_of : bh * plan.far_units + unit;
    float *to = (item.slot >= 0 ? plan.part_sums : plan.unit_sums) + (slot * 32 + lane % 32) * 2 * a.dim;
    store_sums<DP>(keys.dk, a.dim, to);
    store_sums<DP>(keys.dv, a.dim, to + a.dim);
  } else {
    const int64_t row = (b * a.lk + key) * a.kv_heads + kvh;
    store_column<V, DP>(keys.dk, a.grad_scale, a.dim, dk + row * a.dim);
    store_column<V, DP>(keys.dv, 1.0f, a.dim, dv + row * a.dim);
  }
}

// Two tiles of 128 queries where the LDS of a CU holds them (all but wide
// float32 heads).
template <class V, int DP>
constexpr int far_buffers() {
  return 2 * QueryTile<V, DP, 32 * kWaves, kThreads>::kBytes <= 160 * 1024 ? 2 : 1;
}

// Sinks and the queries beyond their block's span: a wave takes every fourth
// 32 queries.
template <class V, int DP>
__global__ __launch_bounds__(kThreads, 1) void backward_keys_far(WindowArgs a, Upstream up,
                                                                 KeyPlan plan, uint32_t blocks) {
  constexpr int kTokens = 32 * kWaves;
  using Tile = QueryTile<V, DP, kTokens, kThreads>;
  constexpr int kBuffers = far_buffers<V, DP>();
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const TilePlaces<V, DP> lanes(lds);

  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t id = xcd_order(blockIdx.x, blocks);
  const int32_t part = static_cast<int32_t>(id % plan.far_parts);
  const int32_t unit = static_cast<int32_t>(id / plan.far_parts % plan.far_units);
  const uint32_t head = id / plan.far_parts / plan.far_units;
  const int64_t bh = head, b = head / a.kv_heads;
  const int32_t kvh = static_cast<int32_t>(head % a.kv_heads);
  const int32_t n = __builtin_amdgcn_readfirstlane(a.length(b)), offset = a.lk - a.lq;
  const int32_t key = unit * 32 + lane % 32;
  const bool live = key < a.sinks && key < n;

  KeyWave<V, DP, false> keys;
  keys.start(a, b, kvh, key, live);

  const int32_t first = max(near_last(a, unit * 32 / kBlockKeys, n) + 1, offset), last = n - 1;
  const int32_t tiles = last >= first ? (last - first) / kTokens + 1 : 0;
  const int64_t total = static_cast<int64_t>(tiles) * a.group;
  const int32_t begin = static_cast<int32_t>(total * part / plan.far_parts);
  const int32_t end = static_cast<int32_t>(total * (part + 1) / plan.far_parts);

  Tile next;
  next.start(a, up);
  const auto fetch = [&](int32_t step, uint32_t to) {
    next.fetch(a, up, b, kvh * a.group + step / tiles, first + step % tiles * kTokens, last, offset,
               lds + to);
  };
  if (begin < end) {
    fetch(begin, 0);
    next.keep(lds);
  }
  sync_tiles();
  for (int32_t step = begin; step < end; ++step) {
    const bool more = step + 1 < end;
    const uint32_t tile = kBuffers == 2 ? (step - begin) % 2 * Tile::kBytes : 0;
    const uint32_t other = kBuffers == 2 ? Tile::kBytes - tile : 0;
    if (kBuffers == 2 && more) fetch(step + 1, other);
    const float *stat = reinterpret_cast<const float *>(lds + tile + 2 * Tile::kTile);
    // all of these queries see the sinks; a key that is none is not stored
    keys.add(a, lanes, tile, tile + Tile::kTile, stat, stat + kTokens, 32 * wave, 0, key, false);
    if (kBuffers == 1) {
      sync_tiles();
      if (more) fetch(step + 1, 0);
    }
    if (more) next.keep(lds + other);
    sync_tiles();
  }
  if (key >= a.sinks || key >= a.lk) return;
  keys.finish();
  const int64_t slot = ((bh * plan.far_units + unit) * plan.far_parts + part) * kWaves + wave;
  float *to = plan.far_sums + (slot * 32 + lane % 32) * 2 * a.dim;
  store_sums<DP>(keys.dk, a.dim, to);
  store_sums<DP>(keys.dv, a.dim, to + a.dim);
}

// dk and dv of the joined units, and dq of the blocks that ran in parts, a few
// rows a workgroup.  Four values a lane, four lanes a sum: each takes every
// fourth part, and the four are added in one order.
constexpr int kJoinKeys = 2, kJoinQueries = 8;

__device__ __forceinline__ void add_parts(const float *first, int32_t parts, int64_t stride, v4f &sum) {
#pragma unroll 8
  for (int32_t part = threadIdx.x % kWave / 16; part < parts; part += 4) {
    const v4f x = *reinterpret_cast<const v4f *>(first + part * stride);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] += x[j];
  }
}
template <class V>
__device__ __forceinline__ void store_joined(v4f sum, float factor, typename V::Storage *to) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sum[j] += __shfl_xor(sum[j], 16);
    sum[j] += __shfl_xor(sum[j], 32);
    sum[j] *= factor;
  }
  if (threadIdx.x % kWave >= 16 || to == nullptr) return;
  if constexpr (sizeof(typename V::Storage) == 2)
    *reinterpret_cast<v2u *>(to) = v2u{Mfma<V>::pack(sum[0], sum[1]), Mfma<V>::pack(sum[2], sum[3])};
  else
    *reinterpret_cast<v4f *>(to) = sum;
}

template <class V>
__global__ __launch_bounds__(256) void join_sums(WindowArgs a, KeyPlan keys, QueryPlan queries,
                                                 int64_t of_keys, typename V::Storage *dq,
                                                 typename V::Storage *dk, typename V::Storage *dv) {
  const int first = threadIdx.x / kWave * 16 + threadIdx.x % 16;  // piece of the workgroup's
  const int32_t pieces = a.dim / 4;
  if (blockIdx.x < of_keys) {
    // rows of the blocks in parts, then of the other far units
    constexpr int kPer = kBlockKeys / kJoinKeys, kPerUnit = 32 / kJoinKeys;
    const uint32_t cut = static_cast<uint32_t>(keys.cut.rest) * kPer, whole = static_cast<uint32_t>(keys.cut.whole);
    const bool in_parts = blockIdx.x < cut;
    const uint32_t id = in_parts ? blockIdx.x : blockIdx.x - cut, rest = id / kPer;
    uint32_t head;
    int32_t unit, row0;
    if (in_parts) {
      head = (whole + rest) / keys.blocks;
      row0 = static_cast<int32_t>(id % kPer * kJoinKeys);
      unit = static_cast<int32_t>((whole + rest) % keys.blocks) * kWaves + row0 / 32;
    } else {
      head = id / kPerUnit / keys.far_units;
      row0 = static_cast<int32_t>(id % kPerUnit * kJoinKeys);
      unit = static_cast<int32_t>(id / kPerUnit % keys.far_units);
      if (head * keys.blocks + unit / kWaves >= whole) return;
    }
    const int64_t bh = head, b = head / a.kv_heads;
    const int32_t kvh = static_cast<int32_t>(head % a.kv_heads), dims = 2 * a.dim;
    const int32_t near_parts = in_parts ? keys.cut.parts : 1, stride = (in_parts ? kBlockKeys : 32) * dims;
    const float *near = in_parts ? keys.part_sums + static_cast<int64_t>(rest) * near_parts * stride + row0 / 32 * 32 * dims
                                 : keys.unit_sums + (bh * keys.far_units + unit) * stride;
    const int32_t far_parts = unit < keys.far_units ? keys.far_parts * kWaves : 0;
    const float *far = keys.far_sums + (bh * keys.far_units + unit) * far_parts * 32 * dims;
    row0 %= 32;
    for (int at = first; at - first % 16 < kJoinKeys * 2 * pieces; at += 64) {
      const int32_t row = row0 + at / (2 * pieces), d = at % (2 * pieces) * 4, key = unit * 32 + row;
      v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
      typename V::Storage *to = nullptr;
      if (row < row0 + kJoinKeys && key < a.lk) {
        add_parts(near + row * dims + d, near_parts, stride, sum);
        if (key < a.sinks) add_parts(far + row * dims + d, far_parts, 32 * dims, sum);
        const int64_t at_row = ((b * a.lk + key) * a.kv_heads + kvh) * a.dim;
        to = d < a.dim ? dk + at_row + d : dv + at_row + d - a.dim;
      }
      store_joined<V>(sum, d < a.dim ? a.grad_scale : 1.0f, to);
    }
  } else {
    constexpr int kRows = kWaves * 32, kPer = kRows / kJoinQueries;
    const int64_t id = blockIdx.x - of_keys, rest = id / kPer, block = queries.cut.whole + rest;
    const int64_t bh = block / queries.per_bh, b = bh / a.kv_heads;
    const int32_t row0 = static_cast<int32_t>(id % kPer) * kJoinQueries;
    const int32_t unit = static_cast<int32_t>(block % queries.per_bh) * kWaves + row0 / 32;
    if (unit >= queries.units) return;
    const int32_t h = static_cast<int32_t>(bh % a.kv_heads) * a.group + unit % a.group;
    const int32_t i0 = unit / a.group * 32 + row0 % 32;
    const float *sums = queries.sums + (rest * queries.cut.parts * kRows + row0) * a.dim;
    for (int at = first; at - first % 16 < kJoinQueries * pieces; at += 64) {
      const int32_t row = at / pieces, d = at % pieces * 4;
      v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
      typename V::Storage *to = nullptr;
      if (row < kJoinQueries && i0 + row < a.lq) {
        add_parts(sums + row * a.dim + d, queries.cut.parts, static_cast<int64_t>(kRows) * a.dim, sum);
        to = dq + ((b * a.lq + i0 + row) * a.heads + h) * a.dim + d;
      }
      store_joined<V>(sum, a.grad_scale, to);
    }
  }
}

// Queries are cut as in the forward pass.
QueryPlan plan_queries(const WindowArgs &a, int32_t tile) {
  QueryPlan p{};
  p.units = (static_cast<int64_t>(a.lq) + 31) / 32 * a.group;
  p.per_bh = (p.units + kWaves - 1) / kWaves;
  const int64_t keys = std::min<int64_t>(a.lk, static_cast<int64_t>(a.window) + a.sinks + 32);
  p.cut = cut_tail(p.per_bh * a.batch * a.kv_heads, 2 * 256, (keys + tile - 1) / tile,
                   join_cost(tile == 32));
  return p;
}

// The far pass's units are cut until there are about as many as CUs, of four
// tiles at least (two a CU lose 12 us of 665 in joining them, for 16,384 tokens).
KeyPlan plan_keys(const WindowArgs &a, int32_t tile) {
  constexpr int64_t kCus = 256;
  KeyPlan p{};
  const int64_t bh = a.batch * a.kv_heads;
  p.blocks = (a.lk + kBlockKeys - 1) / kBlockKeys;
  const int64_t span = std::min<int64_t>(a.lq, static_cast<int64_t>(a.window) + kBlockKeys - 1);
  p.cut = cut_tail(bh * p.blocks, kCus, (span + tile - 1) / tile * a.group,
                   join_cost(tile == 32));
  // queries that see sinks from beyond the first block's span
  const int64_t beyond =
      std::min<int64_t>(a.lq, static_cast<int64_t>(a.lk) - kBlockKeys - a.window + 1);
  if (beyond > 0 && a.sinks > 0) {
    p.far_units = (a.sinks + 31) / 32;
    const int64_t steps = std::max<int64_t>(1, (beyond + 127) / 128 * a.group / 4);
    p.far_parts = static_cast<int32_t>(
        std::min<int64_t>(steps, std::max<int64_t>(1, kCus / std::max<int64_t>(1, bh * p.far_units))));
  }
  return p;
}

size_t part_floats(const WindowArgs &a, const KeyPlan &p) {
  return p.cut.parts > 1 ? static_cast<size_t>(p.cut.rest) * p.cut.parts * kBlockKeys * 2 * a.dim : 0;
}
size_t unit_floats(const WindowArgs &a, const KeyPlan &p) {
  return static_cast<size_t>(a.batch) * a.kv_heads * p.far_units * 32 * 2 * a.dim;
}
size_t query_floats(const WindowArgs &a, const QueryPlan &p) {
  return p.cut.parts > 1 ? static_cast<size_t>(p.cut.rest) * p.cut.parts * kWaves * 32 * a.dim : 0;
}
size_t far_floats(const WindowArgs &a, const KeyPlan &p) {
  return static_cast<size_t>(a.batch) * a.kv_heads * p.far_units * p.far_parts * kWaves * 32 * 2 * a.dim;
}

template <class V, int DP>
msx_status run(const WindowArgs &a, const Upstream &up, const QueryPlan &queries, const KeyPlan &plan,
               void *dq, void *dk, void *dv, hipStream_t stream) {
  using S = typename V::Storage;
  const int64_t bh = a.batch * a.kv_heads, q_blocks = queries.cut.items();
  const int64_t k_blocks = plan.cut.items(), f_blocks = bh * plan.far_units * plan.far_parts;
  const int64_t of_keys =
      plan.cut.rest * (kBlockKeys / kJoinKeys) + bh * plan.far_units * (32 / kJoinKeys);
  const int64_t joined = of_keys + queries.cut.rest * (kWaves * 32 / kJoinQueries);
  static_assert(kThreads <= NearShape<V, DP>::kThreads, "the keys' pass has the most threads");
  for (int64_t blocks : {q_blocks, k_blocks, f_blocks, joined})
    if (queries.units > 0x7fffffff || blocks > max_blocks(NearShape<V, DP>::kThreads))
      return fail(MSX_EINVAL, "window_attention_backward has more rows than a grid holds.");
  if (q_blocks > 0)
    backward_queries<V, DP><<<static_cast<unsigned>(q_blocks), kThreads, 0, stream>>>(
        a, up, queries, static_cast<S *>(dq));
  if (k_blocks > 0)
    backward_keys_near<V, DP><<<static_cast<unsigned>(k_blocks), NearShape<V, DP>::kThreads, 0, stream>>>(
        a, up, plan, static_cast<S *>(dk), static_cast<S *>(dv));
  if (f_blocks > 0) {
    constexpr int lds = far_buffers<V, DP>() * QueryTile<V, DP, 32 * kWaves, kThreads>::kBytes;
    if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(backward_keys_far<V, DP>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        e != hipSuccess)
      return hip_fail(e, "window_attention_backward");
    backward_keys_far<V, DP><<<static_cast<unsigned>(f_blocks), kThreads, lds, stream>>>(
        a, up, plan, static_cast<uint32_t>(f_blocks));
  }
  if (joined > 0)
    join_sums<V><<<static_cast<unsigned>(joined), 256, 0, stream>>>(
        a, plan, queries, of_keys, static_cast<S *>(dq), static_cast<S *>(dk),
        static_cast<S *>(dv));
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "window_attention_backward");
}

template <class V>
msx_status by_dim(const WindowArgs &a, const Upstream &up, const QueryPlan &queries, const KeyPlan &plan,
                  void *dq, void *dk, void *dv, hipStream_t stream) {
  if (a.dim <= 32) return run<V, 32>(a, up, queries, plan, dq, dk, dv, stream);
  if (a.dim <= 64) return run<V, 64>(a, up, queries, plan, dq, dk, dv, stream);
  if (a.dim <= 96) return run<V, 96>(a, up, queries, plan, dq, dk, dv, stream);
  return run<V, 128>(a, up, queries, plan, dq, dk, dv, stream);
}

// Queries of a tile of the near pass (BackwardShape::kTokens).
int32_t tile_of(msx_vtype vt) { return vt == MSX_F32 ? 32 : 64; }

}  // namespace

size_t window_backward_scratch(msx_vtype vt, const WindowArgs &a) {
  const KeyPlan p = plan_keys(a, tile_of(vt));
  return sizeof(float) *
         (part_floats(a, p) + unit_floats(a, p) + far_floats(a, p) +
          query_floats(a, plan_queries(a, tile_of(vt))));
}

msx_status launch_window_backward(msx_vtype vt, const WindowArgs &a, const void *out,
                                  const float *lse, const void *grad, const int64_t *grad_strides,
                                  float *delta, void *dq, void *dk, void *dv, void *scratch,
                                  hipStream_t stream) {
  Upstream up{grad, {grad_strides[0], grad_strides[1], grad_strides[2]}, out, lse, delta};
  KeyPlan plan = plan_keys(a, tile_of(vt));
  plan.part_sums = static_cast<float *>(scratch);
  plan.unit_sums = plan.part_sums + part_floats(a, plan);
  plan.far_sums = plan.unit_sums + unit_floats(a, plan);
  QueryPlan queries = plan_queries(a, tile_of(vt));
  queries.sums = plan.far_sums + far_floats(a, plan);
  switch (vt) {
  case MSX_F32: return by_dim<F32>(a, up, queries, plan, dq, dk, dv, stream);
  case MSX_F16: return by_dim<F16>(a, up, queries, plan, dq, dk, dv, stream);
  default: return by_dim<BF16>(a, up, queries, plan, dq, dk, dv, stream);
  }
}

}  // namespace msx
