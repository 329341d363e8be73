// msx_window_mfma.h - matrix-core tiles of window attention.
//
// Scores are computed transposed, S^T = K Q^T (32 keys x 32 queries a tile):
// a lane then holds one query, lane % 32, and of each 32 keys the sixteen
//   key(i) = 8 (i / 4) + 4 (lane / 32) + i % 4,   i = 0 .. 15,
// so a row of the softmax is a lane's own values and one exchange with the
// lane 32 away.  The next product, O^T = V^T P^T, takes its k index in that
// same order: P needs no shuffle, only its rounding, and V^T is read in the
// matching order (16-bit values through the transposing LDS read, which hands
// a lane four keys of one column).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "msx_device.h"
#include "msx_window.h"

namespace msx {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));

// A tile of rows in LDS: rows of `kPitch` bytes, their 16-byte chunks
// permuted by row so that the reads below spread over the banks.
template <class V, int DP>
struct TileShape {
  static constexpr int kSize = sizeof(typename V::Storage);
  static constexpr int kRowBytes = DP * kSize;
  static constexpr int kPitch = kRowBytes <= 64 ? 64 : kRowBytes <= 128 ? 128 : kRowBytes <= 256 ? 256 : 512;
  static constexpr int kChunks = kPitch / 16;      // of which kRowBytes / 16 are used
  static constexpr int kUsed = kRowBytes / 16;

  // Sixteen rows read at one chunk (a lane a row) fall into sixteen chunks of
  // the 256 bytes that the banks span, and so do the four rows by four chunks
  // that half a wave's transposing read takes.
  __device__ static inline int along(int row, int chunk) {
    const int low = kPitch >= 256 ? (row & 3) << 2 : kPitch == 128 ? (row & 2) << 1 : 0;
    return row * kPitch + ((chunk ^ (low | ((row >> 2) & 3))) * 16);
  }
};

template <class V>
struct Mfma;

// 16-bit operands: 32 x 32 x 16 products; a lane holds eight adjacent values
// of its row, at 8 (lane / 32) of each sixteen.
template <>
struct Mfma<BF16> {
  using Frag = v8bf;
  static constexpr int kDepth = 16;
  __device__ static inline v16f mul(Frag a, Frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static inline uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{lo, hi}), v2bf));
  }
  static constexpr uint32_t kSign = 0x80008000u;
};
template <>
struct Mfma<F16> {
  using Frag = v8h;
  static constexpr int kDepth = 16;
  __device__ static inline v16f mul(Frag a, Frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static inline uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{lo, hi}), v2h));
  }
  static constexpr uint32_t kSign = 0x80008000u;
};
// float32: 32 x 32 x 2 products.  Sixteen bytes a lane serve four of them:
// product j of a group of eight values takes values j and 4 + j.
template <>
struct Mfma<F32> {
  using Frag = v4f;
  static constexpr int kDepth = 8;
  __device__ static inline v16f mul(Frag a, Frag b, v16f c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static constexpr uint32_t kSign = 0x80000000u;
};

// Sixteen bytes of a row for step `s` of a product over the head dimension:
// chunk 2 s + lane / 32 in either type.
template <class V, int DP>
__device__ inline typename Mfma<V>::Frag read_rows(const char *tile, int row, int s) {
  const int half = (threadIdx.x % kWave) / 32;
  return *reinterpret_cast<const typename Mfma<V>::Frag *>(
      tile + TileShape<V, DP>::along(row, 2 * s + half));
}

__device__ inline v4s read_transposed(const char *p) {
  // the builtin takes an LDS pointer
  auto *lds = (__attribute__((address_space(3))) v4s *)(p);
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds);
}

// acc[dt] += X^T P over 32 rows of the tile from `row0` on: p the lane's
// sixteen values in the order above, X read along its columns.
template <class V, int DP>
__device__ inline void mul_transposed(const char *tile, int row0, const float (&p)[16],
                                      v16f (&acc)[DP / 32]) {
  using T = TileShape<V, DP>;
  const int lane = threadIdx.x % kWave, half = lane / 32;
  if constexpr (T::kSize == 2) {
    typename Mfma<V>::Frag b[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v4u w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = Mfma<V>::pack(p[8 * k + 2 * j], p[8 * k + 2 * j + 1]);
      b[k] = __builtin_bit_cast(typename Mfma<V>::Frag, w);
    }
    const int i = lane % 16, column = ((lane / 16) % 2) * 16 + (i % 4) * 4;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v4s part[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int row = row0 + 16 * k + 8 * t + 4 * half + i / 4, d = dt * 32 + column;
          part[t] = read_transposed(tile + T::along(row, d / 8) + (d % 8) * 2);
        }
        const auto lo = __builtin_bit_cast(v2u, part[0]), hi = __builtin_bit_cast(v2u, part[1]);
        const auto a = __builtin_bit_cast(typename Mfma<V>::Frag, (v4u{lo[0], lo[1], hi[0], hi[1]}));
        acc[dt] = Mfma<V>::mul(a, b[k], acc[dt]);
      }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = row0 + 8 * (r / 4) + 4 * half + r % 4;
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) {
        const int d = dt * 32 + lane % 32;
        const float a = *reinterpret_cast<const float *>(tile + T::along(row, d / 4) + (d % 4) * 4);
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[dt], 0, 0, 0);
      }
    }
  }
}

// A span of keys numbered through (sinks before it, then itself), and which of
// them a position sees: those no further back than `window`, any of the first
// `free` numbers.
struct Numbering {
  int32_t far, skip, free, window;
  __device__ inline Numbering(const WindowArgs &a, int32_t near)
      : far(min(a.sinks, near)), skip(near - far), free(skip == 0 ? a.sinks : far), window(a.window) {}
  __device__ inline int32_t key(int32_t c) const { return c < far ? c : c + skip; }
  // p = -1 sees nothing.
  __device__ inline bool seen(int32_t p, int32_t c) const {
    const uint32_t back = static_cast<uint32_t>(p - key(c));
    return back < static_cast<uint32_t>(c < free ? 0x7fffffff : window);
  }
};

// A workgroup's share of a tile's rows on its way from memory to LDS, sixteen
// bytes a piece.  Rows that follow each other in memory are read from one
// uniform address by 32-bit offsets that stay: with an address worked out for
// every piece the forward tiles spent half of their vector instructions on it.
template <class V, int DP, int kTokens, int kThreads>
struct RowLoader {
  using T = TileShape<V, DP>;
  static constexpr int kPer = (kTokens * T::kUsed + kThreads - 1) / kThreads;
  static constexpr bool kEven = kThreads % T::kUsed == 0 && kTokens * T::kUsed % kThreads == 0;
  uint32_t offset;   // of the thread's first piece
  int64_t step;      // bytes between rows
  bool plain;        // whole rows within 2 GB of each other (uniform)

  __device__ inline void start(int64_t stride, int dim) {
    step = stride * T::kSize;
    plain = kEven && dim == DP && step >= 0 && step * kTokens < (int64_t{1} << 31);
    offset = static_cast<uint32_t>(threadIdx.x / T::kUsed) * static_cast<uint32_t>(step) +
             threadIdx.x % T::kUsed * 16;
  }
  // kTokens rows from `first` on, all there.
  __device__ inline void load(const void *first, v4u (&to)[kPer]) const {
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const char *base = static_cast<const char *>(first) + r * (kThreads / T::kUsed) * step;
      to[r] = *reinterpret_cast<const v4u *>(base + offset);
    }
  }
};

// The lane 32 away.
__device__ inline float other_half(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t other = (threadIdx.x % kWave) < 32 ? r[1] : r[0];
  return __builtin_bit_cast(float, other);
}

// Workgroups go to the 8 XCDs in turn; this gives each XCD one contiguous
// part of the work, whose neighbours share what they read through its L2.
__device__ inline int64_t xcd_order(int64_t id, int64_t n) {
  const int64_t per = n / 8, rest = n % 8, x = id % 8, at = id / 8;
  return x * per + (x < rest ? x : rest) + at;
}

// How equal blocks of work are cut over `slots` workgroups that run at once:
// the first `whole` run as they are, each of the rest in `parts`, so that the
// last round does not leave most of the chip waiting for a few blocks.
struct TailCut {
  int64_t whole, rest;
  int32_t parts;
  __host__ __device__ inline int64_t items() const { return whole + rest * parts; }
};

// A part costs what kPartCost of a block does, in writing and joining sums.
inline TailCut cut_tail(int64_t blocks, int64_t slots, int64_t most_parts) {
  constexpr double kPartCost = 0.04;
  const int64_t rest = blocks % slots;
  TailCut cut{blocks, 0, 1};
  double best = rest > 0 ? 1.0 : 0.0;
  for (int64_t p = 2; p <= most_parts && p <= 16 && rest > 0; ++p) {
    const double rounds = static_cast<double>((rest * p + slots - 1) / slots) / p;
    const double cost = rounds + kPartCost * (1 + rest * p / static_cast<double>(slots));
    if (cost < best) {
      best = cost;
      cut = TailCut{blocks - rest, rest, static_cast<int32_t>(p)};
    }
  }
  return cut;
}

// Which block and part of it a workgroup takes; the whole ones in XCD order.
struct CutItem {
  int64_t block;
  int32_t part, parts;
  int64_t slot;  // of its sums in scratch, -1 for a whole block
  __device__ inline CutItem(const TailCut &cut, int64_t id) {
    if (id < cut.whole) {
      block = xcd_order(id, cut.whole);
      part = 0;
      parts = 1;
      slot = -1;
    } else {
      slot = id - cut.whole;
      block = cut.whole + slot / cut.parts;
      part = static_cast<int32_t>(slot % cut.parts);
      parts = cut.parts;
    }
  }
};

}  // namespace msx
