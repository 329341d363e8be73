// msx_step_mfma.h - matrix-core tiles of single-token attention: sixteen queries
// against 32 keys (16 in float32) a wave and step.
#pragma once

#include <algorithm>

#include "msx_window_mfma.h"

namespace msx {

constexpr int kStepWaves = 4;  // of a workgroup
constexpr int kStepRows = 16;  // queries a workgroup

template <class V>
struct Mfma16;
template <>
struct Mfma16<BF16> {
  __device__ static inline v4f mul(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma16<F16> {
  __device__ static inline v4f mul(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma16<F32> {
  __device__ static inline v4f mul(v4u a, v4u b, v4f c) {
    const v4f x = __builtin_bit_cast(v4f, a), y = __builtin_bit_cast(v4f, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    return c;
  }
};

// Lane layout of the products: scores S^T = K Q^T, 16 keys x 16 heads, with
// head = lane % 16 and keys 4 (lane / 16) + i; O^T = V^T P^T takes its keys in
// that order (two 16-key tiles make the 32 of a 16-bit product).
template <class V, int DP>
struct StepShape {
  static constexpr int kSize = sizeof(typename V::Storage);
  static constexpr int kTiles = kSize == 2 ? 2 : 1;  // 16-key tiles a step
  static constexpr int kKeys = 16 * kTiles;
  static constexpr int kUsed = DP * kSize / 16;       // chunks of a row
  static constexpr int kChunks = kUsed <= 4 ? 4 : kUsed <= 8 ? 8 : kUsed <= 16 ? 16 : kUsed <= 32 ? 32 : 64;  // and its pitch
  static constexpr int kSteps = kUsed / 4;            // four lanes a row
  static constexpr int kVPer = kKeys * kChunks / kWave;
  static constexpr int kPitch = kChunks * 16;
  static constexpr int kTile = kKeys * kPitch;
  static constexpr int kLds = std::max(kStepWaves * kTile, kStepWaves * kStepRows * (DP + 4) * 4);

  // 32-byte pairs permuted by row, as in the attention tiles.
  __device__ static inline int at(int row, int chunk) {
    constexpr int rows = kPitch >= 256 ? 1 : 256 / kPitch;
    return row * kPitch + ((chunk ^ (((row / rows) * 2) & (kChunks - 1))) * 16);
  }
};

// Weights of paged attention are 2^(score - m), their sums kept beside that m, which may be any
// number near the row's largest score.  Float16 ends at 2^-24: were m that score, a weight below
// 2^-25 of the largest would be nothing, and many of those may be all that a row adds up to (a
// first key that takes the softmax and whose value is nothing).  So m is as far below it as
// leaves the largest weight 2^15: of a weight w beside the largest, 1, rounding takes 2^-11 w or
// 2^-40, whichever is more, and of one in two values 2^-22 w or 2^-40.  (In tiles, whose m
// may be two lower still, 2^-38.)
template <class V>
constexpr float kWeightsUp = V::kType == MSX_F16 ? 15.0f : 0.0f;

// m, l and dim sums of a query over one part of the keys.
__host__ __device__ inline int64_t part_stride(int32_t dim) { return (dim + 2 + 3) / 4 * 4; }

}  // namespace msx
