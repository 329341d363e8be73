// msx_window.h - device-side view of window attention: the operands, and
// which keys a query sees.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "msx_device.h"
#include "msx_sparse.h"

namespace msx {

// Operands of one product, as the kernels take them (strides in values).
struct WindowArgs {
  int64_t batch;
  int32_t lq, lk, heads, kv_heads, group, dim;
  int32_t window, sinks;  // capped at lk: no wider span changes the pattern
  float scale;            // scale * log2(e): scores are kept in base 2
  float grad_scale;       // scale
  const void *lengths;
  int32_t lengths64;
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];
  void *low;  // the residues of out, see Residue; may be null

  // Where the residue of out[b][i][h][d] lies: eight values of a row, then the
  // rows of 32 queries, as the tiles' waves store and load them.
  __host__ __device__ inline int64_t low_at(int64_t b, int32_t i, int32_t h, int32_t d) const {
    const int64_t units = (lq + 31) / 32, chunks = (dim + 7) / 8;
    return ((((b * heads + h) * units + i / 32) * chunks + d / 8) * 32 + i % 32) * 8 + d % 8;
  }

  // Tokens of sequence b that exist: [0, lk].
  __device__ inline int32_t length(int64_t b) const {
    if (lengths == nullptr) return lk;
    const int64_t n = lengths64 ? static_cast<const int64_t *>(lengths)[b]
                                : static_cast<const int32_t *>(lengths)[b];
    return static_cast<int32_t>(n < 0 ? 0 : n > lk ? lk : n);
  }
};

// Workgroups of `threads` that one launch holds: it counts its threads in 32 bits.
constexpr int64_t max_blocks(int64_t threads) { return 0xffffffff / threads; }

// Logarithms are base 2: exp2 is one instruction, and a score times log2(e)
// costs nothing beside the scale.
constexpr float kLn2 = 0.69314718055994530942f;

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// What a result has beyond its 16 bits, in 16 bits more: kept for delta =
// grad.out of the backward pass, which is subtracted from dP and has to be good to
// a rounding of the difference, not of itself.  float16's is held 2^10 larger, so
// that it is as far above the subnormals as the result.
template <class V>
struct Residue {
  static constexpr float kUp = V::kType == MSX_F16 ? 1024.0f : 1.0f;
  __device__ static inline typename V::Storage of(float x, typename V::Storage kept) {
    return V::narrow((x - V::widen(kept)) * kUp);
  }
  __device__ static inline float value(typename V::Storage low) {
    return V::widen(low) * (1.0f / kUp);
  }
};

__device__ inline float wave_max(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}
__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// The keys that the query at position p sees, numbered: the first `far` are
// keys 0 .. far - 1, the others near .. p.
struct Seen {
  int32_t near, far;
  __device__ inline Seen(int32_t p, int32_t window, int32_t sinks)
      : near(p >= window ? p - window + 1 : 0), far(sinks < near ? sinks : near) {}
  __device__ inline int32_t count(int32_t p) const { return far + p - near + 1; }
  __device__ inline int32_t key(int32_t c) const { return c < far ? c : near + c - far; }
};

// Operands of a single-token step.
struct StepArgs {
  int64_t batch;
  int32_t heads, kv_heads, group, dim, slots, window, sinks;
  float scale;
  const void *lengths;
  int32_t lengths64;
  const void *q, *k, *v;
  int64_t qs[2], ks[2], vs[2];
  void *ck, *cv;
  int64_t cks[3], cvs[3];

  __device__ inline int64_t length(int64_t b) const {
    return lengths64 ? static_cast<const int64_t *>(lengths)[b]
                     : static_cast<const int32_t *>(lengths)[b];
  }
  __device__ inline int32_t slot(int64_t j) const {
    return static_cast<int32_t>(j < sinks ? j : sinks + (j - sinks) % (slots - sinks));
  }
};

// window_forward.hip: operands that takes_tiles (window_attention.hip) admits.
// `scratch`: window_forward_scratch bytes at a sixteen-byte address.
size_t window_forward_scratch(msx_vtype vt, const WindowArgs &a);
msx_status launch_window_forward(msx_vtype vt, const WindowArgs &a, void *out, float *lse,
                                 void *scratch, hipStream_t stream);

// window_backward.hip: the same operands; `grad` aligned as they are.
// `delta`: batch x heads x lq floats, `scratch`: window_backward_scratch bytes.
size_t window_backward_scratch(msx_vtype vt, const WindowArgs &a);
msx_status launch_window_backward(msx_vtype vt, const WindowArgs &a, const void *out,
                                  const float *lse, const void *grad, const int64_t *grad_strides,
                                  float *delta, void *dq, void *dk, void *dv, void *scratch,
                                  hipStream_t stream);

// window_step.hip: rows and caches at sixteen-byte addresses and strides.
// `scratch`: window_step_scratch bytes.
size_t window_step_scratch(msx_vtype vt, const StepArgs &a);
msx_status launch_window_step(msx_vtype vt, const StepArgs &a, void *out, void *scratch,
                              hipStream_t stream);

}  // namespace msx
