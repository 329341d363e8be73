// distill.hip - distillation from a teacher's top logits, the rows of a CSR
// matrix: per-row losses and the gradient in the student's logits.
//
// With z = logits / T, q = softmax(z) over the row and p = softmax(kept / T)
// over the row's kept logits:
//   loss = T^2 sum_r p_r (ln p_r - ln q_r),  ln q_r = z_r - lse
//   grad = weight T (q - p)
// One workgroup a row: a pass over the row for its maximum and the sum of
// exponentials, and for the gradient a second one.  The columns of kept logits
// are written last, each by the thread that holds it, q - p rounded once.
#include <hip/hip_runtime.h>

#include <cmath>

#include "msx_device.h"
#include "msx_internal.h"
#include "msx_window.h"
#include "msx_window_check.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

struct DistillArgs {
  int64_t n_cols, ld, ld_grad, nnz;
  const void *logits;
  const void *data, *indices, *indptr;
  int32_t teacher_vtype, index64;
  const float *weights;
  int64_t weights_stride;
  float scale;        // log2(e) / T: scaled logits are kept in base 2
  float temperature;

  // T^2 of a row's loss comes from these two.
  __device__ inline int64_t offset(int64_t r) const {
    const int64_t p = index64 ? static_cast<const int64_t *>(indptr)[r]
                              : static_cast<const int32_t *>(indptr)[r];
    return p < 0 ? 0 : p > nnz ? nnz : p;
  }
  // Column of entry e, or -1 outside the matrix.
  __device__ inline int64_t column(int64_t e) const {
    const int64_t c = index64 ? static_cast<const int64_t *>(indices)[e]
                              : static_cast<const int32_t *>(indices)[e];
    return c < 0 || c >= n_cols ? -1 : c;
  }
  __device__ inline float kept(int64_t e) const {
    if (teacher_vtype == MSX_F32) return static_cast<const float *>(data)[e] * scale;
    const uint16_t bits = static_cast<const uint16_t *>(data)[e];
    return (teacher_vtype == MSX_F16 ? half_bits_to_float(bits) : bf16_bits_to_float(bits)) * scale;
  }
  __device__ inline float weight(int64_t r) const {
    return weights == nullptr ? 1.0f : weights[r * weights_stride];
  }
};

// Maximum and sum of exponentials of what has been seen, base 2.
struct Stat {
  float top, sum;
  __device__ inline float base() const { return top == -INFINITY ? 0.0f : top; }
  __device__ inline void add(float x) {
    const float t = fmaxf(top, x);
    const float b = t == -INFINITY ? 0.0f : t;
    sum = sum * exp2_fast(top - b) + exp2_fast(x - b);
    top = t;
  }
  __device__ inline void merge(Stat o) {
    const float t = fmaxf(top, o.top);
    const float b = t == -INFINITY ? 0.0f : t;
    sum = sum * exp2_fast(top - b) + o.sum * exp2_fast(o.top - b);
    top = t;
  }
};

__device__ inline Stat block_merge(Stat s, Stat *lds) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) s.merge({__shfl_xor(s.top, d), __shfl_xor(s.sum, d)});
  const int wave = threadIdx.x / kWave;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[wave] = s;
  __syncthreads();
  s = lds[0];
  for (int w = 1; w < kWaves; ++w) s.merge(lds[w]);
  return s;
}

__device__ inline float block_sum(float v, float *lds) {
  v = wave_sum(v);
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
  for (int w = 1; w < kWaves; ++w) v += lds[w];
  return v;
}

// kLoss: losses (and lse where asked); kGrad: the gradient, from `lse_in` or
// from the row's own pass.
template <class V, bool kLoss, bool kGrad>
__global__ __launch_bounds__(kThreads) void distill_rows(DistillArgs a, float *losses, float *lse,
                                                         const float *lse_in,
                                                         typename V::Storage *grad) {
  using S = typename V::Storage;
  __shared__ Stat stat_lds[kWaves];
  __shared__ float sum_lds[kWaves];
  const int64_t row = blockIdx.x;
  const S *z = static_cast<const S *>(a.logits) + row * a.ld;
  S *g = kGrad ? grad + row * a.ld_grad : nullptr;
  const int64_t begin = a.offset(row), end = a.offset(row + 1);
  const float weight = kGrad ? a.weight(row) : 0.0f;

  // the teacher's distribution; ascending: no column is there twice
  Stat kept{-INFINITY, 0.0f};
  int ascending = 1;
  for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
    const int64_t c = a.column(e);
    if (c >= 0) kept.add(a.kept(e));
    if (e + 1 < end && a.column(e + 1) <= c) ascending = 0;
  }
  kept = block_merge(kept, stat_lds);
  ascending = __syncthreads_and(ascending);
  const bool target = !(kept.sum == 0.0f);

  if (!target) {
    if (kLoss && threadIdx.x == 0) {
      losses[row] = 0.0f;
      if (lse != nullptr) lse[row] = 0.0f;
    }
  }
  const bool wanted = kGrad && target && weight != 0.0f;
  if (kGrad && !wanted)
    for (int64_t c = threadIdx.x; c < a.n_cols; c += kThreads) g[c] = 0;
  if (!target || !(kLoss || wanted)) return;

  const float kept_base = kept.base(), kept_inv = 1.0f / kept.sum;
  const float kept_lse = kept_base + log2_fast(kept.sum);
  float total;
  if (kLoss) {
    Stat s{-INFINITY, 0.0f};
    for (int64_t c = threadIdx.x; c < a.n_cols; c += kThreads) s.add(V::widen(z[c]) * a.scale);
    s = block_merge(s, stat_lds);
    total = s.base() + log2_fast(s.sum);
    float part = 0.0f;
    for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
      const int64_t c = a.column(e);
      if (c < 0) continue;
      const float t = a.kept(e), p = exp2_fast(t - kept_base) * kept_inv;
      if (p != 0.0f) part += p * ((t - kept_lse) - (V::widen(z[c]) * a.scale - total));
    }
    part = block_sum(part, sum_lds);
    if (threadIdx.x == 0) {
      losses[row] = part * kLn2 * a.temperature * a.temperature;
      if (lse != nullptr) lse[row] = total;
    }
    if (!wanted) return;
  } else {
    total = lse_in[row];
  }
  if (kGrad) {
    const float factor = weight * a.temperature;
    for (int64_t c = threadIdx.x; c < a.n_cols; c += kThreads)
      g[c] = V::narrow(exp2_fast(V::widen(z[c]) * a.scale - total) * factor);
    __syncthreads();
    for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
      const int64_t c = a.column(e);
      if (c < 0) continue;
      float p = exp2_fast(a.kept(e) - kept_base) * kept_inv;
      if (!ascending) {
        p = 0.0f;
        for (int64_t o = begin; o < end; ++o)
          if (a.column(o) == c) p += exp2_fast(a.kept(o) - kept_base) * kept_inv;
      }
      g[c] = V::narrow((exp2_fast(V::widen(z[c]) * a.scale - total) - p) * factor);
    }
  }
}

DistillArgs args_of(const msx_distill_desc &d, int64_t ld_grad) {
  DistillArgs a{};
  a.n_cols = d.n_cols;
  a.ld = d.ld;
  a.ld_grad = ld_grad;
  a.nnz = d.nnz;
  a.logits = d.logits;
  a.data = d.data;
  a.indices = d.indices;
  a.indptr = d.indptr;
  a.teacher_vtype = d.teacher_vtype;
  a.index64 = d.itype == MSX_I64;
  a.weights = d.weights;
  a.weights_stride = d.weights_stride;
  a.scale = static_cast<float>(1.44269504088896340736 / d.temperature);
  a.temperature = static_cast<float>(d.temperature);
  return a;
}

template <bool kLoss, bool kGrad>
msx_status launch(const msx_distill_desc &d, float *losses, float *lse, const float *lse_in,
                  void *grad, int64_t ld_grad, void *stream) {
  const DistillArgs a = args_of(d, ld_grad);
  const auto run = [&](auto v) {
    using V = decltype(v);
    distill_rows<V, kLoss, kGrad>
        <<<static_cast<unsigned>(d.n_rows), kThreads, 0, static_cast<hipStream_t>(stream)>>>(
            a, losses, lse, lse_in, static_cast<typename V::Storage *>(grad));
  };
  switch (d.vtype) {
  case MSX_F32: run(F32{}); break;
  case MSX_F16: run(F16{}); break;
  default: run(BF16{}); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "distill");
}

msx_status check_grad(const char *op, const msx_distill_desc *d, const void *grad,
                      int64_t ld_grad) {
  if (d->n_rows > 0 && d->n_cols > 0 && grad == nullptr)
    return fail(MSX_EINVAL, std::string(op) + " grad is NULL.");
  if (ld_grad < d->n_cols)
    return fail(MSX_EINVAL, std::string(op) + " leading dimension must be at least the column count.");
  return MSX_OK;
}

}  // namespace
}  // namespace msx

using namespace msx;

extern "C" msx_status msx_distill_loss(const msx_distill_desc *desc, float *losses, float *lse,
                                       void *stream) {
  clear_error();
  if (msx_status st = check_distill("distill_loss", desc); st != MSX_OK) return st;
  if (desc->n_rows == 0) return MSX_OK;
  if (losses == nullptr) return fail(MSX_EINVAL, "distill_loss losses is NULL.");
  return launch<true, false>(*desc, losses, lse, nullptr, nullptr, 0, stream);
}

extern "C" msx_status msx_distill_grad(const msx_distill_desc *desc, const float *lse, void *grad,
                                       int64_t ld_grad, void *stream) {
  clear_error();
  if (msx_status st = check_distill("distill_grad", desc); st != MSX_OK) return st;
  if (msx_status st = check_grad("distill_grad", desc, grad, ld_grad); st != MSX_OK) return st;
  if (desc->n_rows == 0 || desc->n_cols == 0) return MSX_OK;
  if (lse == nullptr) return fail(MSX_EINVAL, "distill_grad lse is NULL.");
  return launch<false, true>(*desc, nullptr, nullptr, lse, grad, ld_grad, stream);
}

extern "C" msx_status msx_distill_loss_grad(const msx_distill_desc *desc, float *losses,
                                            void *grad, int64_t ld_grad, void *stream) {
  clear_error();
  if (msx_status st = check_distill("distill_loss_grad", desc); st != MSX_OK) return st;
  if (msx_status st = check_grad("distill_loss_grad", desc, grad, ld_grad); st != MSX_OK) return st;
  if (desc->n_rows == 0) return MSX_OK;
  if (losses == nullptr) return fail(MSX_EINVAL, "distill_loss_grad losses is NULL.");
  return launch<true, true>(*desc, losses, nullptr, nullptr, grad, ld_grad, stream);
}
