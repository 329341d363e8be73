// window_attention.hip - window attention with sinks: the entry points, and
// the row kernels that take every type, head dimension and alignment.
//
// For the query at position p (sees keys [p - window + 1, p] and [0, sinks)):
//   s_j = scale q.k_j,  out = sum_j exp(s_j) v_j / sum_j exp(s_j)
// in one pass over the keys with the running maximum m and sum l: a larger
// maximum m' rescales what is there by exp(m - m').
// Gradients, with P = exp(s - lse), delta = grad.out (per query):
//   dv_j = sum_i P_ij grad_i,  dS_ij = P_ij (grad_i.v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i
// dq is summed by query, dk and dv by key, each in a fixed order, so nothing
// is added atomically.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>

#include "msx_device.h"
#include "msx_internal.h"
#include "msx_window.h"
#include "msx_window_check.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kRowWaves = 4;
constexpr int kMaxPer = 4;  // head values a lane holds: dim <= 256

template <class V>
__device__ inline const typename V::Storage *row_of(const void *base, const int64_t *strides,
                                                    int64_t b, int64_t t, int64_t h) {
  return static_cast<const typename V::Storage *>(base) + b * strides[0] + t * strides[1] +
         h * strides[2];
}

template <class V>
__device__ inline float dot_row(const float *lds, const typename V::Storage *row, int dim) {
  float acc = 0.0f;
  for (int d = 0; d < dim; ++d) acc += lds[d] * V::widen(row[d]);
  return acc;
}

// One wave a query row; a lane takes a key of each 64 for the scores and
// head values lane, lane + 64, ... for the sum over them.
template <class V>
__global__ __launch_bounds__(kRowWaves * kWave) void forward_rows(WindowArgs a, int64_t first, int64_t rows,
                                                                  typename V::Storage *out,
                                                                  float *lse) {
  __shared__ float q_lds[kRowWaves][kWindowMaxDim];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row = first + static_cast<int64_t>(blockIdx.x) * kRowWaves + wave;  // (b, i, h)
  if (row >= rows) return;  // whole waves leave; there is no barrier below
  const int32_t h = static_cast<int32_t>(row % a.heads);
  const int32_t i = static_cast<int32_t>(row / a.heads % a.lq);
  const int64_t b = row / a.heads / a.lq;
  const int32_t p = i + a.lk - a.lq;
  float m = -INFINITY, l = 0.0f, o[kMaxPer] = {};
  if (p >= 0 && p < a.length(b)) {
    const auto *q = row_of<V>(a.q, a.qs, b, i, h);
    float *ql = q_lds[wave];
    for (int d = lane; d < a.dim; d += kWave) ql[d] = V::widen(q[d]);
    __builtin_amdgcn_wave_barrier();
    const Seen seen(p, a.window, a.sinks);
    const int32_t n = seen.count(p), kvh = h / a.group;
    for (int32_t c0 = 0; c0 < n; c0 += kWave) {
      const int32_t j = seen.key(min(c0 + lane, n - 1));
      float s = dot_row<V>(ql, row_of<V>(a.k, a.ks, b, j, kvh), a.dim) * a.scale;
      if (c0 + lane >= n) s = -INFINITY;
      const float top = fmaxf(m, wave_max(s));
      const float base = top == -INFINITY ? 0.0f : top;
      const float e = exp2_fast(s - base);
      const float keep = exp2_fast(m - base);
      l = l * keep + wave_sum(e);
      m = top;
#pragma unroll
      for (int r = 0; r < kMaxPer; ++r) o[r] *= keep;
      const int32_t here = min(kWave, n - c0);
      for (int32_t t = 0; t < here; ++t) {
        const float w = __shfl(e, t);
        const auto *v = row_of<V>(a.v, a.vs, b, seen.key(c0 + t), kvh);
#pragma unroll
        for (int r = 0; r < kMaxPer; ++r)
          if (lane + kWave * r < a.dim) o[r] += w * V::widen(v[lane + kWave * r]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int r = 0; r < kMaxPer; ++r)
    if (lane + kWave * r < a.dim) {
      const int64_t at = row * a.dim + lane + kWave * r;
      out[at] = V::narrow(o[r] * inv);
      if constexpr (sizeof(*out) == 2)
        if (a.low != nullptr)
          static_cast<typename V::Storage *>(a.low)[a.low_at(b, i, h, lane + kWave * r)] =
              Residue<V>::of(o[r] * inv, out[at]);
    }
  if (lse != nullptr && lane == 0)
    lse[(b * a.heads + h) * a.lq + i] = l == 0.0f ? INFINITY : m + log2_fast(l);
}

// dq by query row; also leaves delta for the keys' pass.
template <class V>
__global__ __launch_bounds__(kRowWaves * kWave) void backward_rows(
    WindowArgs a, int64_t first_row, int64_t rows, const typename V::Storage *out, const float *lse,
    const typename V::Storage *grad, int64_t g0, int64_t g1, int64_t g2, float *delta_out,
    typename V::Storage *dq) {
  __shared__ float q_lds[kRowWaves][kWindowMaxDim];
  __shared__ float g_lds[kRowWaves][kWindowMaxDim];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row = first_row + static_cast<int64_t>(blockIdx.x) * kRowWaves + wave;
  if (row >= rows) return;
  const int32_t h = static_cast<int32_t>(row % a.heads);
  const int32_t i = static_cast<int32_t>(row / a.heads % a.lq);
  const int64_t b = row / a.heads / a.lq;
  const int32_t p = i + a.lk - a.lq;
  const float lse_row = lse[(b * a.heads + h) * a.lq + i];
  float acc[kMaxPer] = {};
  float delta = 0.0f;
  if (p >= 0 && p < a.length(b) && lse_row != INFINITY) {
    const auto *q = row_of<V>(a.q, a.qs, b, i, h);
    const auto *g = grad + b * g0 + i * g1 + h * g2;
    float *ql = q_lds[wave], *gl = g_lds[wave];
    float part = 0.0f;
    for (int d = lane; d < a.dim; d += kWave) {
      ql[d] = V::widen(q[d]);
      gl[d] = V::widen(g[d]);
      float o = V::widen(out[row * a.dim + d]);
      if constexpr (sizeof(*out) == 2)
        if (a.low != nullptr)
          o += Residue<V>::value(static_cast<const typename V::Storage *>(a.low)[a.low_at(b, i, h, d)]);
      part += gl[d] * o;
    }
    delta = wave_sum(part);
    __builtin_amdgcn_wave_barrier();
    const Seen seen(p, a.window, a.sinks);
    const int32_t n = seen.count(p), kvh = h / a.group;
    for (int32_t c0 = 0; c0 < n; c0 += kWave) {
      const int32_t j = seen.key(min(c0 + lane, n - 1));
      const float s = dot_row<V>(ql, row_of<V>(a.k, a.ks, b, j, kvh), a.dim) * a.scale;
      const float dp = dot_row<V>(gl, row_of<V>(a.v, a.vs, b, j, kvh), a.dim);
      const float ds = exp2_fast(s - lse_row) * (dp - delta);
      const int32_t here = min(kWave, n - c0);
      for (int32_t t = 0; t < here; ++t) {
        const float w = __shfl(ds, t);
        const auto *k = row_of<V>(a.k, a.ks, b, seen.key(c0 + t), kvh);
#pragma unroll
        for (int r = 0; r < kMaxPer; ++r)
          if (lane + kWave * r < a.dim) acc[r] += w * V::widen(k[lane + kWave * r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kMaxPer; ++r)
    if (lane + kWave * r < a.dim)
      dq[row * a.dim + lane + kWave * r] = V::narrow(acc[r] * a.grad_scale);
  if (lane == 0) delta_out[(b * a.heads + h) * a.lq + i] = delta;
}

// dk and dv by key: one wave a key row, a lane a query of each 64 that see
// it, over the heads of its group.
template <class V>
__global__ __launch_bounds__(kRowWaves * kWave) void backward_keys(
    WindowArgs a, int64_t first_row, int64_t rows, const float *lse, const typename V::Storage *grad, int64_t g0,
    int64_t g1, int64_t g2, const float *delta, typename V::Storage *dk,
    typename V::Storage *dv) {
  __shared__ float k_lds[kRowWaves][kWindowMaxDim];
  __shared__ float v_lds[kRowWaves][kWindowMaxDim];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t row = first_row + static_cast<int64_t>(blockIdx.x) * kRowWaves + wave;  // (b, j, kv head)
  if (row >= rows) return;
  const int32_t kvh = static_cast<int32_t>(row % a.kv_heads);
  const int32_t j = static_cast<int32_t>(row / a.kv_heads % a.lk);
  const int64_t b = row / a.kv_heads / a.lk;
  const int32_t n = a.length(b);
  float acc_k[kMaxPer] = {}, acc_v[kMaxPer] = {};
  // queries at positions [first, last] see key j
  const int32_t offset = a.lk - a.lq;
  const int32_t first = max(j, max(offset, 0));
  const int32_t last = j < a.sinks || j > n - a.window ? n - 1 : j + a.window - 1;
  if (j < n && first <= last) {
    const auto *k = row_of<V>(a.k, a.ks, b, j, kvh);
    const auto *v = row_of<V>(a.v, a.vs, b, j, kvh);
    float *kl = k_lds[wave], *vl = v_lds[wave];
    for (int d = lane; d < a.dim; d += kWave) {
      kl[d] = V::widen(k[d]);
      vl[d] = V::widen(v[d]);
    }
    __builtin_amdgcn_wave_barrier();
    for (int32_t h = kvh * a.group; h < (kvh + 1) * a.group; ++h) {
      const int64_t stat = (b * a.heads + h) * a.lq;
      for (int32_t p0 = first; p0 <= last; p0 += kWave) {
        const int32_t i = min(p0 + lane, last) - offset;
        const float s = dot_row<V>(kl, row_of<V>(a.q, a.qs, b, i, h), a.dim) * a.scale;
        const float dp = dot_row<V>(vl, grad + b * g0 + i * g1 + h * g2, a.dim);
        const float top = lse[stat + i];
        const float prob = top == INFINITY ? 0.0f : exp2_fast(s - top);
        const float ds = top == INFINITY ? 0.0f : prob * (dp - delta[stat + i]);
        const int32_t here = min(kWave, last - p0 + 1);
        for (int32_t t = 0; t < here; ++t) {
          const float wp = __shfl(prob, t), ws = __shfl(ds, t);
          const int64_t it = p0 + t - offset;
          const auto *q = row_of<V>(a.q, a.qs, b, it, h);
          const auto *g = grad + b * g0 + it * g1 + h * g2;
#pragma unroll
          for (int r = 0; r < kMaxPer; ++r)
            if (lane + kWave * r < a.dim) {
              acc_k[r] += ws * V::widen(q[lane + kWave * r]);
              acc_v[r] += wp * V::widen(g[lane + kWave * r]);
            }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kMaxPer; ++r)
    if (lane + kWave * r < a.dim) {
      dk[row * a.dim + lane + kWave * r] = V::narrow(acc_k[r] * a.grad_scale);
      dv[row * a.dim + lane + kWave * r] = V::narrow(acc_v[r]);
    }
}

// ---------------------------------------------------------------------------
// Single-token step.

// One workgroup a (sequence, kv head): the token's row is written first, then
// a wave takes a query head of the group after the other.
template <class V>
__global__ __launch_bounds__(kRowWaves * kWave) void step_rows(StepArgs a,
                                                               typename V::Storage *out) {
  using S = typename V::Storage;
  __shared__ float q_lds[kRowWaves][kWindowMaxDim];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int32_t kvh = static_cast<int32_t>(blockIdx.x % a.kv_heads);
  const int64_t b = blockIdx.x / a.kv_heads;
  const int64_t p = a.length(b);
  S *ck = static_cast<S *>(a.ck) + b * a.cks[0] + kvh * a.cks[2];
  S *cv = static_cast<S *>(a.cv) + b * a.cvs[0] + kvh * a.cvs[2];
  if (p >= 0) {
    const S *k = static_cast<const S *>(a.k) + b * a.ks[0] + kvh * a.ks[1];
    const S *v = static_cast<const S *>(a.v) + b * a.vs[0] + kvh * a.vs[1];
    const int32_t at = a.slot(p);
    for (int d = threadIdx.x; d < a.dim; d += kRowWaves * kWave) {
      ck[at * a.cks[1] + d] = k[d];
      cv[at * a.cvs[1] + d] = v[d];
    }
  }
  __syncthreads();
  const int64_t near = p >= a.window ? p - a.window + 1 : 0;
  const int32_t far = static_cast<int32_t>(a.sinks < near ? a.sinks : near);
  const int32_t n = p < 0 ? 0 : far + static_cast<int32_t>(p - near) + 1;
  for (int32_t g = wave; g < a.group; g += kRowWaves) {
    const int32_t h = kvh * a.group + g;
    const S *q = static_cast<const S *>(a.q) + b * a.qs[0] + h * a.qs[1];
    float *ql = q_lds[wave];
    __builtin_amdgcn_wave_barrier();
    for (int d = lane; d < a.dim; d += kWave) ql[d] = V::widen(q[d]);
    __builtin_amdgcn_wave_barrier();
    float m = -INFINITY, l = 0.0f, o[kMaxPer] = {};
    for (int32_t c0 = 0; c0 < n; c0 += kWave) {
      const int32_t c = min(c0 + lane, n - 1);
      const int32_t at = a.slot(c < far ? c : near + c - far);
      float s = dot_row<V>(ql, ck + at * a.cks[1], a.dim) * a.scale;
      if (c0 + lane >= n) s = -INFINITY;
      const float top = fmaxf(m, wave_max(s));
      const float base = top == -INFINITY ? 0.0f : top;
      const float e = exp2_fast(s - base), keep = exp2_fast(m - base);
      l = l * keep + wave_sum(e);
      m = top;
#pragma unroll
      for (int r = 0; r < kMaxPer; ++r) o[r] *= keep;
      const int32_t here = min(kWave, n - c0);
      for (int32_t t = 0; t < here; ++t) {
        const float w = __shfl(e, t);
        const S *v = cv + static_cast<int64_t>(__shfl(at, t)) * a.cvs[1];
#pragma unroll
        for (int r = 0; r < kMaxPer; ++r)
          if (lane + kWave * r < a.dim) o[r] += w * V::widen(v[lane + kWave * r]);
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int r = 0; r < kMaxPer; ++r)
      if (lane + kWave * r < a.dim)
        out[(b * a.heads + h) * a.dim + lane + kWave * r] = V::narrow(o[r] * inv);
  }
}

struct StoreArgs {
  int64_t batch;
  int32_t kv_heads, dim, slots, sinks, tokens;
  const void *starts, *lengths;
  int32_t index64;
  const void *k, *v;
  int64_t ks[3], vs[3];
  void *ck, *cv;
  int64_t cks[3], cvs[3];

  __device__ inline int64_t index(const void *p, int64_t b, int64_t none) const {
    if (p == nullptr) return none;
    return index64 ? static_cast<const int64_t *>(p)[b] : static_cast<const int32_t *>(p)[b];
  }
};

// One wave a (sequence, token, kv head).
template <class S>
__global__ __launch_bounds__(kRowWaves * kWave) void store_rows(StoreArgs a, int64_t first, int64_t rows) {
  const int lane = threadIdx.x % kWave;
  const int64_t row = first + static_cast<int64_t>(blockIdx.x) * kRowWaves + threadIdx.x / kWave;
  if (row >= rows) return;
  const int32_t h = static_cast<int32_t>(row % a.kv_heads);
  const int32_t t = static_cast<int32_t>(row / a.kv_heads % a.tokens);
  const int64_t b = row / a.kv_heads / a.tokens;
  const int64_t start = a.index(a.starts, b, 0);
  const int64_t n = min(a.index(a.lengths, b, a.tokens), static_cast<int64_t>(a.tokens));
  const int64_t p = start + t, ring = a.slots - a.sinks;
  // later tokens of the same call take the slots of those a ring before them
  if (start < 0 || t >= n || (p >= a.sinks && p < start + n - ring)) return;
  const int64_t at = p < a.sinks ? p : a.sinks + (p - a.sinks) % ring;
  const S *k = static_cast<const S *>(a.k) + b * a.ks[0] + t * a.ks[1] + h * a.ks[2];
  const S *v = static_cast<const S *>(a.v) + b * a.vs[0] + t * a.vs[1] + h * a.vs[2];
  S *ck = static_cast<S *>(a.ck) + b * a.cks[0] + at * a.cks[1] + h * a.cks[2];
  S *cv = static_cast<S *>(a.cv) + b * a.cvs[0] + at * a.cvs[1] + h * a.cvs[2];
  for (int d = lane; d < a.dim; d += kWave) {
    ck[d] = k[d];
    cv[d] = v[d];
  }
}

WindowArgs args_of(const msx_window_attention_desc &d) {
  WindowArgs a{};
  a.batch = d.batch;
  a.lq = static_cast<int32_t>(d.lq);
  a.lk = static_cast<int32_t>(d.lk);
  a.heads = static_cast<int32_t>(d.heads);
  a.kv_heads = static_cast<int32_t>(d.kv_heads);
  a.group = a.heads / a.kv_heads;
  a.dim = static_cast<int32_t>(d.dim);
  a.window = static_cast<int32_t>(std::min<int64_t>(d.window, std::max<int64_t>(d.lk, 1)));
  a.sinks = static_cast<int32_t>(std::min(d.sinks, d.lk));
  a.scale = static_cast<float>(d.scale * 1.44269504088896340736);
  a.grad_scale = static_cast<float>(d.scale);
  a.lengths = d.lengths;
  a.lengths64 = d.lengths_itype == MSX_I64;
  a.q = d.q;
  a.k = d.k;
  a.v = d.v;
  a.low = d.out_low;
  std::copy(d.q_strides, d.q_strides + 3, a.qs);
  std::copy(d.k_strides, d.k_strides + 3, a.ks);
  std::copy(d.v_strides, d.v_strides + 3, a.vs);
  return a;
}

// Whether the tiles' kernels can read the operands: sixteen-byte rows at
// sixteen-byte strides, a head of at most 128 values, and a scale that a
// masked score (minus infinity times it) survives.
bool rows_aligned(size_t size, const void *p, const int64_t *strides, int n) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < n; ++i) ok = ok && strides[i] * static_cast<int64_t>(size) % 16 == 0;
  return ok;
}

bool takes_tiles(const msx_window_attention_desc &d) {
  const size_t size = value_bytes(static_cast<msx_vtype>(d.vtype));
  return d.dim <= 128 && d.dim * size % 16 == 0 &&
         std::fabs(static_cast<float>(d.scale)) >= std::numeric_limits<float>::min() &&
         rows_aligned(size, d.q, d.q_strides, 3) && rows_aligned(size, d.k, d.k_strides, 3) &&
         rows_aligned(size, d.v, d.v_strides, 3);
}

StepArgs args_of(const msx_window_step_desc &d) {
  StepArgs a{};
  a.batch = d.batch;
  a.heads = static_cast<int32_t>(d.heads);
  a.kv_heads = static_cast<int32_t>(d.kv_heads);
  a.group = a.heads / a.kv_heads;
  a.dim = static_cast<int32_t>(d.dim);
  a.slots = static_cast<int32_t>(d.slots);
  a.window = static_cast<int32_t>(d.window);
  a.sinks = static_cast<int32_t>(d.sinks);
  a.scale = static_cast<float>(d.scale * 1.44269504088896340736);
  a.lengths = d.lengths;
  a.lengths64 = d.lengths_itype == MSX_I64;
  a.q = d.q;
  a.k = d.k;
  a.v = d.v;
  a.ck = d.cache_k;
  a.cv = d.cache_v;
  std::copy(d.q_strides, d.q_strides + 2, a.qs);
  std::copy(d.k_strides, d.k_strides + 2, a.ks);
  std::copy(d.v_strides, d.v_strides + 2, a.vs);
  std::copy(d.cache_k_strides, d.cache_k_strides + 3, a.cks);
  std::copy(d.cache_v_strides, d.cache_v_strides + 3, a.cvs);
  return a;
}

bool takes_tiles(const msx_window_step_desc &d) {
  const size_t size = value_bytes(static_cast<msx_vtype>(d.vtype));
  return d.dim * size % 16 == 0 && rows_aligned(size, d.q, d.q_strides, 2) &&
         rows_aligned(size, d.k, d.k_strides, 2) && rows_aligned(size, d.v, d.v_strides, 2) &&
         rows_aligned(size, d.cache_k, d.cache_k_strides, 3) &&
         rows_aligned(size, d.cache_v, d.cache_v_strides, 3);
}

// delta, before the tiles' sums (which need sixteen-byte addresses).
size_t delta_bytes(const msx_window_attention_desc &d) {
  return (sizeof(float) * static_cast<size_t>(d.batch * d.heads * d.lq) + 255) / 256 * 256;
}

// fn(first row, workgroups) over `rows` rows, a wave each: launches of as many as
// one holds.
template <class Fn>
void each_launch(int64_t rows, Fn &&fn) {
  constexpr int64_t kMost = max_blocks(kRowWaves * kWave) * kRowWaves;
  for (int64_t first = 0; first < rows; first += kMost)
    fn(first, static_cast<unsigned>((std::min(rows - first, kMost) + kRowWaves - 1) / kRowWaves));
}

template <class Fn>
msx_status by_vtype(int vt, Fn &&fn) {
  switch (vt) {
  case MSX_F32: return fn(F32{});
  case MSX_F16: return fn(F16{});
  default: return fn(BF16{});
  }
}

msx_status launched(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, what);
}

}  // namespace
}  // namespace msx

using namespace msx;

extern "C" size_t msx_window_attention_scratch(const msx_window_attention_desc *desc) {
  if (check_window_attention("window_attention", desc) != MSX_OK || desc->batch == 0 ||
      desc->lq == 0 || !takes_tiles(*desc))
    return 0;
  return window_forward_scratch(static_cast<msx_vtype>(desc->vtype), args_of(*desc));
}

extern "C" msx_status msx_window_attention(const msx_window_attention_desc *desc, void *out,
                                           float *lse, void *scratch, size_t scratch_bytes,
                                           void *stream) {
  clear_error();
  if (msx_status st = check_window_attention("window_attention", desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->lq == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "window_attention out is NULL.");
  const WindowArgs a = args_of(*desc);
  if (takes_tiles(*desc) && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
      reinterpret_cast<uintptr_t>(desc->out_low) % 16 == 0) {
    const auto vt = static_cast<msx_vtype>(desc->vtype);
    const size_t need = window_forward_scratch(vt, a);
    if (scratch_bytes < need || (need > 0 && (scratch == nullptr ||
                                              reinterpret_cast<uintptr_t>(scratch) % 16 != 0)))
      return fail(MSX_EINVAL, "window_attention scratch is too small or not aligned.");
    return launch_window_forward(vt, a, out, lse, scratch, static_cast<hipStream_t>(stream));
  }
  const int64_t rows = a.batch * a.lq * a.heads;
  return by_vtype(desc->vtype, [&](auto v) {
    using V = decltype(v);
    each_launch(rows, [&](int64_t first, unsigned blocks) {
      forward_rows<V><<<blocks, kRowWaves * kWave, 0, static_cast<hipStream_t>(stream)>>>(
          a, first, rows, static_cast<typename V::Storage *>(out), lse);
    });
    return launched("window_attention");
  });
}

extern "C" size_t msx_window_attention_backward_scratch(const msx_window_attention_desc *desc) {
  if (check_window_attention("window_attention_backward", desc) != MSX_OK || desc->batch == 0)
    return 0;
  const size_t tiles = takes_tiles(*desc) ? window_backward_scratch(static_cast<msx_vtype>(desc->vtype), args_of(*desc)) : 0;
  return delta_bytes(*desc) + tiles;
}

extern "C" msx_status msx_window_attention_backward(const msx_window_attention_desc *desc,
                                                    const void *out, const float *lse,
                                                    const void *grad, const int64_t *grad_strides,
                                                    void *dq, void *dk, void *dv, void *scratch,
                                                    size_t scratch_bytes, void *stream) {
  clear_error();
  const char *op = "window_attention_backward";
  if (msx_status st = check_window_attention(op, desc); st != MSX_OK) return st;
  const bool queries = desc->batch > 0 && desc->lq > 0, keys = desc->batch > 0 && desc->lk > 0;
  if (!queries && !keys) return MSX_OK;
  if (queries && (out == nullptr || lse == nullptr || grad == nullptr || grad_strides == nullptr ||
                  dq == nullptr))
    return fail(MSX_EINVAL, "window_attention_backward buffers must be non-NULL.");
  if (keys && (dk == nullptr || dv == nullptr))
    return fail(MSX_EINVAL, "window_attention_backward dk and dv must be non-NULL.");
  if (scratch_bytes < msx_window_attention_backward_scratch(desc) || (queries && scratch == nullptr))
    return fail(MSX_EINVAL, "window_attention_backward scratch is too small.");
  const WindowArgs a = args_of(*desc);
  const size_t size = value_bytes(static_cast<msx_vtype>(desc->vtype));
  const auto aligned = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (queries && keys && takes_tiles(*desc) && rows_aligned(size, grad, grad_strides, 3) &&
      aligned(out) && aligned(desc->out_low) && aligned(dq) && aligned(dk) && aligned(dv) && aligned(scratch))
    return launch_window_backward(static_cast<msx_vtype>(desc->vtype), a, out, lse, grad,
                                  grad_strides, static_cast<float *>(scratch), dq, dk, dv,
                                  static_cast<char *>(scratch) + delta_bytes(*desc),
                                  static_cast<hipStream_t>(stream));
  const int64_t q_rows = a.batch * a.lq * a.heads, k_rows = a.batch * a.lk * a.kv_heads;
  const int64_t gs[3] = {queries ? grad_strides[0] : 0, queries ? grad_strides[1] : 0,
                         queries ? grad_strides[2] : 0};
  return by_vtype(desc->vtype, [&](auto v) {
    using V = decltype(v);
    using S = typename V::Storage;
    const auto s = static_cast<hipStream_t>(stream);
    float *delta = static_cast<float *>(scratch);
    each_launch(q_rows, [&](int64_t first, unsigned blocks) {
      backward_rows<V><<<blocks, kRowWaves * kWave, 0, s>>>(
          a, first, q_rows, static_cast<const S *>(out), lse, static_cast<const S *>(grad), gs[0],
          gs[1], gs[2], delta, static_cast<S *>(dq));
    });
    each_launch(k_rows, [&](int64_t first, unsigned blocks) {
      backward_keys<V><<<blocks, kRowWaves * kWave, 0, s>>>(
          a, first, k_rows, lse, static_cast<const S *>(grad), gs[0], gs[1], gs[2], delta,
          static_cast<S *>(dk), static_cast<S *>(dv));
    });
    return launched("window_attention_backward");
  });
}

extern "C" size_t msx_window_attention_step_scratch(const msx_window_step_desc *desc) {
  if (check_window_step("window_attention_step", desc) != MSX_OK || desc->batch == 0) return 0;
  return takes_tiles(*desc)
             ? window_step_scratch(static_cast<msx_vtype>(desc->vtype), args_of(*desc))
             : 0;
}

extern "C" msx_status msx_window_attention_step(const msx_window_step_desc *desc, void *out,
                                                void *scratch, size_t scratch_bytes,
                                                void *stream) {
  clear_error();
  const char *op = "window_attention_step";
  if (msx_status st = check_window_step(op, desc); st != MSX_OK) return st;
  const msx_window_step_desc &d = *desc;
  if (d.batch == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "window_attention_step out is NULL.");
  if (d.batch * d.kv_heads > max_blocks(kRowWaves * kWave))
    return fail(MSX_EINVAL, "window_attention_step has more rows than a grid holds.");
  const StepArgs a = args_of(d);
  const msx_vtype vt = static_cast<msx_vtype>(d.vtype);
  if (takes_tiles(d)) {
    const size_t need = window_step_scratch(vt, a);
    if (scratch_bytes < need || (need > 0 && scratch == nullptr))
      return fail(MSX_EINVAL, "window_attention_step scratch is too small.");
    return launch_window_step(vt, a, out, scratch, static_cast<hipStream_t>(stream));
  }
  return by_vtype(d.vtype, [&](auto v) {
    using V = decltype(v);
    step_rows<V><<<static_cast<unsigned>(a.batch * a.kv_heads), kRowWaves * kWave, 0,
                   static_cast<hipStream_t>(stream)>>>(a, static_cast<typename V::Storage *>(out));
    return launched("window_attention_step");
  });
}

extern "C" msx_status msx_window_cache_store(const msx_window_step_desc *desc, int64_t tokens,
                                             const void *k, const int64_t *k_strides,
                                             const void *v, const int64_t *v_strides,
                                             msx_itype itype, const void *starts,
                                             const void *lengths, void *stream) {
  clear_error();
  const char *op = "window_cache_store";
  if (msx_status st = check_window_store(op, desc, tokens, k, k_strides, v, v_strides, itype);
      st != MSX_OK)
    return st;
  const msx_window_step_desc &d = *desc;
  if (d.batch == 0 || tokens == 0) return MSX_OK;
  StoreArgs a{};
  a.batch = d.batch;
  a.kv_heads = static_cast<int32_t>(d.kv_heads);
  a.dim = static_cast<int32_t>(d.dim);
  a.slots = static_cast<int32_t>(d.slots);
  a.sinks = static_cast<int32_t>(d.sinks);
  a.tokens = static_cast<int32_t>(tokens);
  a.starts = starts;
  a.lengths = lengths;
  a.index64 = itype == MSX_I64;
  a.k = k;
  a.v = v;
  a.ck = d.cache_k;
  a.cv = d.cache_v;
  std::copy(k_strides, k_strides + 3, a.ks);
  std::copy(v_strides, v_strides + 3, a.vs);
  std::copy(d.cache_k_strides, d.cache_k_strides + 3, a.cks);
  std::copy(d.cache_v_strides, d.cache_v_strides + 3, a.cvs);
  const int64_t rows = a.batch * a.tokens * a.kv_heads;
  const auto s = static_cast<hipStream_t>(stream);
  each_launch(rows, [&](int64_t first, unsigned blocks) {
    if (d.vtype == MSX_F32)
      store_rows<uint32_t><<<blocks, kRowWaves * kWave, 0, s>>>(a, first, rows);
    else
      store_rows<uint16_t><<<blocks, kRowWaves * kWave, 0, s>>>(a, first, rows);
  });
  return launched("window_cache_store");
}
