// distill_cpu.cpp - the `use_cpu()` path of distillation from a teacher's top
// logits: one row after the other, statistics and sums in float32.
#include <cmath>
#include <new>

#include "msx_host_values.h"
#include "msx_sparse.h"
#include "msx_window_check.h"

namespace {

using namespace msx;
using namespace msx::host;

float kept_at(const msx_distill_desc &d, int64_t e) {
  float v;
  if (d.teacher_vtype == MSX_F32) v = static_cast<const float *>(d.data)[e];
  else if (d.teacher_vtype == MSX_F16) v = F16::widen(static_cast<const uint16_t *>(d.data)[e]);
  else v = BF16::widen(static_cast<const uint16_t *>(d.data)[e]);
  return v / static_cast<float>(d.temperature);
}

struct Kept {
  std::vector<int64_t> columns;
  std::vector<float> p, log_p;
};

// The row's distribution over its kept logits; empty without one.
void read_kept(const msx_distill_desc &d, int64_t row, Kept &k) {
  k.columns.clear();
  k.log_p.clear();
  const bool i64 = d.itype == MSX_I64;
  const auto clamp = [&](int64_t p) { return std::min(std::max<int64_t>(p, 0), d.nnz); };
  const int64_t begin = clamp(index_at(d.indptr, i64, row));
  const int64_t end = clamp(index_at(d.indptr, i64, row + 1));
  float top = -INFINITY;
  for (int64_t e = begin; e < end; ++e) {
    const int64_t c = index_at(d.indices, i64, e);
    if (c < 0 || c >= d.n_cols) continue;
    k.columns.push_back(c);
    k.log_p.push_back(kept_at(d, e));
    top = std::fmax(top, k.log_p.back());
  }
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (float v : k.log_p) sum += std::exp(v - base);
  if (sum == 0.0f) k.columns.clear();
  k.p.resize(k.columns.size());
  for (size_t r = 0; r < k.columns.size(); ++r) {
    k.log_p[r] = k.log_p[r] - base - std::log(sum);
    k.p[r] = std::exp(k.log_p[r]);
  }
}

template <class V>
void losses_of(const msx_distill_desc &d, float *losses, float *lse, int n_threads) {
  const float t = static_cast<float>(d.temperature);
  split(d.n_rows, n_threads, [&](int64_t first, int64_t last) {
    Kept k;
    for (int64_t row = first; row < last; ++row) {
      read_kept(d, row, k);
      losses[row] = 0.0f;
      if (lse != nullptr) lse[row] = 0.0f;
      if (k.columns.empty()) continue;
      const auto *z = static_cast<const typename V::Storage *>(d.logits) + row * d.ld;
      float top = -INFINITY;
      for (int64_t c = 0; c < d.n_cols; ++c) top = std::fmax(top, V::widen(z[c]) / t);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f;
      for (int64_t c = 0; c < d.n_cols; ++c) sum += std::exp(V::widen(z[c]) / t - base);
      const float total = base + std::log(sum);
      float loss = 0.0f;
      for (size_t r = 0; r < k.columns.size(); ++r)
        if (k.p[r] != 0.0f) loss += k.p[r] * (k.log_p[r] - (V::widen(z[k.columns[r]]) / t - total));
      losses[row] = loss * t * t;
      if (lse != nullptr) lse[row] = total;
    }
  });
}

template <class V>
void gradients_of(const msx_distill_desc &d, const float *lse, void *grad, int64_t ld_grad,
                  int n_threads) {
  const float t = static_cast<float>(d.temperature);
  split(d.n_rows, n_threads, [&](int64_t first, int64_t last) {
    Kept k;
    std::vector<float> g(static_cast<size_t>(d.n_cols));
    for (int64_t row = first; row < last; ++row) {
      read_kept(d, row, k);
      const auto *z = static_cast<const typename V::Storage *>(d.logits) + row * d.ld;
      auto *out = static_cast<typename V::Storage *>(grad) + row * ld_grad;
      const float weight = d.weights == nullptr ? 1.0f : d.weights[row * d.weights_stride];
      if (k.columns.empty() || weight == 0.0f) {
        std::fill(out, out + d.n_cols, typename V::Storage{0});
        continue;
      }
      for (int64_t c = 0; c < d.n_cols; ++c) g[c] = std::exp(V::widen(z[c]) / t - lse[row]);
      for (size_t r = 0; r < k.columns.size(); ++r) g[k.columns[r]] -= k.p[r];
      for (int64_t c = 0; c < d.n_cols; ++c) out[c] = V::narrow(g[c] * weight * t);
    }
  });
}

// No C++ exception leaves a C entry point.
template <class Fn>
msx_status guarded(const char *op, Fn &&fn) {
  try {
    fn();
    return MSX_OK;
  } catch (const std::bad_alloc &) {
    return fail(MSX_ENOMEM, std::string(op) + ": out of host memory.");
  } catch (const std::exception &e) {
    return fail(MSX_ENOMEM, std::string(op) + ": " + e.what());
  }
}

}  // namespace

extern "C" msx_status msx_distill_loss_cpu(const msx_distill_desc *desc, float *losses, float *lse,
                                           int n_threads) {
  clear_error();
  if (msx_status st = check_distill("distill_loss", desc); st != MSX_OK) return st;
  if (desc->n_rows == 0) return MSX_OK;
  if (losses == nullptr) return fail(MSX_EINVAL, "distill_loss losses is NULL.");
  return guarded("distill_loss", [&] {
    by_vtype(desc->vtype, [&](auto v) { losses_of<decltype(v)>(*desc, losses, lse, n_threads); });
  });
}

extern "C" msx_status msx_distill_grad_cpu(const msx_distill_desc *desc, const float *lse,
                                           void *grad, int64_t ld_grad, int n_threads) {
  clear_error();
  if (msx_status st = check_distill("distill_grad", desc); st != MSX_OK) return st;
  if (desc->n_rows == 0 || desc->n_cols == 0) return MSX_OK;
  if (grad == nullptr || lse == nullptr)
    return fail(MSX_EINVAL, "distill_grad grad and lse must be non-NULL.");
  if (ld_grad < desc->n_cols)
    return fail(MSX_EINVAL, "distill_grad leading dimension must be at least the column count.");
  return guarded("distill_grad", [&] {
    by_vtype(desc->vtype,
             [&](auto v) { gradients_of<decltype(v)>(*desc, lse, grad, ld_grad, n_threads); });
  });
}
