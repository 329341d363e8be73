// window_attention_cpu.cpp - the `use_cpu()` path of window attention: a
// query (or a key, for dk and dv) after the other, sums in float32.
#include <cmath>
#include <new>

#include "msx_host_values.h"
#include "msx_sparse.h"
#include "msx_window_check.h"

namespace {

using namespace msx;
using namespace msx::host;

int64_t length_of(const msx_window_attention_desc &d, int64_t b) {
  if (d.lengths == nullptr) return d.lk;
  return std::min(std::max<int64_t>(index_at(d.lengths, d.lengths_itype == MSX_I64, b), 0), d.lk);
}

// Calls fn(j) for every key that position p sees.
template <class Fn>
void each_seen(int64_t p, int64_t window, int64_t sinks, Fn &&fn) {
  const int64_t near = p >= window ? p - window + 1 : 0;
  for (int64_t j = 0; j < std::min(sinks, near); ++j) fn(j);
  for (int64_t j = near; j <= p; ++j) fn(j);
}

template <class V>
const typename V::Storage *at(const void *base, const int64_t *strides, int64_t b, int64_t t,
                              int64_t h) {
  return static_cast<const typename V::Storage *>(base) + b * strides[0] + t * strides[1] +
         h * strides[2];
}

template <class V>
float dot(const typename V::Storage *x, const typename V::Storage *y, int64_t n) {
  float acc = 0.0f;
  for (int64_t i = 0; i < n; ++i) acc += V::widen(x[i]) * V::widen(y[i]);
  return acc;
}

// float16's residues are held 2^10 larger: see Residue in msx_window.h.
template <class V>
constexpr float kLowUp = 1.0f;
template <>
constexpr float kLowUp<F16> = 1024.0f;

// Where the residues of query i, head h lie: a sequence's after the other's as on
// the device (a batch can be cut or joined), a sequence's in out's order.
int64_t low_at(const msx_window_attention_desc &d, int64_t b, int64_t i, int64_t h) {
  return b * d.heads * ((d.lq + 31) / 32 * 32) * ((d.dim + 7) / 8 * 8) + (i * d.heads + h) * d.dim;
}

// Attention of one query over the listed rows; returns the base-2 logarithm
// of the softmax's sum (+inf without one).  `low` (or null): what rounding
// leaves of the output, as the device keeps it.
template <class V>
float attend(const typename V::Storage *q, const std::vector<const typename V::Storage *> &k,
             const std::vector<const typename V::Storage *> &v, int64_t dim, float scale,
             std::vector<float> &s, std::vector<float> &o, typename V::Storage *out,
             typename V::Storage *low = nullptr) {
  float top = -INFINITY, sum = 0.0f;
  s.resize(k.size());
  for (size_t j = 0; j < k.size(); ++j) {
    s[j] = dot<V>(q, k[j], dim) * scale;
    top = std::fmax(top, s[j]);
  }
  const float base = top == -INFINITY ? 0.0f : top;
  o.assign(static_cast<size_t>(dim), 0.0f);
  for (size_t j = 0; j < k.size(); ++j) {
    const float e = std::exp(s[j] - base);
    sum += e;
    for (int64_t x = 0; x < dim; ++x) o[x] += e * V::widen(v[j][x]);
  }
  for (int64_t x = 0; x < dim; ++x) {
    const float value = sum == 0.0f ? 0.0f : o[x] / sum;
    out[x] = V::narrow(value);
    if (low != nullptr) low[x] = V::narrow((value - V::widen(out[x])) * kLowUp<V>);
  }
  return sum == 0.0f ? INFINITY : (base + std::log(sum)) * 1.44269504088896340736f;
}

template <class V>
void forward(const msx_window_attention_desc &d, void *out, float *lse, int n_threads) {
  using S = typename V::Storage;
  const int64_t group = d.heads / d.kv_heads;
  S *low = sizeof(S) == 2 ? static_cast<S *>(d.out_low) : nullptr;
  split(d.batch * d.heads * d.lq, n_threads, [&](int64_t first, int64_t last) {
    std::vector<const S *> k, v;
    std::vector<float> s, o;
    for (int64_t r = first; r < last; ++r) {
      const int64_t i = r % d.lq, h = r / d.lq % d.heads, b = r / d.lq / d.heads;
      const int64_t p = i + d.lk - d.lq;
      k.clear();
      v.clear();
      if (p >= 0 && p < length_of(d, b))
        each_seen(p, d.window, d.sinks, [&](int64_t j) {
          k.push_back(at<V>(d.k, d.k_strides, b, j, h / group));
          v.push_back(at<V>(d.v, d.v_strides, b, j, h / group));
        });
      const int64_t to = ((b * d.lq + i) * d.heads + h) * d.dim;
      const float l = attend<V>(at<V>(d.q, d.q_strides, b, i, h), k, v, d.dim,
                                static_cast<float>(d.scale), s, o, static_cast<S *>(out) + to,
                                low == nullptr ? nullptr : low + low_at(d, b, i, h));
      if (lse != nullptr) lse[r] = l;
    }
  });
}

// One (sequence, kv head) after the other: its dk and dv are summed by one
// thread, so in one order.
template <class V>
void backward(const msx_window_attention_desc &d, const void *out, const float *lse,
              const void *grad, const int64_t *gs, void *dq, void *dk, void *dv, int n_threads) {
  using S = typename V::Storage;
  const int64_t group = d.heads / d.kv_heads, dim = d.dim;
  const float scale = static_cast<float>(d.scale);
  const S *low = sizeof(S) == 2 ? static_cast<const S *>(d.out_low) : nullptr;
  split(d.batch * d.kv_heads, n_threads, [&](int64_t first, int64_t last) {
    std::vector<float> sum_k(static_cast<size_t>(d.lk * dim)), sum_v(sum_k.size()), sum_q(dim);
    for (int64_t r = first; r < last; ++r) {
      const int64_t kvh = r % d.kv_heads, b = r / d.kv_heads, n = length_of(d, b);
      std::fill(sum_k.begin(), sum_k.end(), 0.0f);
      std::fill(sum_v.begin(), sum_v.end(), 0.0f);
      for (int64_t h = kvh * group; h < (kvh + 1) * group; ++h)
        for (int64_t i = 0; i < d.lq; ++i) {
          const int64_t p = i + d.lk - d.lq, at_out = ((b * d.lq + i) * d.heads + h) * dim;
          const float l = lse[(b * d.heads + h) * d.lq + i];
          std::fill(sum_q.begin(), sum_q.end(), 0.0f);
          if (p >= 0 && p < n && l != INFINITY) {
            const S *q = at<V>(d.q, d.q_strides, b, i, h), *g = at<V>(grad, gs, b, i, h);
            float delta = dot<V>(g, static_cast<const S *>(out) + at_out, dim);
            if (low != nullptr) delta += dot<V>(g, low + low_at(d, b, i, h), dim) / kLowUp<V>;
            each_seen(p, d.window, d.sinks, [&](int64_t j) {
              const S *k = at<V>(d.k, d.k_strides, b, j, kvh), *v = at<V>(d.v, d.v_strides, b, j, kvh);
              const float prob = std::exp2(dot<V>(q, k, dim) * scale * 1.44269504088896340736f - l);
              const float ds = prob * (dot<V>(g, v, dim) - delta);
              for (int64_t x = 0; x < dim; ++x) {
                sum_q[x] += ds * V::widen(k[x]);
                sum_k[j * dim + x] += ds * V::widen(q[x]);
                sum_v[j * dim + x] += prob * V::widen(g[x]);
              }
            });
          }
          for (int64_t x = 0; x < dim; ++x)
            static_cast<S *>(dq)[at_out + x] = V::narrow(sum_q[x] * scale);
        }
      for (int64_t j = 0; j < d.lk; ++j)
        for (int64_t x = 0; x < dim; ++x) {
          const int64_t to = ((b * d.lk + j) * d.kv_heads + kvh) * dim + x;
          static_cast<S *>(dk)[to] = V::narrow(sum_k[j * dim + x] * scale);
          static_cast<S *>(dv)[to] = V::narrow(sum_v[j * dim + x]);
        }
    }
  });
}

int64_t slot_of(const msx_window_step_desc &d, int64_t j) {
  return j < d.sinks ? j : d.sinks + (j - d.sinks) % (d.slots - d.sinks);
}

template <class V>
void step(const msx_window_step_desc &d, void *out, int n_threads) {
  using S = typename V::Storage;
  const int64_t group = d.heads / d.kv_heads;
  split(d.batch * d.kv_heads, n_threads, [&](int64_t first, int64_t last) {
    std::vector<const S *> k, v;
    std::vector<float> s, o;
    for (int64_t r = first; r < last; ++r) {
      const int64_t kvh = r % d.kv_heads, b = r / d.kv_heads;
      const int64_t p = index_at(d.lengths, d.lengths_itype == MSX_I64, b);
      S *ck = static_cast<S *>(d.cache_k) + b * d.cache_k_strides[0] + kvh * d.cache_k_strides[2];
      S *cv = static_cast<S *>(d.cache_v) + b * d.cache_v_strides[0] + kvh * d.cache_v_strides[2];
      k.clear();
      v.clear();
      if (p >= 0) {
        const S *new_k = static_cast<const S *>(d.k) + b * d.k_strides[0] + kvh * d.k_strides[1];
        const S *new_v = static_cast<const S *>(d.v) + b * d.v_strides[0] + kvh * d.v_strides[1];
        std::copy(new_k, new_k + d.dim, ck + slot_of(d, p) * d.cache_k_strides[1]);
        std::copy(new_v, new_v + d.dim, cv + slot_of(d, p) * d.cache_v_strides[1]);
        each_seen(p, d.window, d.sinks, [&](int64_t j) {
          k.push_back(ck + slot_of(d, j) * d.cache_k_strides[1]);
          v.push_back(cv + slot_of(d, j) * d.cache_v_strides[1]);
        });
      }
      for (int64_t h = kvh * group; h < (kvh + 1) * group; ++h)
        attend<V>(static_cast<const S *>(d.q) + b * d.q_strides[0] + h * d.q_strides[1], k, v,
                  d.dim, static_cast<float>(d.scale), s, o,
                  static_cast<S *>(out) + (b * d.heads + h) * d.dim);
    }
  });
}

template <class S>
void store(const msx_window_step_desc &d, int64_t tokens, const void *k, const int64_t *ks,
           const void *v, const int64_t *vs, bool i64, const void *starts, const void *lengths) {
  const int64_t ring = d.slots - d.sinks;
  for (int64_t b = 0; b < d.batch; ++b) {
    const int64_t start = starts == nullptr ? 0 : index_at(starts, i64, b);
    const int64_t n = std::min(lengths == nullptr ? tokens : index_at(lengths, i64, b), tokens);
    if (start < 0) continue;
    for (int64_t t = 0; t < n; ++t) {
      const int64_t p = start + t;
      if (p >= d.sinks && p < start + n - ring) continue;
      const int64_t to = slot_of(d, p);
      for (int64_t h = 0; h < d.kv_heads; ++h) {
        const S *from_k = static_cast<const S *>(k) + b * ks[0] + t * ks[1] + h * ks[2];
        const S *from_v = static_cast<const S *>(v) + b * vs[0] + t * vs[1] + h * vs[2];
        std::copy(from_k, from_k + d.dim, static_cast<S *>(d.cache_k) + b * d.cache_k_strides[0] +
                                              to * d.cache_k_strides[1] + h * d.cache_k_strides[2]);
        std::copy(from_v, from_v + d.dim, static_cast<S *>(d.cache_v) + b * d.cache_v_strides[0] +
                                              to * d.cache_v_strides[1] + h * d.cache_v_strides[2]);
      }
    }
  }
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

extern "C" msx_status msx_window_attention_cpu(const msx_window_attention_desc *desc, void *out,
                                               float *lse, int n_threads) {
  clear_error();
  if (msx_status st = check_window_attention("window_attention", desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->lq == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "window_attention out is NULL.");
  return guarded("window_attention", [&] {
    by_vtype(desc->vtype, [&](auto v) { forward<decltype(v)>(*desc, out, lse, n_threads); });
  });
}

extern "C" msx_status msx_window_attention_backward_cpu(const msx_window_attention_desc *desc,
                                                        const void *out, const float *lse,
                                                        const void *grad,
                                                        const int64_t *grad_strides, void *dq,
                                                        void *dk, void *dv, int n_threads) {
  clear_error();
  const char *op = "window_attention_backward";
  if (msx_status st = check_window_attention(op, desc); st != MSX_OK) return st;
  if (desc->batch == 0) return MSX_OK;
  if ((desc->lq > 0 && (out == nullptr || lse == nullptr || grad == nullptr ||
                        grad_strides == nullptr || dq == nullptr)) ||
      (desc->lk > 0 && (dk == nullptr || dv == nullptr)))
    return fail(MSX_EINVAL, "window_attention_backward buffers must be non-NULL.");
  return guarded(op, [&] {
    by_vtype(desc->vtype, [&](auto v) {
      backward<decltype(v)>(*desc, out, lse, grad, grad_strides, dq, dk, dv, n_threads);
    });
  });
}

extern "C" msx_status msx_window_attention_step_cpu(const msx_window_step_desc *desc, void *out,
                                                    int n_threads) {
  clear_error();
  if (msx_status st = check_window_step("window_attention_step", desc); st != MSX_OK) return st;
  if (desc->batch == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "window_attention_step out is NULL.");
  return guarded("window_attention_step", [&] {
    by_vtype(desc->vtype, [&](auto v) { step<decltype(v)>(*desc, out, n_threads); });
  });
}

extern "C" msx_status msx_window_cache_store_cpu(const msx_window_step_desc *desc, int64_t tokens,
                                                 const void *k, const int64_t *k_strides,
                                                 const void *v, const int64_t *v_strides,
                                                 msx_itype itype, const void *starts,
                                                 const void *lengths) {
  clear_error();
  if (msx_status st = check_window_store("window_cache_store", desc, tokens, k, k_strides, v,
                                         v_strides, itype);
      st != MSX_OK)
    return st;
  if (desc->vtype == MSX_F32)
    store<uint32_t>(*desc, tokens, k, k_strides, v, v_strides, itype == MSX_I64, starts, lengths);
  else
    store<uint16_t>(*desc, tokens, k, k_strides, v, v_strides, itype == MSX_I64, starts, lengths);
  return MSX_OK;
}
