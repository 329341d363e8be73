// paged_cpu.cpp - the `use_cpu()` path of rotary positions, paged caches and the
// attention over them: a token (or a query and head) after the other, angles in
// 64 bits, sums in float32.
#include <cmath>
#include <new>

#include "msx_host_values.h"
#include "msx_paged_check.h"
#include "msx_sparse.h"

namespace {

using namespace msx;
using namespace msx::host;

// Cosines and sines of a token's pairs.
struct Turned {
  std::vector<float> cosine, sine;
  void at(const msx_rotation &r, double position) {
    const size_t pairs = static_cast<size_t>(r.dim / 2);
    cosine.resize(pairs);
    sine.resize(pairs);
    for (size_t i = 0; i < pairs; ++i) {
      double t = r.turns[i] * position;
      t = (t - std::rint(t)) * 6.28318530717958647693;
      cosine[i] = static_cast<float>(std::cos(t) * r.magnitude);
      sine[i] = static_cast<float>(std::sin(t) * (r.inverse ? -r.magnitude : r.magnitude));
    }
  }
  template <class V>
  void head(const msx_rotation &r, const typename V::Storage *from, typename V::Storage *to,
            int64_t dim) const {
    const int64_t half = r.dim / 2;
    for (int64_t i = 0; i < half; ++i) {
      const int64_t x = r.interleaved ? 2 * i : i, y = r.interleaved ? 2 * i + 1 : i + half;
      const float a = V::widen(from[x]), b = V::widen(from[y]);
      to[x] = V::narrow(a * cosine[i] - b * sine[i]);
      to[y] = V::narrow(a * sine[i] + b * cosine[i]);
    }
    std::copy(from + r.dim, from + dim, to + r.dim);
  }
};

template <class V>
void rotate(const msx_rotary_desc &d, void *out, int n_threads) {
  using S = typename V::Storage;
  const bool wide = d.itype == MSX_I64;
  split(d.batch * d.tokens, n_threads, [&](int64_t first, int64_t last) {
    Turned turned;
    for (int64_t row = first; row < last; ++row) {
      const int64_t b = row / d.tokens, t = row % d.tokens;
      const int64_t p =
          d.positions != nullptr
              ? index_at(d.positions, wide, b * d.position_strides[0] + t * d.position_strides[1])
              : t + (d.starts != nullptr ? index_at(d.starts, wide, b) : 0);
      turned.at(d.rotation, static_cast<double>(p));
      for (int64_t h = 0; h < d.heads; ++h)
        turned.head<V>(d.rotation,
                       static_cast<const S *>(d.x) + b * d.x_strides[0] + t * d.x_strides[1] +
                           h * d.x_strides[2],
                       static_cast<S *>(out) + (row * d.heads + h) * d.dim, d.dim);
    }
  });
}

// The page of position j of sequence b, or -1.
int64_t page_of(const msx_paged_cache &c, int64_t b, int64_t j) {
  const int64_t page = index_at(c.pages, c.pages_itype == MSX_I64, b * c.pages_stride + j / c.page_size);
  return page >= 0 && page < c.n_pages ? page : -1;
}

template <class V>
void append(const msx_paged_append_desc &d, void *q_out, int n_threads) {
  using S = typename V::Storage;
  const msx_paged_cache &c = d.cache;
  const bool wide = d.itype == MSX_I64;
  const uint64_t capacity = static_cast<uint64_t>(c.width * c.page_size);
  split(d.batch * d.tokens, n_threads, [&](int64_t first, int64_t last) {
    Turned turned;
    for (int64_t row = first; row < last; ++row) {
      const int64_t b = row / d.tokens, t = row % d.tokens;
      const int64_t start = d.starts != nullptr ? index_at(d.starts, wide, b) : 0;
      const int64_t n = d.lengths != nullptr ? index_at(d.lengths, wide, b) : d.tokens;
      const bool live = start >= 0 && t < n;
      const uint64_t p = static_cast<uint64_t>(start) + static_cast<uint64_t>(t);
      if (live) turned.at(d.rotation, static_cast<double>(p));
      for (int64_t h = 0; h < d.heads; ++h) {
        S *to = static_cast<S *>(q_out) + (row * d.heads + h) * c.dim;
        if (live)
          turned.head<V>(d.rotation,
                         static_cast<const S *>(d.q) + b * d.q_strides[0] + t * d.q_strides[1] +
                             h * d.q_strides[2],
                         to, c.dim);
        else
          std::fill(to, to + c.dim, S{0});
      }
      if (!live || p >= capacity) continue;
      const int64_t page = page_of(c, b, static_cast<int64_t>(p)), slot = static_cast<int64_t>(p) % c.page_size;
      if (page < 0) continue;
      for (int64_t h = 0; h < c.kv_heads; ++h) {
        const S *k = static_cast<const S *>(d.k) + b * d.k_strides[0] + t * d.k_strides[1] + h * d.k_strides[2];
        const S *v = static_cast<const S *>(d.v) + b * d.v_strides[0] + t * d.v_strides[1] + h * d.v_strides[2];
        turned.head<V>(d.rotation, k,
                       static_cast<S *>(c.k) + page * c.k_strides[0] + slot * c.k_strides[1] + h * c.k_strides[2],
                       c.dim);
        std::copy(v, v + c.dim,
                  static_cast<S *>(c.v) + page * c.v_strides[0] + slot * c.v_strides[1] + h * c.v_strides[2]);
      }
    }
  });
}

template <class V>
void attend(const msx_paged_attention_desc &d, void *out, int n_threads) {
  using S = typename V::Storage;
  const msx_paged_cache &c = d.cache;
  const bool wide = d.itype == MSX_I64;
  const int64_t group = d.heads / c.kv_heads, capacity = c.width * c.page_size;
  const float scale = static_cast<float>(d.scale);
  split(d.batch * d.tokens * d.heads, n_threads, [&](int64_t first, int64_t last) {
    std::vector<const S *> k, v;
    std::vector<float> s, o;
    for (int64_t row = first; row < last; ++row) {
      const int64_t h = row % d.heads, t = row / d.heads % d.tokens, b = row / d.heads / d.tokens;
      const int64_t start = d.starts != nullptr ? index_at(d.starts, wide, b) : 0;
      const int64_t n = d.lengths != nullptr ? index_at(d.lengths, wide, b) : d.tokens;
      k.clear();
      v.clear();
      if (start >= 0 && t < n) {
        const int64_t p = std::min(start, int64_t{1} << 62) + t, hi = std::min(p, capacity - 1);
        const int64_t lo = std::min(std::max<int64_t>(p - std::min(d.window, int64_t{1} << 40) + 1, 0), capacity);
        const int64_t far = std::min(std::min(d.sinks, lo), hi + 1);
        const auto see = [&](int64_t j) {
          const int64_t page = page_of(c, b, j), slot = j % c.page_size;
          if (page < 0) return;
          k.push_back(static_cast<const S *>(c.k) + page * c.k_strides[0] + slot * c.k_strides[1] +
                      h / group * c.k_strides[2]);
          v.push_back(static_cast<const S *>(c.v) + page * c.v_strides[0] + slot * c.v_strides[1] +
                      h / group * c.v_strides[2]);
        };
        for (int64_t j = 0; j < far; ++j) see(j);
        for (int64_t j = lo; j <= hi; ++j) see(j);
      }
      const S *q = static_cast<const S *>(d.q) + b * d.q_strides[0] + t * d.q_strides[1] + h * d.q_strides[2];
      float top = -INFINITY, sum = 0.0f;
      s.assign(k.size(), 0.0f);
      for (size_t j = 0; j < k.size(); ++j) {
        for (int64_t x = 0; x < c.dim; ++x) s[j] += V::widen(q[x]) * V::widen(k[j][x]);
        s[j] *= scale;
        top = std::fmax(top, s[j]);
      }
      const float base = top == -INFINITY ? 0.0f : top;
      o.assign(static_cast<size_t>(c.dim), 0.0f);
      for (size_t j = 0; j < k.size(); ++j) {
        const float e = std::exp(s[j] - base);
        sum += e;
        for (int64_t x = 0; x < c.dim; ++x) o[x] += e * V::widen(v[j][x]);
      }
      for (int64_t x = 0; x < c.dim; ++x)
        static_cast<S *>(out)[row * c.dim + x] = V::narrow(sum == 0.0f ? 0.0f : o[x] / sum);
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

extern "C" msx_status msx_rotary_cpu(const msx_rotary_desc *desc, void *out, int n_threads) {
  clear_error();
  if (msx_status st = check_rotary("rotary", desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->tokens == 0 || desc->heads == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "rotary out is NULL.");
  return guarded("rotary", [&] {
    by_vtype(desc->vtype, [&](auto v) { rotate<decltype(v)>(*desc, out, n_threads); });
  });
}

extern "C" msx_status msx_paged_cache_append_cpu(const msx_paged_append_desc *desc, void *q_out,
                                                 int n_threads) {
  clear_error();
  const char *op = "paged_cache_append";
  if (msx_status st = check_paged_append(op, desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->tokens == 0) return MSX_OK;
  if (desc->heads > 0 && q_out == nullptr) return fail(MSX_EINVAL, "paged_cache_append q_out is NULL.");
  return guarded(op, [&] {
    by_vtype(desc->vtype, [&](auto v) { append<decltype(v)>(*desc, q_out, n_threads); });
  });
}

extern "C" msx_status msx_paged_attention_cpu(const msx_paged_attention_desc *desc, void *out,
                                              int n_threads) {
  clear_error();
  const char *op = "paged_attention";
  if (msx_status st = check_paged_attention(op, desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->tokens == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "paged_attention out is NULL.");
  return guarded(op, [&] {
    by_vtype(desc->vtype, [&](auto v) { attend<decltype(v)>(*desc, out, n_threads); });
  });
}
