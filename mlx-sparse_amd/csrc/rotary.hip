// rotary.hip - rotary positions: of queries and keys as they are, and of those
// on their way into a paged cache.
//
// Pair i of a head is turned by turns[i] p whole turns at position p.  Only the
// fraction of a turn matters, and a position of a million leaves float32 a
// thirtieth of a turn of it: product and fraction are 64-bit, the eighth of a turn
// that is left goes through the series of sine and cosine.  A thread has
// the pairs of one place of the head and takes the heads of a token in turn, so
// that their angles are worked out once.
//
// Bound by memory, calls of a few tokens by the launch.  16,384 tokens of 40 heads of 128,
// bfloat16: 59 us, 5.7 TB/s read and written, more than a copy; 129 of 10 of 80, float32: 3.4 us.
// Appended: 64 tokens' 48 heads 4.5 us; 5 prompts of up to 2,049 tokens, 32 heads, float16, 17 us
// (4.0 TB/s).  Heads of which a half (interleaved, the rotated part) is no multiple of sixteen
// bytes go a value a thread: 8,192 tokens of 20 heads of 128, 62 values rotated, 30 us in bfloat16 and 29.5
// in float32 where whole heads take 14.8 and 26; 4,096 tokens of 16 + 4 appended 30 where they take 11 and 17.5.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "msx_device.h"
#include "msx_internal.h"
#include "msx_paged.h"
#include "msx_paged_check.h"
#include "msx_window_mfma.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kThreads = 256;

// Cosine and sine of t turns, in T (float: to 2^-23; double: to 2^-37, for
// results that are float32).
template <class T>
__device__ __forceinline__ void turn(double t, float magnitude, float &cosine, float &sine) {
  t -= rint(t);
  const double quarter = 4.0 * t, whole = rint(quarter);
  const T x = static_cast<T>(quarter - whole) * static_cast<T>(1.57079632679489661923);
  const T y = x * x;
  // Taylor's series up to x^11 / 11! and x^12 / 12!, |x| <= pi / 4
  T s = T(-1.0 / 39916800);
  s = s * y + T(1.0 / 362880);
  s = s * y + T(-1.0 / 5040);
  s = s * y + T(1.0 / 120);
  s = s * y + T(-1.0 / 6);
  s = s * y * x + x;
  T c = T(1.0 / 479001600);
  c = c * y + T(-1.0 / 3628800);
  c = c * y + T(1.0 / 40320);
  c = c * y + T(-1.0 / 720);
  c = c * y + T(1.0 / 24);
  c = c * y + T(-0.5);
  c = c * y + T(1.0);
  const int n = static_cast<int>(whole);
  const T a = n & 1 ? s : c, b = n & 1 ? c : s;
  cosine = static_cast<float>((n + 1) & 2 ? -a * T(magnitude) : a * T(magnitude));
  sine = static_cast<float>(n & 2 ? -b * T(magnitude) : b * T(magnitude));
}

// E adjacent values, as they lie in memory; kPast: past the caches.
template <class V, int E>
struct Values {
  using S = typename V::Storage;
  using Raw = std::conditional_t<E == 1, S, v4u>;
  template <bool kPast>
  __device__ static __forceinline__ Raw load(const S *p) {
    if constexpr (kPast) return __builtin_nontemporal_load(reinterpret_cast<const Raw *>(p));
    return *reinterpret_cast<const Raw *>(p);
  }
  template <bool kPast>
  __device__ static __forceinline__ void store(S *p, Raw r) {
    if constexpr (kPast)
      __builtin_nontemporal_store(r, reinterpret_cast<Raw *>(p));
    else
      *reinterpret_cast<Raw *>(p) = r;
  }
  __device__ static __forceinline__ void widen(Raw r, float (&x)[E]) {
    if constexpr (E == 1) {
      x[0] = V::widen(r);
    } else if constexpr (E == 4) {
      const v4f f = __builtin_bit_cast(v4f, r);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = f[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t pair = r[j];
        x[2 * j] = V::widen(static_cast<uint16_t>(pair));
        x[2 * j + 1] = V::widen(static_cast<uint16_t>(pair >> 16));
      }
    }
  }
  __device__ static __forceinline__ Raw narrow(const float (&x)[E]) {
    if constexpr (E == 1) {
      return V::narrow(x[0]);
    } else if constexpr (E == 4) {
      return __builtin_bit_cast(Raw, (v4f{x[0], x[1], x[2], x[3]}));
    } else {
      Raw r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = Mfma<V>::pack(x[2 * j], x[2 * j + 1]);
      return r;
    }
  }
};

// How a head is cut into units, a thread each.  Halves: E values and the E that
// they are paired with; interleaved: E values that are pairs (with E = 1 the two of
// one).  Units from `rotated` on are values that are copied.
template <class V, int E, bool kInterleaved>
struct Unit {
  static constexpr int kVectors = kInterleaved && E > 1 ? 1 : 2;  // of a rotated unit
  static constexpr int kPairs = kVectors * E / 2;
  int32_t at[2];  // places of its vectors; of a copied unit both the same
  bool rotated;
  float cosine[kPairs], sine[kPairs];

  __host__ __device__ static inline int32_t rotated_units(int32_t r) { return r / (kVectors * E); }
  __host__ __device__ static inline int32_t units(int32_t r, int32_t dim) {
    return rotated_units(r) + (dim - r) / E;
  }
  __device__ __forceinline__ Unit(int32_t u, int32_t r) {
    rotated = u < rotated_units(r);
    at[0] = rotated ? (kInterleaved ? u * kVectors * E : u * E) : r + (u - rotated_units(r)) * E;
    at[1] = rotated && kVectors == 2 ? at[0] + (kInterleaved ? E : r / 2) : at[0];
  }
  __device__ __forceinline__ void angles(const double *turns, double position, float magnitude,
                                         float sign) {
    if (!rotated) return;
    const int32_t first = kInterleaved ? at[0] / 2 : at[0];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      // 16-bit results: float32's 2^-23 of a cosine is nothing beside their rounding
      using T = std::conditional_t<sizeof(typename V::Storage) == 4, double, float>;
      turn<T>(turns[first + i] * position, magnitude, cosine[i], sine[i]);
      sine[i] *= sign;
    }
  }
  using Raw = typename Values<V, E>::Raw;
  __device__ __forceinline__ void apply(Raw (&raw)[kVectors]) const {
    if constexpr (kVectors == 2) {
      float a[E], b[E], x[E], y[E];
      Values<V, E>::widen(raw[0], a);
      Values<V, E>::widen(raw[1], b);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        x[i] = a[i] * cosine[i] - b[i] * sine[i];
        y[i] = a[i] * sine[i] + b[i] * cosine[i];
      }
      raw[0] = Values<V, E>::narrow(x);
      raw[1] = Values<V, E>::narrow(y);
    } else {
      float a[E], x[E];
      Values<V, E>::widen(raw[0], a);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        x[2 * i] = a[2 * i] * cosine[i] - a[2 * i + 1] * sine[i];
        x[2 * i + 1] = a[2 * i] * sine[i] + a[2 * i + 1] * cosine[i];
      }
      raw[0] = Values<V, E>::narrow(x);
    }
  }
};

struct Turning {
  int32_t r;  // values of a head that are rotated
  float magnitude, sign;
  const double *turns;
};

// Where a token's heads come from and go to: one tensor to another.
template <class S>
struct Whole {
  int32_t tokens, heads, dim, index64;
  const S *x;
  int64_t xs[3];
  const void *starts, *positions;
  int64_t ps[2];
  S *out;

  struct Token {
    const S *from;
    S *to;
    double position;
  };
  struct Place {
    const S *from;
    S *to;
    bool rotated, zero;
  };
  __device__ __forceinline__ Token token(int64_t row, int64_t b, int32_t t) const {
    int64_t p;
    if (positions != nullptr)
      p = count_of(positions, index64, b * ps[0] + t * ps[1], 0);
    else
      p = count_of(starts, index64, b, 0) + t;
    return {x + b * xs[0] + t * xs[1], out + row * heads * dim, static_cast<double>(p)};
  }
  __device__ __forceinline__ Place place(const Token &k, int32_t h) const {
    return {k.from + h * xs[2], k.to + h * dim, true, false};
  }
};

// Queries to a tensor, keys and values to their pages.
template <class S>
struct Append {
  int32_t tokens, q_heads, kv_heads, dim, index64;
  const S *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];
  const void *starts, *lengths;
  PageTable table;
  S *cache_k, *cache_v, *q_out;
  int64_t cks[3], cvs[3];

  struct Token {
    const S *q, *k, *v;
    S *q_to, *k_to, *v_to;  // k_to null: no place in the cache
    double position;
    bool live;
  };
  struct Place {
    const S *from;
    S *to;
    bool rotated, zero;
  };
  __device__ __forceinline__ Token token(int64_t row, int64_t b, int32_t t) const {
    const int64_t start = count_of(starts, index64, b, 0);
    const int64_t n = count_of(lengths, index64, b, tokens);
    Token k{};
    k.live = start >= 0 && t < n;
    const uint64_t p = static_cast<uint64_t>(start) + static_cast<uint64_t>(t);
    k.position = static_cast<double>(static_cast<int64_t>(p));
    k.q = q + b * qs[0] + t * qs[1];
    k.q_to = q_out + row * q_heads * dim;
    if (k.live && p < static_cast<uint64_t>(table.capacity)) {
      const int32_t j = static_cast<int32_t>(p), page = table.page(b, j), slot = table.slot(j);
      if (page >= 0) {
        k.k = this->k + b * ks[0] + t * ks[1];
        k.v = v + b * vs[0] + t * vs[1];
        k.k_to = cache_k + page * cks[0] + slot * cks[1];
        k.v_to = cache_v + page * cvs[0] + slot * cvs[1];
      }
    }
    return k;
  }
  // Heads are numbered through: queries, keys, values.
  __device__ __forceinline__ Place place(const Token &k, int32_t h) const {
    if (h < q_heads) return {k.q + h * qs[2], k.q_to + h * dim, true, !k.live};
    if (k.k_to == nullptr) return {nullptr, nullptr, false, false};
    h -= q_heads;
    if (h < kv_heads) return {k.k + h * ks[2], k.k_to + h * cks[2], true, false};
    h -= kv_heads;
    return {k.v + h * vs[2], k.v_to + h * cvs[2], false, false};
  }
};

struct Split {
  int64_t rows;       // tokens of the batch
  int32_t heads;      // of a token, together
  int32_t units;      // of a head
  int32_t side;       // heads that run side by side
  int32_t per_block;  // tokens
  int32_t parts;      // of a token's heads, a workgroup each
};

template <class V, int E, bool kInterleaved, bool kPast, class Rows>
__global__ __launch_bounds__(kThreads) void rotate_rows(Rows rows, Turning how, Split s, int64_t first) {
  using U = Unit<V, E, kInterleaved>;
  using Raw = typename U::Raw;
  const int32_t u = threadIdx.x % s.units, g = threadIdx.x / s.units;
  const int32_t part = blockIdx.x % s.parts;
  const int64_t row = first + static_cast<int64_t>(blockIdx.x / s.parts) * s.per_block + g / s.side;
  if (g >= s.per_block * s.side || row >= s.rows) return;
  const int64_t b = row / rows.tokens;
  const auto token = rows.token(row, b, static_cast<int32_t>(row - b * rows.tokens));
  U unit(u, how.r);
  unit.angles(how.turns, token.position, how.magnitude, how.sign);
  constexpr int kAhead = 4;  // heads whose loads are in flight
  const int32_t step = s.side * s.parts;
  for (int32_t h0 = part * s.side + g % s.side; h0 < s.heads; h0 += kAhead * step) {
    Raw raw[kAhead][U::kVectors];
    decltype(rows.place(token, 0)) place[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      place[j] = {nullptr, nullptr, false, false};
      if (h0 + j * step < s.heads) place[j] = rows.place(token, h0 + j * step);
      if (place[j].to == nullptr) continue;
#pragma unroll
      for (int k = 0; k < U::kVectors; ++k) {
        raw[j][k] = Raw{};
        if (!place[j].zero) raw[j][k] = Values<V, E>::template load<kPast>(place[j].from + unit.at[k]);
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (place[j].to == nullptr) continue;
      if (unit.rotated && place[j].rotated && !place[j].zero) unit.apply(raw[j]);
#pragma unroll
      for (int k = 0; k < U::kVectors; ++k) Values<V, E>::template store<kPast>(place[j].to + unit.at[k], raw[j][k]);
    }
  }
}

// More values, read and written, than the Infinity Cache (256 MB) holds until the next reader go past the
// caches, in us: of 40 heads of 128, bfloat16, 16,384 tokens (336 MB) 65 to 59, 24,000 91 to 82; 8,192 of 20
// (84 MB) 14.8 and 16.4, 13,300 of 40 (272 MB) 44 and 47, 14,200 (291 MB) 47 and 50, in float32 55 and 53.
constexpr int64_t kCached = int64_t{288} << 20;

template <class V, int E, bool kInterleaved, class Rows>
msx_status launch(const Rows &rows, const Turning &how, int64_t tokens, int32_t heads, int32_t dim,
                  const char *op, hipStream_t stream) {
  Split s;
  s.rows = tokens;
  s.heads = heads;
  s.units = Unit<V, E, kInterleaved>::units(how.r, dim);
  const int32_t groups = kThreads / s.units;
  // A thread takes four of a token's heads, its loads in flight together and their angles
  // worked out once, where that leaves a workgroup a CU (bf16 appends of 512 tokens' 32 + 16
  // heads of 128, interleaved: 7.0 us, a head a thread 7.5; of 1,024 7.3 and 11.3; of 8,192
  // 31 and 63).  Fewer tokens are spread over as many workgroups as their heads give, for
  // which both ways take less than the call itself.
  const bool many = tokens * heads * s.units >= int64_t{4} * 256 * kThreads;
  s.side = std::min(many ? (heads + 3) / 4 : heads, groups);
  s.per_block = groups / s.side;
  s.parts = many ? 1 : (heads + s.side - 1) / s.side;
  const int64_t most = max_blocks(kThreads) / s.parts * s.per_block;
  for (int64_t first = 0; first < tokens; first += most) {
    const int64_t here = std::min(tokens - first, most);
    const auto blocks = static_cast<unsigned>((here + s.per_block - 1) / s.per_block * s.parts);
    if constexpr (E > 1) {
      if (2 * tokens * heads * dim * static_cast<int64_t>(sizeof(typename V::Storage)) > kCached) {
        rotate_rows<V, E, kInterleaved, true><<<blocks, kThreads, 0, stream>>>(rows, how, s, first);
        continue;
      }
    }
    rotate_rows<V, E, kInterleaved, false><<<blocks, kThreads, 0, stream>>>(rows, how, s, first);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, op);
}

// Whether rows of this layout start at sixteen bytes.
bool aligned(size_t size, const void *p, const int64_t *strides, const int64_t *shape, int n) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < n; ++i)
    ok = ok && (shape[i] < 2 || strides[i] * static_cast<int64_t>(size) % 16 == 0);
  return ok;
}

template <class V, class Rows>
msx_status by_layout(const Rows &rows, const msx_rotation &r, int64_t tokens, int64_t heads,
                     int64_t dim, bool wide, const char *op, hipStream_t stream) {
  constexpr int E = 16 / sizeof(typename V::Storage);
  const Turning how{static_cast<int32_t>(r.dim), static_cast<float>(r.magnitude),
                    r.inverse ? -1.0f : 1.0f, r.turns};
  const auto h = static_cast<int32_t>(heads), d = static_cast<int32_t>(dim);
  // sixteen bytes a load where each lies within the rotated values, one half of them or
  // the rest
  wide = wide && dim % E == 0 && r.dim % (r.interleaved ? E : 2 * E) == 0;
  if (r.interleaved)
    return wide ? launch<V, E, true>(rows, how, tokens, h, d, op, stream)
                : launch<V, 1, true>(rows, how, tokens, h, d, op, stream);
  return wide ? launch<V, E, false>(rows, how, tokens, h, d, op, stream)
              : launch<V, 1, false>(rows, how, tokens, h, d, op, stream);
}

template <class Fn>
msx_status by_vtype(int vt, Fn &&fn) {
  switch (vt) {
  case MSX_F32: return fn(F32{});
  case MSX_F16: return fn(F16{});
  default: return fn(BF16{});
  }
}

}  // namespace
}  // namespace msx

using namespace msx;

extern "C" msx_status msx_rotary(const msx_rotary_desc *desc, void *out, void *stream) {
  clear_error();
  const char *op = "rotary";
  if (msx_status st = check_rotary(op, desc); st != MSX_OK) return st;
  const msx_rotary_desc &d = *desc;
  if (d.batch == 0 || d.tokens == 0 || d.heads == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "rotary out is NULL.");
  return by_vtype(d.vtype, [&](auto v) {
    using V = decltype(v);
    using S = typename V::Storage;
    Whole<S> w{};
    w.tokens = static_cast<int32_t>(d.tokens);
    w.heads = static_cast<int32_t>(d.heads);
    w.dim = static_cast<int32_t>(d.dim);
    w.index64 = d.itype == MSX_I64;
    w.x = static_cast<const S *>(d.x);
    std::copy(d.x_strides, d.x_strides + 3, w.xs);
    w.starts = d.starts;
    w.positions = d.positions;
    std::copy(d.position_strides, d.position_strides + 2, w.ps);
    w.out = static_cast<S *>(out);
    const int64_t shape[3] = {d.batch, d.tokens, d.heads};
    const bool wide = aligned(sizeof(S), d.x, d.x_strides, shape, 3) &&
                      reinterpret_cast<uintptr_t>(out) % 16 == 0;
    return by_layout<V>(w, d.rotation, d.batch * d.tokens, d.heads, d.dim, wide, op,
                        static_cast<hipStream_t>(stream));
  });
}

extern "C" msx_status msx_paged_cache_append(const msx_paged_append_desc *desc, void *q_out,
                                             void *stream) {
  clear_error();
  const char *op = "paged_cache_append";
  if (msx_status st = check_paged_append(op, desc); st != MSX_OK) return st;
  const msx_paged_append_desc &d = *desc;
  if (d.batch == 0 || d.tokens == 0) return MSX_OK;
  if (d.heads > 0 && q_out == nullptr) return fail(MSX_EINVAL, "paged_cache_append q_out is NULL.");
  return by_vtype(d.vtype, [&](auto v) {
    using V = decltype(v);
    using S = typename V::Storage;
    const msx_paged_cache &c = d.cache;
    Append<S> a{};
    a.tokens = static_cast<int32_t>(d.tokens);
    a.q_heads = static_cast<int32_t>(d.heads);
    a.kv_heads = static_cast<int32_t>(c.kv_heads);
    a.dim = static_cast<int32_t>(c.dim);
    a.index64 = d.itype == MSX_I64;
    a.q = static_cast<const S *>(d.q);
    a.k = static_cast<const S *>(d.k);
    a.v = static_cast<const S *>(d.v);
    std::copy(d.q_strides, d.q_strides + 3, a.qs);
    std::copy(d.k_strides, d.k_strides + 3, a.ks);
    std::copy(d.v_strides, d.v_strides + 3, a.vs);
    a.starts = d.starts;
    a.lengths = d.lengths;
    a.table = table_of(c);
    a.cache_k = static_cast<S *>(c.k);
    a.cache_v = static_cast<S *>(c.v);
    a.q_out = static_cast<S *>(q_out);
    std::copy(c.k_strides, c.k_strides + 3, a.cks);
    std::copy(c.v_strides, c.v_strides + 3, a.cvs);
    const int64_t given[3] = {d.batch, d.tokens, c.kv_heads}, q_shape[3] = {d.batch, d.tokens, d.heads},
                  held[3] = {c.n_pages, c.page_size, c.kv_heads};
    const bool wide = aligned(sizeof(S), d.k, d.k_strides, given, 3) &&
                      aligned(sizeof(S), d.v, d.v_strides, given, 3) &&
                      (d.heads == 0 || (aligned(sizeof(S), d.q, d.q_strides, q_shape, 3) &&
                                        reinterpret_cast<uintptr_t>(q_out) % 16 == 0)) &&
                      aligned(sizeof(S), c.k, c.k_strides, held, 3) &&
                      aligned(sizeof(S), c.v, c.v_strides, held, 3);
    return by_layout<V>(a, d.rotation, d.batch * d.tokens, d.heads + 2 * c.kv_heads, c.dim, wide, op,
                        static_cast<hipStream_t>(stream));
  });
}
