// msx_paged.h - device-side view of paged caches: where a position lies, and
// which positions a query sees.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "msx_device.h"
#include "msx_sparse.h"
#include "msx_window.h"

namespace msx {

// n / d for n, d < 2^31 by one high product: with s = ceil(log2 d) and m =
// floor(2^32 (2^s - d) / d) + 1, n / d = (high(m n) + n) >> s (the sum stays
// below 2^32).
struct FastDiv {
  uint32_t m, s;
  static FastDiv by(uint32_t d) {
    FastDiv f{0, 0};
    while ((uint64_t{1} << f.s) < d) ++f.s;
    f.m = static_cast<uint32_t>((((uint64_t{1} << f.s) - d) << 32) / d + 1);
    return f;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return (__umulhi(m, n) + n) >> s;
  }
};

// One count of a batch; `none` where the caller has no array.
__device__ inline int64_t count_of(const void *counts, int32_t wide, int64_t b, int64_t none) {
  if (counts == nullptr) return none;
  return wide ? static_cast<const int64_t *>(counts)[b] : static_cast<const int32_t *>(counts)[b];
}

// The caches and the table of their pages, as the kernels take them.
struct PageTable {
  const void *pages;
  int64_t stride;
  int32_t n_pages;
  int32_t wide;  // numbers of 64 bits
  int32_t size;  // tokens a page
  int32_t capacity;
  FastDiv by_size;

  // A page's number as it is loaded, to be looked at where it is wanted: looked at
  // once it is asked for, each would be waited for.
  struct Number {
    int32_t low, high;
  };
  __device__ static __forceinline__ Number none() { return {-1, 0}; }
  // of position j of row b, 0 <= j < capacity
  __device__ __forceinline__ Number number(int64_t b, int32_t j) const {
    const int64_t at = b * stride + static_cast<int32_t>(by_size(j));
    if (!wide) return {static_cast<const int32_t *>(pages)[at], 0};
    const int2 both = static_cast<const int2 *>(pages)[at];
    return {both.x, both.y};
  }
  // The page, or -1 for one that is not there.
  __device__ __forceinline__ int32_t checked(Number n) const {
    return ((static_cast<uint32_t>(n.low) < static_cast<uint32_t>(n_pages)) & (n.high == 0)) ? n.low : -1;
  }
  __device__ __forceinline__ int32_t page(int64_t b, int32_t j) const { return checked(number(b, j)); }
  __device__ __forceinline__ int32_t slot(int32_t j) const {
    return j - static_cast<int32_t>(by_size(j)) * size;
  }
};

inline PageTable table_of(const msx_paged_cache &c) {
  PageTable t;
  t.pages = c.pages;
  t.stride = c.pages_stride;
  t.n_pages = static_cast<int32_t>(c.n_pages);
  t.wide = c.pages_itype == MSX_I64;
  t.size = static_cast<int32_t>(c.page_size);
  t.capacity = static_cast<int32_t>(c.width * c.page_size);
  t.by_size = FastDiv::by(static_cast<uint32_t>(c.page_size));
  return t;
}

// The keys that a query sees: [0, far) and [lo, hi], far <= lo; of both those from
// `from` on, where those before are another kernel's.
struct Keys {
  int32_t far, lo, hi, from;
  __device__ __forceinline__ int32_t count() const { return far + (hi < lo ? 0 : hi - lo + 1); }
  __device__ __forceinline__ int32_t key(int32_t c) const { return c < far ? c : lo + c - far; }
  __device__ __forceinline__ bool sees(int32_t j) const {
    return (j >= from) & (j <= hi) & ((j >= lo) | (j < far));
  }
};

struct PagedArgs {
  int64_t batch;
  int32_t tokens, heads, kv_heads, group, dim;
  int64_t window;
  int32_t sinks;  // at most the table's capacity
  float scale;    // scale * log2(e): scores are kept in base 2
  const void *starts, *lengths;
  int32_t counts64;
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];  // caches: page, slot, head
  PageTable table;

  __device__ __forceinline__ int64_t start(int64_t b) const { return count_of(starts, counts64, b, 0); }
  // Queries of sequence b that are there.
  __device__ __forceinline__ int32_t length(int64_t b) const {
    if (start(b) < 0) return 0;
    const int64_t n = count_of(lengths, counts64, b, tokens);
    return static_cast<int32_t>(n < 0 ? 0 : n > tokens ? tokens : n);
  }
  // What queries `first` to `last` of a sequence that starts at `start` see
  // together (of one: what it sees).  A position past 2^62 is one that far: nothing
  // is cached there.
  __device__ __forceinline__ Keys keys(int64_t start, int32_t first, int32_t last) const {
    const int64_t from = min(start, int64_t{1} << 62) + first, to = min(start, int64_t{1} << 62) + last;
    const int64_t cap = table.capacity;
    Keys k;
    k.from = 0;
    k.hi = static_cast<int32_t>(min(to, cap - 1));
    k.lo = static_cast<int32_t>(min(max(from - window + 1, int64_t{0}), cap));
    k.far = min(min(sinks, k.lo), k.hi + 1);
    return k;
  }
};


}  // namespace msx
