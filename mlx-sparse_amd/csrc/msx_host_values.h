// msx_host_values.h - host-side value types and row loops of the window
// attention and distillation CPU paths.
#pragma once

#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <exception>
#include <thread>
#include <vector>

#include "msx_sparse.h"

namespace msx {
namespace host {

inline float bits_float(uint32_t u) {
  float f;
  memcpy(&f, &u, 4);
  return f;
}
inline uint32_t float_bits(float f) {
  uint32_t u;
  memcpy(&u, &f, 4);
  return u;
}

struct F32 {
  using Storage = float;
  static float widen(float v) { return v; }
  static float narrow(float v) { return v; }
};

struct BF16 {
  using Storage = uint16_t;
  static float widen(uint16_t v) { return bits_float(static_cast<uint32_t>(v) << 16); }
  static uint16_t narrow(float f) {  // nearest, ties to even; NaN stays NaN
    uint32_t u = float_bits(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((u >> 16) | 0x40u);
    return static_cast<uint16_t>((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
  }
};

struct F16 {
  using Storage = uint16_t;
  static float widen(uint16_t h) {
    const uint32_t sign = static_cast<uint32_t>(h & 0x8000u) << 16;
    const uint32_t e = (h >> 10) & 31u, m = h & 0x3ffu;
    if (e == 31) return bits_float(sign | 0x7f800000u | (m << 13));
    if (e != 0) return bits_float(sign | ((e + 112) << 23) | (m << 13));
    const float v = static_cast<float>(m) * 0x1p-24f;
    return sign ? -v : v;
  }
  static uint16_t narrow(float f) {  // nearest, ties to even; NaN stays NaN
    const uint32_t u = float_bits(f), sign = (u >> 16) & 0x8000u, a = u & 0x7fffffffu;
    if (a > 0x7f800000u) return static_cast<uint16_t>(sign | 0x7e00u);
    if (a >= 0x477ff000u) return static_cast<uint16_t>(sign | 0x7c00u);  // rounds past 65504
    if (a < 0x38800000u) {  // subnormal: the float addition rounds to a multiple of 2^-24
      const float v = bits_float(a) + 0.5f;
      return static_cast<uint16_t>(sign | (float_bits(v) - 0x3f000000u));
    }
    const uint32_t r = a + 0xfffu + ((a >> 13) & 1u);
    return static_cast<uint16_t>(sign | ((r - 0x38000000u) >> 13));
  }
};

// fn(first, last) over [0, n) in contiguous parts on `n_threads` threads.
// Exceptions of a part, or of starting a thread, reach the caller.
template <class Fn>
void split(int64_t n, int n_threads, Fn &&fn) {
  const int64_t parts = std::min<int64_t>(n, n_threads > 0 ? n_threads : msx_cpu_worker_count());
  if (parts <= 1) {
    if (n > 0) fn(int64_t{0}, n);
    return;
  }
  std::vector<std::exception_ptr> failed(static_cast<size_t>(parts));
  std::vector<std::thread> threads;
  threads.reserve(static_cast<size_t>(parts));
  const auto part = [&](int64_t i) {
    try {
      fn(i * n / parts, (i + 1) * n / parts);
    } catch (...) {
      failed[static_cast<size_t>(i)] = std::current_exception();
    }
  };
  try {
    for (int64_t i = 1; i < parts; ++i) threads.emplace_back(part, i);
  } catch (...) {
    for (auto &t : threads) t.join();
    throw;
  }
  part(0);
  for (auto &t : threads) t.join();
  for (auto &e : failed)
    if (e) std::rethrow_exception(e);
}

template <class Fn>
void by_vtype(int vt, Fn &&fn) {
  if (vt == MSX_F32) fn(F32{});
  else if (vt == MSX_F16) fn(F16{});
  else fn(BF16{});
}

inline int64_t index_at(const void *p, bool i64, int64_t i) {
  return i64 ? static_cast<const int64_t *>(p)[i] : static_cast<const int32_t *>(p)[i];
}

}  // namespace host
}  // namespace msx
