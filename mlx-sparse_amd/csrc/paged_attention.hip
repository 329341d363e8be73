// paged_attention.hip - attention over paged caches: the entry points, and the row
// kernel that takes every type, head dimension, alignment and page size.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>

#include "msx_device.h"
#include "msx_internal.h"
#include "msx_paged.h"
#include "msx_paged_check.h"
#include "msx_paged_row.h"
#include "msx_paged_tiles.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

constexpr int kRowWaves = 4;
// One wave a (sequence, query, head).
template <class V>
__global__ __launch_bounds__(kRowWaves * kWave) void paged_rows(PagedArgs a, int64_t first, int64_t rows,
                                                                typename V::Storage *out) {
  __shared__ float q_lds[kRowWaves][kWindowMaxDim];
  const int wave = threadIdx.x / kWave;
  const int64_t row = first + static_cast<int64_t>(blockIdx.x) * kRowWaves + wave;
  if (row >= rows) return;  // whole waves leave; there is no barrier below
  paged_row<V>(a, row / a.heads / a.tokens, static_cast<int32_t>(row / a.heads % a.tokens),
               static_cast<int32_t>(row % a.heads), q_lds[wave], out);
}

PagedArgs args_of(const msx_paged_attention_desc &d) {
  PagedArgs a{};
  a.batch = d.batch;
  a.tokens = static_cast<int32_t>(d.tokens);
  a.heads = static_cast<int32_t>(d.heads);
  a.kv_heads = static_cast<int32_t>(d.cache.kv_heads);
  a.group = a.heads / a.kv_heads;
  a.dim = static_cast<int32_t>(d.cache.dim);
  a.table = table_of(d.cache);
  a.window = std::min(d.window, int64_t{1} << 40);  // no sequence is as long
  a.sinks = static_cast<int32_t>(std::min<int64_t>(d.sinks, a.table.capacity));
  a.scale = static_cast<float>(d.scale * 1.44269504088896340736);
  a.starts = d.starts;
  a.lengths = d.lengths;
  a.counts64 = d.itype == MSX_I64;
  a.q = d.q;
  a.k = d.cache.k;
  a.v = d.cache.v;
  std::copy(d.q_strides, d.q_strides + 3, a.qs);
  std::copy(d.cache.k_strides, d.cache.k_strides + 3, a.ks);
  std::copy(d.cache.v_strides, d.cache.v_strides + 3, a.vs);
  return a;
}

// Whether the tiles' kernels can read the operands: sixteen-byte rows at sixteen-byte
// strides, and queries that share a kv head that 32 bits count.
bool takes_tiles(const msx_paged_attention_desc &d) {
  const auto size = static_cast<int64_t>(value_bytes(static_cast<msx_vtype>(d.vtype)));
  const auto aligned = [&](const void *p, const int64_t *strides) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && strides[0] * size % 16 == 0 &&
           strides[1] * size % 16 == 0 && strides[2] * size % 16 == 0;
  };
  return d.cache.dim * size % 16 == 0 &&
         d.tokens * (d.heads / d.cache.kv_heads) <= kWindowIntMax - 256 && aligned(d.q, d.q_strides) &&
         aligned(d.cache.k, d.cache.k_strides) && aligned(d.cache.v, d.cache.v_strides);
}

template <class Fn>
msx_status by_vtype(int vt, Fn &&fn) {
  switch (vt) {
  case MSX_F32: return fn(F32{});
  case MSX_F16: return fn(F16{});
  default: return fn(BF16{});
  }
}

enum class Route { kRows, kStep, kTiles, kShared };

// Rows that share a kv head: up to so many a sequence go through paged_step, a read of
// the keys for each sixteen of them; more in 16 bits through paged_tiles, where the second read
// would be long.  Measured, by tiles and by steps, in us, heads of 128:
//   bfloat16   5 tokens of 16 heads on 4: 32 of 4,000 keys 27.7 32.9; 8 of 32 on 8: 1 of 30,000 37.9 55.1,
//              17 of 3 on 3: 8 of 2,000 21.7 17.7
//   float32    5 of 16 on 4: 32 of 4,000 61.6 48.1; 8 of 32 on 8: 1 of 30,000 155 92
constexpr int64_t kFewRows = 32;
constexpr int64_t kLongRead = int64_t{48} << 20;  // bytes that the table has room for

// Whether the shared pages are worth kernels of their own.  Reading them for each sequence takes
// their bytes at 5 TB/s; once for all of them, the products of 128 queries a tile at what
// paged_tiles reaches at such sizes, or the bytes once, some 8 us for more workgroups' starts
// and a second set of parts to join, and the sequences' own keys half the chip.  Measured,
// without and with, in us, one token a sequence:
//   32 heads of 128 on 8, bfloat16   4 sequences of 1,024 shared keys 15.2 18.0, 4,096 22.4 17.9;
//                                    64 of 64 12.9 31.6, 256 17.2 33.9, 1,024 42.5 38.9, 16,384 558 53
//   8 heads of 64 on 2, float16      64 of 256 8.6 17.8, 4,096 28.7 21.9
//   16 heads of 128, float32         2 of 16,384 98 166, 8 286 169; 64 of 256 60.5 70.4, 1,024 140 66
bool shares(const msx_paged_attention_desc &d, int64_t rows) {
  const msx_paged_cache &c = d.cache;
  // (with a window narrower than the table few sequences see much of what they share)
  if (d.shared_pages == 0 || d.batch < 2 || d.window < c.width * c.page_size ||
      d.batch * rows > kWindowIntMax - kTileRows)
    return false;
  const double keys = static_cast<double>(d.shared_pages * c.page_size * c.kv_heads);
  const double size = static_cast<double>(value_bytes(static_cast<msx_vtype>(d.vtype)));
  const double once = keys * c.dim * 2 * size / 5e6, rate = d.vtype == MSX_F32 ? 80e6 : 500e6;
  const double products = static_cast<double>((d.batch * rows + kTileRows - 1) / kTileRows) * kTileRows * keys *
                          c.dim * 4 / rate;
  const double own = 0.01 * static_cast<double>(d.batch * c.kv_heads * ((rows + kStepRows - 1) / kStepRows));
  return std::max(once, products) + 8 + own < once * static_cast<double>(d.batch);
}

// The most keys that a query of this call may see.
int64_t held_keys(const msx_paged_attention_desc &d) {
  const int64_t wide = int64_t{1} << 40;  // no sequence is as long
  return std::min(d.cache.width * d.cache.page_size,
                  std::min(d.window, wide) + std::min(d.sinks, wide) + d.tokens);
}

// The bytes of as many keys and values, of one sequence and kv head.
int64_t held_bytes(const msx_paged_attention_desc &d) {
  return 2 * held_keys(d) * d.cache.dim * static_cast<int64_t>(value_bytes(static_cast<msx_vtype>(d.vtype)));
}

// Keys that are read once go past the caches where there may be more of them than the Infinity Cache holds
// (256 MB) from one call to the next: 64 sequences of up to 16,384 tokens, 32 heads of 128 on 8, bfloat16, 125 us
// to 113; one of 131,072 114.5 to 107; 300 of 2,048 439 to 403; 60 of 1,500 in float32 150 to 136.  What is there
// is read faster from it: 262 MB of 32 of 4,000 keys, 52 us so, 58 past it.
constexpr int64_t kCached = int64_t{320} << 20;

Route route_of(const msx_paged_attention_desc &d) {
  if (!takes_tiles(d)) return Route::kRows;
  const int64_t rows = d.tokens * (d.heads / d.cache.kv_heads);
  const bool wide = (d.cache.dim > 128 && d.vtype == MSX_F32) ||  // (a masked score is minus infinity times the scale)
                    !(std::fabs(static_cast<float>(d.scale)) >= std::numeric_limits<float>::min());
  if (wide) return Route::kStep;
  if (rows > kFewRows) return Route::kTiles;
  const int64_t held = held_keys(d), read = d.batch * d.cache.kv_heads * held * d.cache.dim * 4;
  if (rows > kStepRows && d.vtype != MSX_F32 && held > 512 && read >= kLongRead) return Route::kTiles;
  return shares(d, rows) ? Route::kShared : Route::kStep;
}

// Whether tiles of queries are as few as the kernels count.
bool countable(const msx_paged_attention_desc &d) {
  const int64_t rows = d.tokens * (d.heads / d.cache.kv_heads);
  return !takes_tiles(d) || d.batch * ((rows + kStepRows - 1) / kStepRows) <= kWindowIntMax;
}

// What a call's kernels are given, and where in its scratch their parts lie.
struct Plan {
  Route route;
  StepGrid step{}, tiles{};
  TileParts step_to{}, tiles_to{};
  size_t bytes = 0;

  Plan(const msx_paged_attention_desc &d, const PagedArgs &a, void *out, void *scratch)
      : route(route_of(d)) {
    const int64_t rows = static_cast<int64_t>(a.tokens) * a.group, all = a.batch * a.tokens * a.heads;
    char *base = static_cast<char *>(scratch);
    const auto take = [&](int64_t each, int64_t count) {
      char *p = base + bytes;
      bytes += (static_cast<size_t>(each * count) + 255) / 256 * 256;
      return p;
    };
    const int64_t part = sizeof(float) * part_stride(a.dim);
    const auto parts_of = [&](const StepGrid &g, int64_t entries, int32_t tile_rows) {
      TileParts to{};
      to.out = out;
      if (g.whole) return to;
      to.spans = reinterpret_cast<StepSpan *>(take(sizeof(StepSpan), entries * a.kv_heads));
      to.parts = reinterpret_cast<float *>(take(part, 2 * static_cast<int64_t>(g.groups) * tile_rows));
      if (route == Route::kShared) to.whole = reinterpret_cast<float *>(take(part, all));
      return to;
    };
    // as many workgroups as run at once: registers allow two a CU, of wide heads one
    if (route == Route::kStep || route == Route::kShared) {
      step.tiles = static_cast<int32_t>((rows + kStepRows - 1) / kStepRows);
      step.groups = a.dim > 128 || route == Route::kShared ? 256 : 512;
      step.waves = kStepWaves;
      if (route == Route::kStep) whole(d, a);
      step.past = route == Route::kStep && !step.whole && step.tiles == 1 &&
                  held_bytes(d) * d.batch * d.cache.kv_heads > kCached;
      step.from = route == Route::kShared ? static_cast<int32_t>(d.shared_pages * d.cache.page_size) : 0;
      step_to = parts_of(step, a.batch * step.tiles, kStepRows);
    }
    if (route == Route::kTiles || route == Route::kShared) {
      const int64_t together = route == Route::kShared ? a.batch * rows : rows;
      tiles.tiles = static_cast<int32_t>((together + kTileRows - 1) / kTileRows);
      tiles.groups = route == Route::kShared || a.dim * value_bytes(static_cast<msx_vtype>(d.vtype)) > 256 ? 256 : 512;
      tiles.from = step.from;
      if (route == Route::kTiles) whole_tiles(d, a);
      tiles_to = parts_of(tiles, route == Route::kShared ? tiles.tiles : a.batch * tiles.tiles, kTileRows);
    }
  }
  // Few keys a sequence: a workgroup takes all of a tile's, of eight waves where the chip has
  // room, and nothing is to be joined, which takes 5 us and more.  The longest sequence then
  // takes 4.5 us and, for every 32 KB of its keys and as many of values, 1.8 (0.8 more in float32,
  // whose products are slower), which few workgroups would share better; from 129 on they fill the
  // chip anyway, those of heads above 128, one a CU, up to four rounds of it.
  // Measured, cut and whole, in us, one token of sequences of as many keys, or of up to as many:
  //   8 heads of 64 on 2, bfloat16     1 of 1,000 13.1 10.6, 1,500 13.4 13.0, 2,000 13.5 15.7
  //   32 of 64 on 8, bfloat16          30 of 1,500 29.6 19.4, up to 15.4 13.3; 3,000 43.9 34.1, up to 19.8 20.6;
  //                                    300 of 1,500 178 194, up to 60 39
  //   32 of 128 on 8, bfloat16         1 of 700 14.1 12.5, 1,000 14.1 15.0; 30 of 700 28.6 18.9, up to 16.4 12.9,
  //                                    1,500 44.3 32.1, up to 18.2 19.6; 128 of 1,000 107 102, up to 38.8 31.9
  //   32 of 64 on 8, float32           8 of 500 15.8 13.7, 1,000 21.4 21.9, up to 14.5 21.2; 30 of 700 30.8 18.6,
  //                                    up to 17.2 16.2, 1,000 37.1 24.0, up to 20.2 21.3
  //   32 of 256 on 8, bfloat16         8 of 300 17.3 18.5, 500 21.1 23.2, up to 16.9 22.2; 16 of 500 27.2 24.0, up to
  //                                    17.1 22.2; 30 of 500 38.6 28.0, up to 24.0 22.2; 60 of 500 58.9 51.7, up to
  //                                    32.7 27.0; 128 of 500 116 116, up to 58 55; 300 of 500 251 267, up to 107 118
  void whole(const msx_paged_attention_desc &d, const PagedArgs &a) {
    const int64_t units = a.batch * step.tiles * a.kv_heads;
    const int64_t bytes = held_bytes(d) / 2;
    int64_t most = 224 << 10;
    if (a.dim > 128)
      most = units > 128 && units <= 1024 ? 256 << 10 : 128 << 10;
    else if (units <= 128)
      most = d.vtype == MSX_F32 ? 128 << 10 : 192 << 10;
    if (units > max_blocks(8 * kWave) || bytes > most) return;
    step.whole = 1;
    step.waves = units <= 256 && a.dim <= 128 ? 8 : kStepWaves;
    step.groups = static_cast<int32_t>(units);
  }
  // The same of tiles of 128 queries.  Measured, cut and whole, in us, 16 heads on 4:
  //   bfloat16, heads of 64    300 tokens 24.0 13.3, 512 19.9 16.7, 64 on 1,000 20.1 26.3; 8 x 1,000 67 57
  //             heads of 128   512 tokens 25.6 22.9, 64 on 1,000 23.8 34.4; 8 x 1,000 102 81
  //             heads of 256   128 tokens 30.0 21.5, 512 35.6 43.5; 4 x 512 66.0 46.5
  //   float32, heads of 64     128 tokens 25.8 17.4, 300 29.5 31.5; 8 x 1,000 196 220
  void whole_tiles(const msx_paged_attention_desc &d, const PagedArgs &a) {
    const int64_t units = a.batch * tiles.tiles * a.kv_heads;
    const int64_t few = d.vtype == MSX_F32 ? 128 : a.dim <= 128 ? 512 : 256;
    if (units > max_blocks(256) || held_keys(d) > (units >= 512 ? 2 * few : few)) return;
    tiles.whole = 1;
    tiles.groups = static_cast<int32_t>(units);
  }
  PartSource source(const StepGrid &g, const TileParts &to, int32_t rows, bool batched) const {
    return {to.spans, to.whole, to.parts, rows, g.tiles, batched};
  }
};

}  // namespace
}  // namespace msx

using namespace msx;

extern "C" size_t msx_paged_attention_scratch(const msx_paged_attention_desc *desc) {
  if (check_paged_attention("paged_attention", desc) != MSX_OK || desc->batch == 0 ||
      desc->tokens == 0 || !countable(*desc))
    return 0;
  return Plan(*desc, args_of(*desc), nullptr, nullptr).bytes;
}

extern "C" msx_status msx_paged_attention(const msx_paged_attention_desc *desc, void *out,
                                          void *scratch, size_t scratch_bytes, void *stream) {
  clear_error();
  if (msx_status st = check_paged_attention("paged_attention", desc); st != MSX_OK) return st;
  if (desc->batch == 0 || desc->tokens == 0) return MSX_OK;
  if (out == nullptr) return fail(MSX_EINVAL, "paged_attention out is NULL.");
  if (!countable(*desc)) return fail(MSX_EINVAL, "paged_attention has more rows than its kernels count.");
  const PagedArgs a = args_of(*desc);
  const auto s = static_cast<hipStream_t>(stream);
  const auto vt = static_cast<msx_vtype>(desc->vtype);
  const Plan p(*desc, a, out, scratch);
  if (p.route == Route::kRows) {
    const int64_t rows = a.batch * a.tokens * a.heads;
    return by_vtype(desc->vtype, [&](auto v) {
      using V = decltype(v);
      constexpr int64_t kMost = max_blocks(kRowWaves * kWave) * kRowWaves;
      for (int64_t first = 0; first < rows; first += kMost)
        paged_rows<V><<<static_cast<unsigned>((std::min(rows - first, kMost) + kRowWaves - 1) / kRowWaves),
                        kRowWaves * kWave, 0, s>>>(a, first, rows, static_cast<typename V::Storage *>(out));
      const hipError_t e = hipGetLastError();
      return e == hipSuccess ? MSX_OK : hip_fail(e, "paged_attention");
    });
  }
  if (p.bytes > 0 && (scratch == nullptr || scratch_bytes < p.bytes || reinterpret_cast<uintptr_t>(scratch) % 16 != 0))
    return fail(MSX_EINVAL, "paged_attention scratch is too small or not aligned.");
  const PartSource none{};
  const PartSource by_step = p.source(p.step, p.step_to, kStepRows, false);
  const PartSource by_tiles = p.source(p.tiles, p.tiles_to, kTileRows, p.route == Route::kShared);
  msx_status st;
  switch (p.route) {
  case Route::kStep:
    st = launch_paged_step(vt, a, p.step, p.step_to, s);
    if (p.step.whole) return st;
    break;
  case Route::kTiles:
    st = launch_paged_tiles(vt, a, p.tiles, p.tiles_to, s);
    if (p.tiles.whole) return st;
    break;
  default: st = launch_paged_shared(vt, a, p.tiles, p.tiles_to, p.step, p.step_to, s); break;
  }
  if (st != MSX_OK) return st;
  switch (p.route) {
  case Route::kStep: return launch_paged_join(vt, a, by_step, none, out, s);
  case Route::kTiles: return launch_paged_join(vt, a, by_tiles, none, out, s);
  default: return launch_paged_join(vt, a, by_tiles, by_step, out, s);
  }
}
