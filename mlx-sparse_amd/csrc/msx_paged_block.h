// msx_paged_block.h - many queries against the same pages, chunks of prompts and the
// queries of a batch against the pages that it shares: what a workgroup does.
//
// A wave takes 32 rows (a row is a query and head; those of a query that share a kv
// head follow each other), a workgroup four such units, which share the tiles of
// keys in LDS.  Per tile: S^T = K Q^T, the running maximum and sum, O^T += V^T P^T,
// as in window_forward.hip; the next tile's rows are on their way to LDS meanwhile,
// the numbers of the pages after those in registers.  A row's probabilities are rounded
// to the operands' 16 bits for the second product, unnormalised, at most 2^8 (float16: 2^15):
// their errors are independent and no larger than the output's own rounding.
//
// Bound by products, exponentials and LDS reads taking turns, two waves a SIMD, at the clocks that power
// allows: 2,048 queries on 18,432 keys, 16 heads of 128 on 8, float16, 361 us, 809 TFLOP/s where a
// large matrix product reaches 1,080; 1,024 on 8,192, 16 heads on 4, bfloat16, 95 us (681), float32
// 616 (105 of 153).  What a score takes beside its products is the same for narrow heads, whose
// matrix cores wait for it: bfloat16 heads of 32 270 TFLOP/s, of 64 450, of 80 474, of 96 576; those of
// 256, a wave a SIMD and 32 keys a tile, 501.  64 sequences' queries against 8,192 shared keys: 36 us with
// their own keys beside.
//
// As in msx_paged_step.h each workgroup takes an equal stretch of all tiles, numbered by
// kv head, sequence and unit; of its first and last unit it may have a part, which
// paged_join joins.
#pragma once

#include "msx_paged.h"
#include "msx_paged_row.h"
#include "msx_paged_tiles.h"
#include "msx_window_mfma.h"

#pragma clang fp contract(fast)

namespace msx {

constexpr int kTileWaves = kTileRows / 32;
constexpr int kTileThreads = kTileWaves * kWave;

template <class V, int DP>
struct PagedShape {
  using T = TileShape<V, DP>;
  static constexpr int kSub = T::kSize == 2 && DP <= 128 ? 2 : 1;  // 32-key parts of a tile
  static constexpr int kKeys = 32 * kSub;
  static constexpr int kTile = kKeys * T::kPitch;
  static constexpr int kLds = 4 * kTile;  // K and V, twice
  // workgroups a CU: two hide each other's waits; wide float32 heads need the
  // registers of one
  static constexpr int kBlocks = T::kRowBytes > 256 ? 1 : 2;
};

__device__ __forceinline__ int32_t wave_least(int32_t v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = min(v, __shfl_xor(v, d));
  return __builtin_amdgcn_readfirstlane(v);
}

// The rows of a tile of keys and of their values, from the pages to LDS, sixteen bytes a
// piece.  Whole tiles go there directly: no registers on the way.  A wave's load takes a
// few rows that follow each other; where pages hold whole such groups, their address
// is uniform but for the lane's own offset.  (Caches whose strides differ go through
// registers: with an address for each, scalar registers run out.)
//
// A direct load puts lane i's piece at sixteen i bytes: the piece at place c of a row
// is the row's chunk c ^ f(row), the permutation of TileShape::along.
template <class V, int DP, int kKeys>
struct PageLoader {
  using T = TileShape<V, DP>;
  static constexpr int kPieces = kKeys * T::kChunks;
  static constexpr int kPer = kPieces / kTileThreads;
  static constexpr int kRows = kTileThreads / T::kChunks;     // between a thread's pieces
  static constexpr int kTogether = kWave / T::kChunks;    // rows of a wave's load
  static constexpr int kKinds = kRows % 16 == 0 ? 1 : 2;  // the permutation repeats after sixteen rows
  static_assert(kPieces % kTileThreads == 0 && kRows * kKinds % 16 == 0, "a thread's pieces are of one or two kinds");
  uint32_t offset[kKinds];  // of the thread's pieces from its wave's first row
  uint32_t page_step, slot_step;  // of both caches, in bytes
  int32_t dim;
  bool plain, grouped;            // uniform

  __device__ __forceinline__ explicit PageLoader(const PagedArgs &a)
      : page_step(static_cast<uint32_t>(a.ks[0] * T::kSize)), slot_step(static_cast<uint32_t>(a.ks[1] * T::kSize)), dim(a.dim) {
    plain = a.ks[0] == a.vs[0] && a.ks[1] == a.vs[1] && a.ks[0] * T::kSize == page_step &&
            a.ks[1] * T::kSize == slot_step && a.ks[1] * T::kSize * kTogether < (int64_t{1} << 31);
    grouped = a.table.size % kTogether == 0;
    const int row = threadIdx.x / T::kChunks;
#pragma unroll
    for (int kind = 0; kind < kKinds; ++kind)
      offset[kind] = static_cast<uint32_t>(row % kTogether) * slot_step +
                     chunk_at(row + kind * kRows, threadIdx.x % T::kChunks, a.dim) * 16;
  }
  // The chunk that goes to a place of a row.  Beyond the head's values it is the head's first:
  // there queries are zero and results are not kept.
  __device__ static __forceinline__ int chunk_at(int row, int place, int dim) {
    const int chunk = T::logical(row, place);
    return chunk * 16 < dim * T::kSize ? chunk : 0;
  }
  // The thread, for what is worked out where it is needed: the addresses of ways that a tile
  // seldom takes would otherwise be kept in registers.
  __device__ static __forceinline__ int this_thread() {
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    return thread;
  }
  __device__ static __forceinline__ void load(const char *from, char *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from),
                                     (__attribute__((address_space(3))) void *)(to), 16, 0, 0);
  }
  // The kKeys keys from j on, whose pages the lanes hold, all there.
  __device__ __forceinline__ void direct(const PageTable &table, const char *k, const char *v, int32_t pages,
                                         int32_t j, char *k_tile, char *v_tile) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    // where key `lane` lies: worked out by all lanes at once, a scalar a row group would take
    // ten times the instructions
    const uint64_t place = static_cast<uint64_t>(static_cast<uint32_t>(pages)) * page_step +
                           static_cast<uint64_t>(static_cast<uint32_t>(table.slot(j + lane))) * slot_step;
    const auto low = static_cast<int32_t>(place), high = static_cast<int32_t>(place >> 32);
    const auto both = [&](int r, uint64_t at, uint32_t more) {
      char *const to = k_tile + (r * kTileThreads + wave * kWave) * 16;
      load(k + at + more, to);
      load(v + at + more, to + (v_tile - k_tile));
    };
    if (grouped) {
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        const int row = r * kRows + wave * kTogether;
        both(r, static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(high, row))) << 32 |
                    static_cast<uint32_t>(__builtin_amdgcn_readlane(low, row)), offset[r % kKinds]);
      }
    } else {
      const int thread = this_thread();
#pragma unroll
      for (int r = 0; r < kPer; ++r) {
        const int row = r * kRows + thread / T::kChunks;
        both(r, static_cast<uint64_t>(static_cast<uint32_t>(__shfl(high, row))) << 32 |
                    static_cast<uint32_t>(__shfl(low, row)), chunk_at(row, thread % T::kChunks, dim) * 16);
      }
    }
  }
  // Of one cache, zeros for those that are not there.
  __device__ __forceinline__ void each(const PagedArgs &a, const char *cache, const int64_t *strides,
                                       int32_t pages, int32_t j, char *tile) const {
    const int thread = this_thread();
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int at = thread + r * kTileThreads, row = at / T::kChunks, chunk = at % T::kChunks;
      const int64_t page = __shfl(pages, row);
      if (chunk >= T::kUsed) continue;
      v4u piece = {0, 0, 0, 0};
      if (page >= 0 && chunk * 16 < a.dim * T::kSize)
        piece = *reinterpret_cast<const v4u *>(
            cache + (page * strides[0] + a.table.slot(j + row) * strides[1]) * T::kSize + chunk * 16);
      *reinterpret_cast<v4u *>(tile + T::along(row, chunk)) = piece;
    }
  }
};

// The values of 32 keys, from LDS as the second product takes them.
template <class V, int DP>
struct ValueColumns {
  using Frag = typename Mfma<V>::Frag;
  Frag a[DP / 32][2];
  __device__ __forceinline__ void read(const TileLanes<V, DP> &lanes, uint32_t tile, int row0) {
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v4s part[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) part[t] = read_transposed(lanes.column_at(tile, row0, 16 * k + 8 * t, dt));
        const auto lo = __builtin_bit_cast(v2u, part[0]), hi = __builtin_bit_cast(v2u, part[1]);
        a[dt][k] = __builtin_bit_cast(Frag, (v4u{lo[0], lo[1], hi[0], hi[1]}));
      }
  }
  // acc += V^T P, P rounded to the operands' type, or with `twice` that and what it leaves:
  // shared pages wait for loads, so that this costs nothing there and gives the results
  // their own rounding alone, as the sequences' own keys do.
  template <bool twice>
  __device__ __forceinline__ void times(const float (&p)[16], v16f (&acc)[DP / 32]) const {
    const Column<V> high(p);
    float rest[16];
    if constexpr (twice) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const v4u w = __builtin_bit_cast(v4u, high.b[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t pair = w[j];
          rest[8 * k + 2 * j] = p[8 * k + 2 * j] - V::widen(static_cast<uint16_t>(pair));
          rest[8 * k + 2 * j + 1] = p[8 * k + 2 * j + 1] - V::widen(static_cast<uint16_t>(pair >> 16));
        }
      }
    }
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int k = 0; k < 2; ++k) acc[dt] = Mfma<V>::mul(a[dt][k], high.b[k], acc[dt]);
    if constexpr (twice) {
      const Column<V> low(rest);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int k = 0; k < 2; ++k) acc[dt] = Mfma<V>::mul(a[dt][k], low.b[k], acc[dt]);
    }
  }
};
template <int DP>
struct ValueColumns<F32, DP> {
  float a[16][DP / 32];
  __device__ __forceinline__ void read(const TileLanes<F32, DP> &lanes, uint32_t tile, int row0) {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
        a[r][dt] = read_lds<float>(lanes.column_at(tile, row0, 8 * (r / 4) + r % 4, dt));
  }
  template <bool>
  __device__ __forceinline__ void times(const float (&p)[16], v16f (&acc)[DP / 32]) const {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[r][dt], p[r], acc[dt], 0, 0, 0);
  }
};

// The most and least of a workgroup's threads.
__device__ __forceinline__ void extremes(int32_t &most, int32_t &least, StretchLds &own) {
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) {
    most = max(most, __shfl_xor(most, d));
    least = min(least, __shfl_xor(least, d));
  }
  if (threadIdx.x % kWave == 0) {
    own.most[threadIdx.x / kWave] = most;
    own.least[threadIdx.x / kWave] = least;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kTileWaves; ++w) {
    most = max(most, own.most[w]);
    least = min(least, own.least[w]);
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
}

// The launch's first argument, read anew: what a unit needs of it once would otherwise be kept in
// scalar registers through the loop over its keys, and there are too few (280 spilled to
// vector registers, which are as scarce, at heads of 128).
__device__ __forceinline__ const PagedArgs &kernel_args() {
  auto p = (const __attribute__((address_space(4))) PagedArgs *)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PagedArgs *)p;
}

// Row r of those that share kv head `head`: of sequence b0, or of the batch.
template <bool kShared>
struct TileRow {
  int64_t b;
  int32_t t, h;
  bool held;  // has a place in the results
  __device__ __forceinline__ TileRow(const PagedArgs &a, int64_t b0, int32_t head, int32_t r) : b(b0) {
    t = r / a.group;
    h = head * a.group + r - t * a.group;
    if constexpr (kShared) {
      b = t / a.tokens;
      t -= static_cast<int32_t>(b) * a.tokens;
    }
    held = b < a.batch && t < a.tokens;
  }
};

// The first sequence that has queries here (0 where none has): slots without one need not hold
// the pages that the batch shares.
__device__ __forceinline__ int32_t first_live(const PagedArgs &a) {
  for (int64_t b0 = 0; b0 < a.batch; b0 += kWave) {
    const int64_t b = b0 + threadIdx.x % kWave;
    const uint64_t live = __ballot(b < a.batch && a.length(b) > 0);
    if (live != 0) return static_cast<int32_t>(b0) + __builtin_ctzll(live);
  }
  return 0;
}

// kShared: rows are those of the whole batch, keys those of the pages that it shares
// (grid.from of them, as the first sequence's row of the table lists them), and all results are parts.
// Where grid.whole a workgroup has all keys of one unit.  Workgroup `id` of grid.groups; `args`: the
// launch's first argument; `lds`: PagedShape's kLds bytes at a multiple of 1,024.
template <class V, int DP, bool kShared>
__device__ __forceinline__ void tiles_stretch(const PagedArgs &args, const StepGrid &grid, uint32_t id, const TileParts &to,
                                              char *lds, StretchLds &own) {
  using S = typename V::Storage;
  using F = PagedShape<V, DP>;
  using T = TileShape<V, DP>;
  using Frag = typename Mfma<V>::Frag;
  constexpr int kSteps = DP / Mfma<V>::kDepth;
  auto *const out = static_cast<S *>(to.out);
  const TileLanes<V, DP> lanes(lds);

  const int lane = threadIdx.x % kWave, half = lane / 32;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);

  // this workgroup's stretch of all tiles: numbered by kv head, then (sequence, unit)
  const int64_t entries = kShared ? grid.tiles : args.batch * grid.tiles;
  const int32_t shared_count = (grid.from + F::kKeys - 1) / F::kKeys;
  const auto count_at = [&](int64_t e) -> int32_t {
    const int64_t b = quotient(e, grid.tiles);
    return steps_of<F::kKeys, kTileRows>(args, b, static_cast<int32_t>(e - b * grid.tiles), 0).count;
  };
  const auto cost_at = [&](int64_t e) -> int64_t { return e < entries ? kStart + count_at(e) : 0; };
  bool even = false;
  int64_t unit_cost = 1, g = 0, begin = 0, end = 0, x = 0;  // x: where the next (kv head, entry) begins
  int32_t kvh, entry;
  StepShare share(0, int64_t{1});
  if (!kShared && grid.whole) {
    g = xcd_order(id, static_cast<uint32_t>(grid.groups));
    kvh = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(quotient(g, entries)));
    // (a prompt's last queries see most: they begin first)
    entry = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(entries - 1 - (g - kvh * entries)));
  } else {
    int64_t total = entries * (shared_count + kStart), cost = 0, upto = 0;
    int32_t most = shared_count, least = shared_count;
    if constexpr (!kShared) {
      int64_t mine = 0;
      most = 0;
      least = 0x7fffffff;
      for (int64_t e = threadIdx.x; e < entries; e += kTileThreads) {
        const int32_t count = count_at(e);
        if (e < kTileThreads) cost = kStart + count;
        mine += kStart + count;
        most = max(most, count);
        least = min(least, count);
      }
      upto = running_sums<kTileWaves>(mine, own.sums, total);
      extremes(most, least, own);
    }
    // Units that are nearly as long and fill the workgroups are cut alike: their workgroups then
    // read the same keys at the same time, through their XCD's L2 (2,048 queries on 18,432 keys: of
    // 1.54 GB that missed it 0.14 did, 393 to 367 us).
    const int64_t units = entries * args.kv_heads;
    const int64_t parts = units <= grid.groups ? quotient(grid.groups, units) : 1;
    even = least >= parts && total * 16 >= entries * (most + kStart) * 15 &&
                      (units <= grid.groups ? units * parts * 10 >= int64_t{grid.groups} * 9
                                            : units - quotient(units, grid.groups) * grid.groups == 0);
    unit_cost = quotient(most + kStart + parts - 1, parts) * parts;  // where even
    if (even) total = entries * unit_cost;
    share = even ? StepShare(total * args.kv_heads, min(units * parts, int64_t{grid.groups}))
                 : StepShare(total * args.kv_heads, grid.groups);
    if (id >= share.groups) return;  // whole workgroups leave
    g = xcd_order(id, static_cast<uint32_t>(share.groups));
    begin = share.first(g);
    end = share.first(g + 1);
    kvh = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(quotient(begin, total)));
    if (kShared || even) {
      const int64_t each = even ? unit_cost : shared_count + kStart;
      entry = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(quotient(begin - kvh * total, each)));
      x = kvh * total + entry * each;
    } else {
      const int64_t at = begin - kvh * total;
      int64_t before = 0;
      for (int64_t e0 = 0;; e0 += kTileThreads) {  // (all that is to be done is some entry's)
        int64_t here = total;
        if (entries > kTileThreads) {
          cost = cost_at(e0 + threadIdx.x);
          upto = running_sums<kTileWaves>(cost, own.sums, here);
        }
        if (before + upto - cost <= at && at < before + upto) {
          own.found = static_cast<int32_t>(e0 + threadIdx.x);
          own.found_first = before + upto - cost;
        }
        before += here;
        if (at < before || e0 + kTileThreads >= entries) break;
      }
      __syncthreads();
      entry = __builtin_amdgcn_readfirstlane(own.found);
      x = kvh * total + uniform(own.found_first);
    }
  }

  const int32_t lister = kShared ? __builtin_amdgcn_readfirstlane(first_live(args)) : 0;
  const PageLoader<V, DP, F::kKeys> rows(args);
  // a negative scale moves its sign to the queries, so that the largest product is the
  // largest score
  const float scale = fabsf(args.scale);

  for (bool more = (!kShared && grid.whole) || x < end; more;) {
    const PagedArgs &a = kernel_args();
    const int64_t b0 = kShared ? 0 : quotient(entry, grid.tiles);
    const int32_t block = kShared ? entry : entry - static_cast<int32_t>(b0) * grid.tiles;
    Steps steps;
    if constexpr (kShared) {
      steps.keys = Keys{0, 0, grid.from - 1, 0};
      steps.sinks = steps.window = 0;
      steps.count = shared_count;
    } else {
      steps = uniform(steps_of<F::kKeys, kTileRows>(a, b0, block, 0));
    }
    const int64_t first = x;
    int64_t from, upto_step;
    if (even) {
      x += unit_cost;
      from = quotient(max(begin - first, int64_t{0}) * steps.count, unit_cost);
      upto_step = quotient(min(end - first, unit_cost) * steps.count, unit_cost);
    } else {
      x += kStart + steps.count;
      if (!kShared && grid.whole) end = x;
      from = max(begin - first - kStart, int64_t{0});
      upto_step = min(end - first - kStart, static_cast<int64_t>(steps.count));
    }
    const int32_t s_begin = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(min(from, static_cast<int64_t>(steps.count))));
    const int32_t s_end = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(max(upto_step, int64_t{0})));
    more = x < end;
    const int32_t head = kvh, this_entry = entry;
    if (++entry == entries) {
      entry = 0;
      ++kvh;
    }
    if (s_begin >= s_end) continue;  // what this workgroup has of it is no step

    // this lane's row
    const TileRow<kShared> row(a, b0, head, block * kTileRows + wave * 32 + lane % 32);
    const bool live = row.held && row.t < a.length(row.b);
    Keys mine{0, 0, -1, 0};
    if (live) mine = a.keys(a.start(row.b), row.t, row.t);
    // (a window as wide as the table still hides keys from queries that stand behind it)
    if constexpr (kShared) mine.hi = min(mine.hi, grid.from - 1);
    // what the wave's rows see: all of them [all_lo, all_hi], any of them the rest
    const int32_t all_lo = -wave_least(live ? -mine.lo : 0), all_hi = wave_least(live ? mine.hi : 0x7fffffff);
    const int32_t any_hi = -wave_least(live ? -mine.hi : 1), any_lo = wave_least(live ? mine.lo : 0x7fffffff);
    const int32_t any_far = -wave_least(live ? -mine.far : 0);

    Frag qf[kSteps];
    {
      const char *q = reinterpret_cast<const char *>(static_cast<const S *>(a.q) + row.b * a.qs[0] +
                                                     row.t * a.qs[1] + row.h * a.qs[2]);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        v4u w = {0, 0, 0, 0};
        const int chunk = 2 * s + half;
        if (live && chunk * 16 < a.dim * T::kSize) w = *reinterpret_cast<const v4u *>(q + chunk * 16);
        if (a.scale < 0.0f) w ^= Mfma<V>::kSign;
        qf[s] = __builtin_bit_cast(Frag, w);
      }
    }
    const char *k_base = reinterpret_cast<const char *>(static_cast<const S *>(a.k) + head * a.ks[2]);
    const char *v_base = reinterpret_cast<const char *>(static_cast<const S *>(a.v) + head * a.vs[2]);

    PageTable table = a.table;  // of this sequence
    table.pages = static_cast<const char *>(table.pages) + (kShared ? lister : b0) * table.stride * (table.wide ? 8 : 4);

    // the page of key `lane` of a tile, none where nobody sees it
    const auto numbers_of = [&](int32_t s) {
      const int32_t j = steps.template key<F::kKeys>(s) + lane;
      return s < s_end && lane < F::kKeys && steps.keys.sees(j) ? table.number(0, j) : PageTable::none();
    };
    constexpr uint64_t kAll = ~uint64_t{0} >> (64 - F::kKeys);
    const auto fetch = [&](int32_t s, int32_t pages, int parity) {
      const int32_t j = steps.template key<F::kKeys>(s);
      char *k_to = lds + parity * F::kTile, *v_to = lds + (2 + parity) * F::kTile;
      if (rows.plain && __ballot(pages >= 0) == kAll) {
        rows.direct(table, k_base, v_base, pages, j, k_to, v_to);
      } else {
        rows.each(a, k_base, a.ks, pages, j, k_to);
        rows.each(a, v_base, a.vs, pages, j, v_to);
      }
    };

    v16f o[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
    float m = -INFINITY, base = 0.0f, l = 0.0f;  // l: of this lane's keys only

    const auto exponentials = [&](const v16f &from, float (&e)[16]) {
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        e[r] = exp2_fast(from[r] * scale - base);
        sum[r % 2] += e[r];
      }
      l += sum[0] + sum[1];
    };
    // masks the scores of the tile at j0 and moves the maximum.  It is moved only where
    // it has grown by more than 2^kLag: until then exponentials up to 2^kLag times those of its
    // scale stand beside sums of their own.  Float16's range holds that beside the weights below (see
    // kWeightsUp), 1,024 queries on 8,192 keys of scores that vary by a nat, and by three, in us:
    //   heads of 128   2^8 99.5 100.5, 2^4 99.1 101.8, 2^2 100.1 103.4, 2 102.1 104.1, 1 104.1 105.2
    //   heads of 256       257   264       257   276       267   288    282   297      307   307
    constexpr float kLag = kWeightsUp<V> > 0.0f ? 2.0f : 8.0f, kUp = std::max(kWeightsUp<V> - kLag, 0.0f);
    const auto settle = [&](int32_t j0, uint64_t there, v16f (&y)[F::kSub]) {
      const bool whole = there == kAll && j0 >= all_lo && j0 + F::kKeys - 1 <= all_hi;
      if (!whole) {
        const uint64_t seen = there >> (4 * half);
        const int32_t first = j0 + 4 * half;
#pragma unroll
        for (int i = 0; i < F::kSub; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int place = 32 * i + 8 * (r / 4) + r % 4;
            y[i][r] = (((seen >> place & 1) != 0) & mine.sees(first + place)) ? y[i][r] : -INFINITY;
          }
      }
      float tops[2] = {y[0][0], y[0][1]};
#pragma unroll
      for (int i = 0; i < F::kSub; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) tops[r % 2] = fmaxf(tops[r % 2], y[i][r]);
      float top = fmaxf(tops[0], tops[1]);
      top = fmaxf(top, other_half(top)) * scale;
      if (__any(top > m + (kUp + kLag))) {
        const float grown = fmaxf(m, top - kUp);
        const float shrink = grown == -INFINITY ? 1.0f : exp2_fast(m - grown);
        m = grown;
        base = m == -INFINITY ? 0.0f : m;
        l *= shrink;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[dt][r] *= shrink;
      }
    };

    int32_t pages = table.checked(numbers_of(s_begin));
    PageTable::Number ahead = numbers_of(s_begin + 1);
    fetch(s_begin, pages, 0);
    sync_tiles();
    const auto step = [&](int32_t s, int parity) __attribute__((always_inline)) {
      const int32_t j0 = steps.template key<F::kKeys>(s), j1 = j0 + F::kKeys - 1;
      const bool seen = j0 <= any_hi && (j1 >= any_lo || j0 < any_far);
      const uint64_t there = __ballot(pages >= 0);
      pages = table.checked(ahead);
      ahead = numbers_of(s + 2);
      const bool next = s + 1 < s_end;
      // (into the other tiles, which all waves are past; after this tile is read from LDS, since a
      // read that followed would wait for the loads)
      if (!seen) {
        if (next) fetch(s + 1, pages, parity ^ 1);
      } else {
        v16f y[F::kSub];
        {
          Frag kf[F::kSub][kSteps];
#pragma unroll
          for (int i = 0; i < F::kSub; ++i)
#pragma unroll
            for (int st = 0; st < kSteps; ++st)
              kf[i][st] = read_rows<V>(lanes, static_cast<uint32_t>(parity * F::kTile), 32 * i, st);
#pragma unroll
          for (int i = 0; i < F::kSub; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) y[i][r] = 0.0f;
#pragma unroll
            for (int st = 0; st < kSteps; ++st) y[i] = Mfma<V>::mul(kf[i][st], qf[st], y[i]);
          }
        }
        ValueColumns<V, DP> values;
        values.read(lanes, static_cast<uint32_t>((2 + parity) * F::kTile), 0);
        if (next) fetch(s + 1, pages, parity ^ 1);
        settle(j0, there, y);
#pragma unroll
        for (int i = 0; i < F::kSub; ++i) {
          float e[16];
          exponentials(y[i], e);
          if (i > 0) values.read(lanes, static_cast<uint32_t>((2 + parity) * F::kTile), 32 * i);
          values.template times<kShared && T::kSize == 2>(e, o);
        }
      }
      sync_tiles();
    };
    for (int32_t s = s_begin; s < s_end; s += 2) {
      step(s, 0);
      if (s + 1 < s_end) step(s + 1, 1);
    }

    l += other_half(l);
    // the row once more: its places would take registers all through the loop
    int32_t again = block * kTileRows + wave * 32 + lane % 32;
    asm volatile("" : "+v"(again));
    const TileRow<kShared> to_row(a, b0, head, again);
    if (mine.hi < 0) {  // sees nothing
      l = 0.0f;
      m = -INFINITY;
    }
    const bool all_of_it = s_begin == 0 && s_end == steps.count;
    const int64_t unit = static_cast<int64_t>(head) * entries + this_entry;
    if (threadIdx.x == 0 && s_begin == 0 && (kShared || !grid.whole))
      to.spans[unit] = all_of_it ? StepSpan{0, -1}
                              : StepSpan{static_cast<int32_t>(g),
                                         static_cast<int32_t>(share.owner(x - 1))};
    const bool held = to_row.held;
    const int64_t place = (to_row.b * a.tokens + to_row.t) * a.heads + to_row.h;
    if (kShared || !all_of_it) {
      float *part = all_of_it ? to.whole + place * part_stride(a.dim)
                            : to.parts + ((2 * g + (s_begin == 0 ? 1 : 0)) * kTileRows + wave * 32 + lane % 32) *
                                          part_stride(a.dim);
      if (held) {
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            const int d = dt * 32 + 2 * r + 4 * half;
            if (d < a.dim) *reinterpret_cast<v4f *>(part + d) = v4f{o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]};
          }
        if (half == 0) {
          part[a.dim] = m;
          part[a.dim + 1] = l;
        }
      }
      continue;  // (the last tile's waits are behind all waves)
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    bool odd = false;  // something is not finite: the row is computed anew
    if (held) {
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const int d = dt * 32 + 2 * r + 4 * half;
          float y[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            y[k] = l == 0.0f ? 0.0f : o[dt][r + k] * inv;
            odd = odd || !(fabsf(y[k]) < INFINITY);
          }
          if (d < a.dim) store_four<V>(y, y, out + place * a.dim + d, nullptr);
        }
    }
    uint64_t anew = __ballot(odd);
    anew = (anew | anew >> 32) & 0xffffffffu;
    if (__syncthreads_or(anew != 0)) {
      while (anew != 0) {  // the tiles in LDS are done with: all waves left the loop
        const int i = __builtin_ctzll(anew);
        anew &= anew - 1;
        paged_row<V>(a, b0, __shfl(to_row.t, i), __shfl(to_row.h, i), reinterpret_cast<float *>(lds) + wave * kWindowMaxDim, out);
      }
      __syncthreads();
    }
  }
}

}  // namespace msx
