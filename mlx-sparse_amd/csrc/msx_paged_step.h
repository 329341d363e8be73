// msx_paged_step.h - a few queries of every sequence against its pages: what a
// workgroup does.
//
// Bound by memory: every visible key and value is read once, 2 flops a byte, query
// and head.  The queries and heads that share a kv head (sixteen at a time) share
// each read, as the sixteen columns of matrix products; a wave takes 32 keys (16 in
// float32) after the other, with the next ones in flight and their pages' numbers
// a step ahead of them, and keeps running maximum, sum and output of its own.
//
// Sequences differ in length, and the host knows none of them.  The steps of all
// (sequence, sixteen queries, kv head) are numbered through, and each workgroup takes
// an equal stretch of them, whatever it begins and ends in: every workgroup adds
// up the batch's lengths to find its own.  Of a stretch only the first and the last tile
// of queries can be another's as well; what it has of them goes to two places
// of scratch, and paged_join adds those up in the order of the keys.
//
// One token of 131,072 keys, 32 heads of 128 on 8, bfloat16: 103 us, 5.2 TB/s; 64 sequences of up
// to 16,384, cold, 113 us with joining (4.9 TB/s); 32 of 4,000, 16 heads on 4, 52 us (5.1); 32 of
// 4,000 in float32, heads of 256, 193 us (5.4).  Rows that end within a line of 128 bytes move the
// lines that two kv heads share once for each, their workgroups lying on different XCDs: 16-bit heads of 32
// take 33 us, of 80 50 and of 96 49, where heads of 64 take 34 and of 128 52.  Two workgroups a CU are what
// registers allow; for heads of 64 at most, where they would allow four, one took up to 60 % more, three or
// four 25 % less to 20 more.
#pragma once

#include "msx_paged.h"
#include "msx_paged_row.h"
#include "msx_paged_tiles.h"
#include "msx_step_mfma.h"

#pragma clang fp contract(fast)

namespace msx {

template <class V, int DP, int kWaves>
constexpr int step_lds() {
  return std::max(kWaves * StepShape<V, DP>::kTile, kWaves * kStepRows * (DP + 4) * 4);
}

// Workgroup g of grid.groups.  `lds`: step_lds bytes at a sixteen-byte address.
// Where grid.whole (a workgroup of eight waves always is) it has all keys of one tile.
// kPast: keys and values go past the caches.
template <class V, int DP, int kWaves = kStepWaves, bool kPast = false>
__device__ __forceinline__ void step_stretch(const PagedArgs &a, const StepGrid &grid, int64_t g, const TileParts &to,
                                             char *lds, StretchLds &own) {
  using S = typename V::Storage;
  using F = StepShape<V, DP>;
  constexpr int kThreads = kWaves * kWave;
  // steps of a row's sixty-four bytes that every head of this kernel has
  constexpr int kSure = (DP <= 128 ? DP - 32 : 128) * F::kSize / 64;
  constexpr uint32_t kAll = static_cast<uint32_t>((uint64_t{1} << F::kKeys) - 1);
  const bool alike = a.ks[0] == a.vs[0] && a.ks[1] == a.vs[1];
  constexpr bool kAlwaysWhole = kWaves != kStepWaves;
  auto *const out = static_cast<S *>(to.out);

  const int lane = threadIdx.x % kWave, quad = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int bytes = a.dim * F::kSize;

  // this workgroup's stretch of all steps
  const int64_t entries = a.batch * grid.tiles;  // (sequence, sixteen queries)
  const auto cost_at = [&](int64_t e) -> int64_t {
    if (e >= entries) return 0;
    const int64_t b = grid.tiles == 1 ? e : e / grid.tiles;
    return kStart + steps_of<F::kKeys, kStepRows>(a, b, static_cast<int32_t>(e - b * grid.tiles), grid.from).count;
  };
  int32_t entry, kvh = -1;
  int64_t begin = 0, end = 0, x = 0;  // x: where the next (entry, kv head) begins
  StepShare share(0, int64_t{1});
  const bool whole_grid = kAlwaysWhole || grid.whole;
  if (whole_grid) {
    entry = static_cast<int32_t>(quotient(g, a.kv_heads));
    kvh = static_cast<int32_t>(g - entry * static_cast<int64_t>(a.kv_heads));
  } else {
    int64_t total = 0, cost = cost_at(threadIdx.x), upto = running_sums<kWaves>(cost, own.sums, total);
    if (entries > kThreads) {
      int64_t mine = cost;
      for (int64_t e = threadIdx.x + kThreads; e < entries; e += kThreads) mine += cost_at(e);
      running_sums<kWaves>(mine, own.sums, total);
    }
    share = StepShare(total * a.kv_heads, grid.groups);
    if (g >= share.groups) return;  // whole workgroups leave
    begin = share.first(g);
    end = share.first(g + 1);
    int64_t before = 0;
    for (int64_t e0 = 0;; e0 += kThreads) {  // (all that is to be done is some entry's)
      int64_t here = total;
      if (entries > kThreads) {
        if (e0 > 0) cost = cost_at(e0 + threadIdx.x);
        upto = running_sums<kWaves>(cost, own.sums, here);
      }
      const int64_t low = (before + upto - cost) * a.kv_heads, high = (before + upto) * a.kv_heads;
      if (low <= begin && begin < high) {
        own.found = static_cast<int32_t>(e0 + threadIdx.x);
        own.found_first = low;
      }
      before += here;
      if (begin < before * a.kv_heads || e0 + kThreads >= entries) break;
    }
    __syncthreads();
    entry = __builtin_amdgcn_readfirstlane(own.found);
    x = uniform(own.found_first);
  }

  for (;;) {
    const int64_t b = grid.tiles == 1 ? entry : entry / grid.tiles;
    const int32_t row_tile = entry - static_cast<int32_t>(b) * grid.tiles;
    const Steps steps = uniform(steps_of<F::kKeys, kStepRows>(a, b, row_tile, grid.from));
    if (kvh < 0) {
      kvh = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(quotient(begin - x, steps.count + kStart)));
      x += static_cast<int64_t>(kvh) * (steps.count + kStart);
    }
    const int64_t first_step = x + kStart;
    x = first_step + steps.count;
    if (whole_grid) end = x;
    const int32_t s_begin = __builtin_amdgcn_readfirstlane(
        static_cast<int32_t>(min(max(begin - first_step, int64_t{0}), static_cast<int64_t>(steps.count))));
    const int32_t s_end = __builtin_amdgcn_readfirstlane(
        static_cast<int32_t>(max(min(end - first_step, static_cast<int64_t>(steps.count)), int64_t{0})));
    const int32_t head = kvh, mine_entry = entry;
    if (++kvh == a.kv_heads) {
      kvh = 0;
      ++entry;
    }
    if (s_begin >= s_end) {  // what this workgroup has of it is no step
      if (x >= end) break;
      continue;
    }
    const auto key_of = [&](int32_t s) { return steps.template key<F::kKeys>(s); };

    // this lane's query, and what it sees
    const int32_t row = row_tile * kStepRows + lane % 16, t = row / a.group;
    const int32_t h = head * a.group + row % a.group;
    const bool live = t <= steps.last;
    Keys mine{0, 0, -1, 0};
    if (live) mine = a.keys(a.start(b), t, t);

    v4u qf[F::kSteps];
    {
      const char *q = reinterpret_cast<const char *>(static_cast<const S *>(a.q) + b * a.qs[0] +
                                                     t * a.qs[1] + h * a.qs[2]);
#pragma unroll
      for (int s = 0; s < F::kSteps; ++s) {
        const int c = 4 * s + quad;
        qf[s] = v4u{0, 0, 0, 0};
        if (live && c * 16 < bytes) qf[s] = *reinterpret_cast<const v4u *>(q + c * 16);
      }
    }
    // all of the tile's queries that are there see [all_lo, all_hi]
    const int32_t first_t = row_tile * kStepRows / a.group;
    const int32_t all_lo = __builtin_amdgcn_readfirstlane(a.keys(a.start(b), steps.last, steps.last).lo);
    const int32_t all_hi = steps.keys.hi - (steps.last - first_t);
    const char *ck = reinterpret_cast<const char *>(static_cast<const S *>(a.k) + head * a.ks[2]);
    const char *cv = reinterpret_cast<const char *>(static_cast<const S *>(a.v) + head * a.vs[2]);

    // the page of key `lane` of a step, none where nobody sees it
    const auto numbers_of = [&](int32_t s) {
      const int32_t j = key_of(s) + lane;
      return s < s_end && lane < F::kKeys && steps.keys.sees(j) ? a.table.number(b, j) : PageTable::none();
    };
    v4u kf[F::kTiles][F::kSteps], vf[F::kVPer];
    // Where the keys of a step lie, a key a lane, and their values.  Those that nobody sees are given the
    // first one's place: their weight is zero, and no load asks whether it may.
    struct Places {
      uint64_t k, v;
    };
    const auto places_of = [&](int32_t s, int32_t pages, uint32_t there) {
      const auto slot = static_cast<uint32_t>(a.table.slot(key_of(s) + lane)), page = static_cast<uint32_t>(pages);
      const auto at = [&](const int64_t *strides) {
        const uint64_t place = (static_cast<uint64_t>(strides[0]) * page + static_cast<uint64_t>(strides[1]) * slot) * F::kSize;
        const int first = __builtin_ctz(there);
        const auto low = __builtin_amdgcn_readlane(static_cast<int32_t>(place), first);
        const auto high = __builtin_amdgcn_readlane(static_cast<int32_t>(place >> 32), first);
        return pages >= 0 ? place : static_cast<uint64_t>(static_cast<uint32_t>(high)) << 32 | static_cast<uint32_t>(low);
      };
      Places p;
      p.k = at(a.ks);
      p.v = alike ? p.k : at(a.vs);
      return p;
    };
    const auto of_key = [](uint64_t places, int key) {
      const auto low = static_cast<uint32_t>(__shfl(static_cast<int32_t>(places), key));
      return static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int32_t>(places >> 32), key))) << 32 | low;
    };
    const auto piece = [](const char *from) {
      if constexpr (kPast) return __builtin_nontemporal_load(reinterpret_cast<const v4u *>(from));
      return *reinterpret_cast<const v4u *>(from);
    };
    const auto fetch_k = [&](const Places &places) {
#pragma unroll
      for (int i = 0; i < F::kTiles; ++i) {
        const char *from = ck + of_key(places.k, 16 * i + lane % 16) + quad * 16;
#pragma unroll
        for (int c = 0; c < F::kSteps; ++c) {
          // beyond the head's values its first: queries are zero there
          const int more = c < kSure || (4 * c + quad) * 16 < bytes ? 64 * c : -quad * 16;
          kf[i][c] = piece(from + more);
        }
      }
    };
    const auto fetch_v = [&](const Places &places) {
      const int chunk = lane % F::kChunks * 16 < bytes ? lane % F::kChunks * 16 : 0;  // (nor are such sums kept)
#pragma unroll
      for (int r = 0; r < F::kVPer; ++r)
        vf[r] = piece(cv + of_key(places.v, (lane + r * kWave) / F::kChunks) + chunk);
    };

    char *tile = lds + wave * F::kTile;
    v4f o[DP / 16];
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[d] = v4f{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;  // l: this lane's keys only

    int32_t step = s_begin + wave;
    PageTable::Number ahead = numbers_of(step + kWaves);
    uint32_t there;  // keys of a step that somebody sees
    {
      const int32_t pages = a.table.checked(numbers_of(step));
      there = static_cast<uint32_t>(__ballot(pages >= 0));
      if (there != 0) {
        const Places places = places_of(step, pages, there);
        fetch_k(places);
        fetch_v(places);
      }
    }
    for (; step < s_end; step += kWaves) {
      const uint32_t here = there;
      v4f s[F::kTiles];
      if (here != 0) {
#pragma unroll
        for (int i = 0; i < F::kTiles; ++i) {
          s[i] = v4f{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < F::kSteps; ++c) s[i] = Mfma16<V>::mul(kf[i][c], qf[c], s[i]);
        }
      }
      const int32_t pages = a.table.checked(ahead);
      there = static_cast<uint32_t>(__ballot(pages >= 0));
      ahead = numbers_of(step + 2 * kWaves);
      Places places{0, 0};
      if (there != 0) {
        places = places_of(step + kWaves, pages, there);
        fetch_k(places);
      }
      if (here != 0) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < F::kVPer; ++r) {
          const int at = lane + r * kWave;
          *reinterpret_cast<v4u *>(tile + F::at(at / F::kChunks, at % F::kChunks)) = vf[r];
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      if (there != 0) fetch_v(places);
      if (here == 0) continue;

      float x[F::kTiles * 4], top = -INFINITY;
      const int32_t j0 = key_of(step);
      if (here == kAll && j0 >= all_lo && j0 + F::kKeys - 1 <= all_hi) {
#pragma unroll
        for (int i = 0; i < F::kTiles; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) x[4 * i + k] = s[i][k] * a.scale;
      } else {
        const uint32_t mine_here = here >> (4 * quad);
#pragma unroll
        for (int i = 0; i < F::kTiles; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int place = 16 * i + k;
            const bool seen = ((mine_here >> place & 1) != 0) & mine.sees(j0 + 4 * quad + place);
            x[4 * i + k] = seen ? s[i][k] * a.scale : -INFINITY;
          }
      }
#pragma unroll
      for (int k = 0; k < F::kTiles * 4; ++k) top = fmaxf(top, x[k]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float grown = fmaxf(m, top - kWeightsUp<V>);
      const float base = grown == -INFINITY ? 0.0f : grown;
      if (__any(grown > m)) {
        const float shrink = exp2_fast(m - base);
        l *= shrink;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[d] *= shrink;
      }
      m = grown;
#pragma unroll
      for (int k = 0; k < F::kTiles * 4; ++k) {
        x[k] = exp2_fast(x[k] - base);
        l += x[k];
      }
      if constexpr (F::kSize == 2) {
        v4u p, low;  // rounded, and what that leaves: of a weight 2^-22 at most in float16, 2^-16 in bfloat16
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t pair = Mfma<V>::pack(x[2 * k], x[2 * k + 1]);
          p[k] = pair;
          low[k] = Mfma<V>::pack(x[2 * k] - V::widen(static_cast<uint16_t>(pair)),
                                 x[2 * k + 1] - V::widen(static_cast<uint16_t>(pair >> 16)));
        }
        const int i = lane % 16;
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) {
          v4s part[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int place = 16 * k + 4 * quad + i / 4, column = d * 16 + (i % 4) * 4;
            part[k] = read_transposed(tile + F::at(place, column / 8) + (column % 8) * 2);
          }
          const auto lo = __builtin_bit_cast(v2u, part[0]), hi = __builtin_bit_cast(v2u, part[1]);
          const v4u values{lo[0], lo[1], hi[0], hi[1]};
          o[d] = Mfma16<V>::mul(values, p, o[d]);
          o[d] = Mfma16<V>::mul(values, low, o[d]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) {
            const int place = 4 * quad + i, column = d * 16 + lane % 16;
            const float v = *reinterpret_cast<const float *>(tile + F::at(place, column / 4) + (column % 4) * 4);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, x[i], o[d], 0, 0, 0);
          }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (!live) {
      l = 0.0f;
      m = -INFINITY;
    }

    // the waves' parts, joined: a row of DP sums, m and l a query and wave
    __syncthreads();
    float *sums = reinterpret_cast<float *>(lds) + (wave * kStepRows + lane % 16) * (DP + 4);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) *reinterpret_cast<v4f *>(sums + 16 * d + 4 * quad) = o[d];
    if (quad == 0) {
      sums[DP] = m;
      sums[DP + 1] = l;
    }
    if (threadIdx.x == 0) own.odd = 0;
    __syncthreads();
    const bool whole = s_begin == 0 && s_end == steps.count;
    const int64_t unit = static_cast<int64_t>(head) * entries + mine_entry;
    if (threadIdx.x == 0 && s_begin == 0 && !whole_grid)
      to.spans[unit] = whole ? StepSpan{0, -1}
                          : StepSpan{static_cast<int32_t>(g),
                                     static_cast<int32_t>(share.owner(first_step + steps.count - 1))};
    const float *all = reinterpret_cast<const float *>(lds);
    const int32_t rows = min(kStepRows, a.tokens * a.group - row_tile * kStepRows);
    for (int at = threadIdx.x; at < rows * DP; at += kThreads) {
      const int i = at / DP, d = at % DP;
      if (d >= a.dim) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, all[(w * kStepRows + i) * (DP + 4) + DP]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, norm = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float *from = all + (w * kStepRows + i) * (DP + 4);
        const float f = exp2_fast(from[DP] - base);
        sum += from[d] * f;
        norm += from[DP + 1] * f;
      }
      const int32_t r = row_tile * kStepRows + i;
      const int64_t place = (b * a.tokens + r / a.group) * a.heads + head * a.group + r % a.group;
      if (whole && to.whole == nullptr) {
        const float value = norm == 0.0f ? 0.0f : sum / norm;
        if (!(fabsf(value) < INFINITY)) atomicOr(&own.odd, 1u << i);
        out[place * a.dim + d] = V::narrow(value);
      } else {
        float *part = whole ? to.whole + place * part_stride(a.dim)
                            : to.parts + ((2 * g + (s_begin == 0 ? 1 : 0)) * kStepRows + i) * part_stride(a.dim);
        part[d] = sum;
        if (d == 0) {
          part[a.dim] = top;
          part[a.dim + 1] = norm;
        }
      }
    }
    __syncthreads();
    for (uint32_t anew = own.odd; anew != 0; anew &= anew - 1) {
      const int i = __builtin_ctz(anew);
      if (i % kWaves != wave) continue;
      const int32_t r = row_tile * kStepRows + i;
      paged_row<V>(a, b, r / a.group, head * a.group + r % a.group,
                   reinterpret_cast<float *>(lds) + wave * DP, out);
    }
    if (x >= end) break;
    __syncthreads();
  }
}

}  // namespace msx
