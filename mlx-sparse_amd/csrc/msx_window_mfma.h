// msx_window_mfma.h - matrix-core tiles of window attention.
//
// Scores are computed transposed, S^T = K Q^T (32 keys x 32 queries a tile):
// a lane then holds one query, lane % 32, and of each 32 keys the sixteen
//   key(i) = 8 (i / 4) + 4 (lane / 32) + i % 4,   i = 0 .. 15,
// so a row of the softmax is a lane's own values and one exchange with the
// lane 32 away.  The next product, O^T = V^T P^T, takes its k index in that
// same order: P needs no shuffle, only its rounding, and V^T is read in the
// matching order (16-bit values through the transposing LDS read, which hands
// a lane four keys of one column).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "msx_device.h"
#include "msx_window.h"

namespace msx {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));

// A tile of rows in LDS: rows of `kPitch` bytes, their 16-byte chunks
// permuted by row so that the reads below spread over the banks.
template <class V, int DP>
struct TileShape {
  static constexpr int kSize = sizeof(typename V::Storage);
  static constexpr int kRowBytes = DP * kSize;
  static constexpr int kPitch = kRowBytes <= 64 ? 64 : kRowBytes <= 128 ? 128 : kRowBytes <= 256 ? 256 : 512;
  static constexpr int kChunks = kPitch / 16;      // of which kRowBytes / 16 are used
  static constexpr int kUsed = kRowBytes / 16;

  // Sixteen rows read at one chunk (a lane a row) fall into sixteen chunks of
  // the 256 bytes that the banks span, and so do the four rows by four chunks
  // that half a wave's transposing read takes.
  __device__ static __forceinline__ int along(int row, int chunk) {
    return row * kPitch + logical(row, chunk) * 16;
  }
  // The chunk at a place of the row, and the place of a chunk.
  __device__ static __forceinline__ int logical(int row, int chunk) {
    const int low = kPitch >= 256 ? (row & 3) << 2 : kPitch == 128 ? (row & 2) << 1 : 0;
    return chunk ^ (low | ((row >> 2) & 3));
  }
};

template <class V>
struct Mfma;

// 16-bit operands: 32 x 32 x 16 products; a lane holds eight adjacent values
// of its row, at 8 (lane / 32) of each sixteen.
template <>
struct Mfma<BF16> {
  using Frag = v8bf;
  static constexpr int kDepth = 16;
  __device__ static __forceinline__ v16f mul(Frag a, Frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{lo, hi}), v2bf));
  }
  static constexpr uint32_t kSign = 0x80008000u;
};
template <>
struct Mfma<F16> {
  using Frag = v8h;
  static constexpr int kDepth = 16;
  __device__ static __forceinline__ v16f mul(Frag a, Frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{lo, hi}), v2h));
  }
  static constexpr uint32_t kSign = 0x80008000u;
};
// float32: 32 x 32 x 2 products.  Sixteen bytes a lane serve four of them:
// product j of a group of eight values takes values j and 4 + j.
template <>
struct Mfma<F32> {
  using Frag = v4f;
  static constexpr int kDepth = 8;
  __device__ static __forceinline__ v16f mul(Frag a, Frag b, v16f c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static constexpr uint32_t kSign = 0x80000000u;
};

// What a pair of results has beyond `kept`.
template <class V>
__device__ __forceinline__ uint32_t residues(float x0, float x1, uint32_t kept) {
  return Mfma<V>::pack((x0 - V::widen(static_cast<uint16_t>(kept))) * Residue<V>::kUp,
                       (x1 - V::widen(static_cast<uint16_t>(kept >> 16))) * Residue<V>::kUp);
}

// Four results of a row in the operands' type, and where asked for what
// `better` ones have beyond that.
template <class V>
__device__ __forceinline__ void store_four(const float (&x)[4], const float (&better)[4],
                                           typename V::Storage *out, typename V::Storage *low) {
  if constexpr (sizeof(typename V::Storage) == 2) {
    const v2u w{Mfma<V>::pack(x[0], x[1]), Mfma<V>::pack(x[2], x[3])};
    *reinterpret_cast<v2u *>(out) = w;
    if (low != nullptr)
      *reinterpret_cast<v2u *>(low) = v2u{residues<V>(better[0], better[1], w[0]),
                                          residues<V>(better[2], better[3], w[1])};
  } else {
    *reinterpret_cast<v4f *>(out) = v4f{x[0], x[1], x[2], x[3]};
  }
}

using LdsPtr = const __attribute__((address_space(3))) char *;
__device__ __forceinline__ uint32_t lds_address(const char *p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LdsPtr)(p)));
}

// Where a lane reads tiles in LDS.  TileShape's permutation is linear over the
// bits of row and chunk, and what varies by lane and what is known when
// compiling lie in different bits of both: an address is the lane's part, an
// exclusive or with a constant, and the instruction's own offset.  (Worked out
// from row and chunk each, the addresses of a tile took forty registers.)
template <class V, int DP>
struct TileLanes {
  using T = TileShape<V, DP>;
  uint32_t rows;     // a row a lane: row lane % 32, chunk lane / 32
  uint32_t columns;  // see mul_transposed

  __device__ __forceinline__ explicit TileLanes(const char *lds) {
    const int lane = threadIdx.x % kWave, half = lane / 32;
    const uint32_t base = lds_address(lds);
    rows = base + T::along(lane % 32, half);
    if constexpr (T::kSize == 2) {
      const int i = lane % 16, place = ((lane / 16) % 2) * 16 + (i % 4) * 4;
      columns = base + T::along(4 * half + i / 4, place / 8) + (place % 8) * 2;
    } else {
      columns = base + T::along(4 * half, (lane % 32) / 4) + (lane % 4) * 4;
    }
  }
  // Of the tile at byte `tile` of LDS, row row0 + lane % 32, chunk 2 step + half.
  __device__ __forceinline__ const char *row_at(uint32_t tile, int row0, int step) const {
    return at(rows, tile + row0 * T::kPitch, 0, 2 * step);
  }
  // The lane's place of the columns from 32 dt on, `row` rows below row0.
  __device__ __forceinline__ const char *column_at(uint32_t tile, int row0, int row, int dt) const {
    return at(columns, tile + row0 * T::kPitch, row, dt * (32 * T::kSize / 16));
  }

 private:
  __device__ static __forceinline__ const char *at(uint32_t lane, uint32_t tile, int row, int chunk) {
    return (const char *)(LdsPtr)(static_cast<uintptr_t>(
        (lane ^ static_cast<uint32_t>(T::logical(row, chunk) * 16)) + tile + row * T::kPitch));
  }
};

// The same addresses worked out from row and chunk each, of an array that the
// compiler knows: it then moves reads past what is written elsewhere.
template <class V, int DP>
struct TilePlaces {
  using T = TileShape<V, DP>;
  const char *base;
  __device__ __forceinline__ explicit TilePlaces(const char *lds) : base(lds) {}
  __device__ __forceinline__ const char *row_at(uint32_t tile, int row0, int step) const {
    const int lane = threadIdx.x % kWave;
    return base + tile + T::along(row0 + lane % 32, 2 * step + lane / 32);
  }
  __device__ __forceinline__ const char *column_at(uint32_t tile, int row0, int row, int dt) const {
    const int lane = threadIdx.x % kWave, half = lane / 32;
    if constexpr (T::kSize == 2) {
      const int i = lane % 16, d = dt * 32 + ((lane / 16) % 2) * 16 + (i % 4) * 4;
      return base + tile + T::along(row0 + row + 4 * half + i / 4, d / 8) + (d % 8) * 2;
    } else {
      const int d = dt * 32 + lane % 32;
      return base + tile + T::along(row0 + row + 4 * half, d / 4) + (d % 4) * 4;
    }
  }
};

template <class X>
__device__ __forceinline__ X read_lds(const char *at) {
  return *reinterpret_cast<const X *>(at);
}

// Sixteen bytes of a row for step `s` of a product over the head dimension:
// chunk 2 s + lane / 32 in either type, of row row0 + lane % 32 (row0 a
// multiple of 32: the permutation starts anew there).
template <class V, class Lanes>
__device__ __forceinline__ typename Mfma<V>::Frag read_rows(const Lanes &lanes, uint32_t tile,
                                                            int row0, int s) {
  return read_lds<typename Mfma<V>::Frag>(lanes.row_at(tile, row0, s));
}

__device__ __forceinline__ v4s read_transposed(const char *at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) v4s *)(static_cast<uintptr_t>(lds_address(at))));
}

// A lane's sixteen values in the order above as the second operand of a
// product: rounded to 16 bits, or as they are.
template <class V>
struct Column {
  typename Mfma<V>::Frag b[2];
  __device__ __forceinline__ explicit Column(const float (&p)[16]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v4u w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = Mfma<V>::pack(p[8 * k + 2 * j], p[8 * k + 2 * j + 1]);
      b[k] = __builtin_bit_cast(typename Mfma<V>::Frag, w);
    }
  }
};
template <>
struct Column<F32> {
  float p[16];
  __device__ __forceinline__ explicit Column(const float (&from)[16]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = from[r];
  }
};

// The sum of a column as the products take it: divided by this, probabilities
// sum to one however they were rounded.
__device__ __forceinline__ float rounded_sum(const Column<BF16> &c) {
  constexpr v2bf kOnes = {1.0f, 1.0f};
  float sum[2] = {0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const v4u w = __builtin_bit_cast(v4u, c.b[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = w[j];
      sum[j % 2] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pair), kOnes, sum[j % 2], false);
    }
  }
  return sum[0] + sum[1];
}
__device__ __forceinline__ float rounded_sum(const Column<F16> &c) {
  constexpr v2h kOnes = {1.0f, 1.0f};
  float sum[2] = {0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const v4u w = __builtin_bit_cast(v4u, c.b[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = w[j];
      sum[j % 2] = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, pair), kOnes, sum[j % 2], false);
    }
  }
  return sum[0] + sum[1];
}

// acc[dt] += X^T P over 32 rows of the tile from `row0` on (a multiple of 32), X
// read along its columns.
template <class V, class Lanes, int kBlocks>
__device__ __forceinline__ void mul_transposed(const Lanes &lanes, uint32_t tile, int row0,
                                               const Column<V> &column, v16f (&acc)[kBlocks]) {
  if constexpr (sizeof(typename V::Storage) == 2) {
#pragma unroll
    for (int dt = 0; dt < kBlocks; ++dt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        v4s part[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
          part[t] = read_transposed(lanes.column_at(tile, row0, 16 * k + 8 * t, dt));
        const auto lo = __builtin_bit_cast(v2u, part[0]), hi = __builtin_bit_cast(v2u, part[1]);
        const auto a = __builtin_bit_cast(typename Mfma<V>::Frag, (v4u{lo[0], lo[1], hi[0], hi[1]}));
        acc[dt] = Mfma<V>::mul(a, column.b[k], acc[dt]);
      }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int dt = 0; dt < kBlocks; ++dt) {
        const float a = read_lds<float>(lanes.column_at(tile, row0, 8 * (r / 4) + r % 4, dt));
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, column.p[r], acc[dt], 0, 0, 0);
      }
  }
}

// A span of keys numbered through (sinks before it, then itself), and which of
// them a position sees: those no further back than `window`, any of the first
// `free` numbers.
struct Numbering {
  int32_t far, skip, free, window;
  __device__ __forceinline__ Numbering(const WindowArgs &a, int32_t near)
      : far(min(a.sinks, near)), skip(near - far), free(skip == 0 ? a.sinks : far), window(a.window) {}
  __device__ __forceinline__ int32_t key(int32_t c) const { return c < far ? c : c + skip; }
};

// What the query at p (-1 sees nothing) sees of numbers c0 + e, e known when
// compiling.  A sink before the span is never ahead of the span's queries, so that
// one comparison serves sinks on both sides of it: not past p, not past the
// sinks.
struct SeenFrom {
  int32_t back, ahead;
  uint32_t window;
  __device__ __forceinline__ SeenFrom(const Numbering &n, int32_t p, int32_t c0)
      : back(p - n.skip - c0), ahead(min(p, n.free - 1) - c0), window(n.window) {}
  __device__ __forceinline__ bool operator()(int32_t e) const {
    return (static_cast<uint32_t>(back - e) < window) | (e <= ahead);
  }
};

// A workgroup's share of a tile's rows, from memory to LDS, sixteen bytes a
// piece.  Whole tiles go there directly: no registers on the way, and the
// address of a tile is uniform, so that a piece costs one instruction (a prompt
// of 8,192 tokens: 198 us with an address a piece, 180 through registers with
// a uniform one, 171 directly).
//
// A direct load puts lane i's piece at sixteen i bytes: the piece at place c
// of a row is the row's chunk c ^ f(row), the permutation of TileShape::along.
template <class V, int DP, int kTokens, int kThreads>
struct RowLoader {
  using T = TileShape<V, DP>;
  static constexpr int kPieces = kTokens * T::kChunks;
  static constexpr int kPer = (kPieces + kThreads - 1) / kThreads;
  static constexpr int kRows = kThreads / T::kChunks;  // between a thread's pieces
  static constexpr bool kEven = T::kUsed == T::kChunks && kPieces % kThreads == 0;
  // the permutation repeats after sixteen rows
  static constexpr int kKinds = kRows % 16 == 0 ? 1 : 2;
  static_assert(!kEven || kRows * kKinds % 16 == 0, "a thread's pieces are of one or two kinds");
  uint32_t offset[kKinds];  // of the thread's pieces from the first row it has of a kind
  int64_t step;      // bytes between rows
  bool plain;        // whole rows within 2 GB of each other (uniform)

  __device__ __forceinline__ void start(int64_t stride, int dim) {
    step = stride * T::kSize;
    plain = kEven && dim == DP && step >= 0 && step * kTokens < (int64_t{1} << 31);
    const int row = threadIdx.x / T::kChunks;
#pragma unroll
    for (int kind = 0; kind < kKinds; ++kind)
      offset[kind] = static_cast<uint32_t>(row) * static_cast<uint32_t>(step) +
                     T::logical(row + kind * kRows, threadIdx.x % T::kChunks) * 16;
  }
  // kTokens rows from `first` on, all there, to `tile`: done when the loads
  // in flight are.
  __device__ __forceinline__ void direct(const void *first, char *tile) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const char *from = static_cast<const char *>(first) + r * kRows * step + offset[r % kKinds];
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void *)(from),
          (__attribute__((address_space(3))) void *)(tile + (r * kThreads + wave * kWave) * 16), 16, 0, 0);
    }
  }
  // Rows one by one: `row_at(row)` gives a row's address, null for zeros.
  template <class RowAt>
  __device__ __forceinline__ void each(const RowAt &row_at, int dim, char *tile) const {
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int at = threadIdx.x + r * kThreads, row = at / T::kChunks, chunk = at % T::kChunks;
      if (row >= kTokens || chunk >= T::kUsed) continue;
      const void *from = row_at(row);
      v4u piece = {0, 0, 0, 0};
      if (from != nullptr && chunk * 16 < dim * T::kSize)
        piece = *reinterpret_cast<const v4u *>(static_cast<const char *>(from) + chunk * 16);
      *reinterpret_cast<v4u *>(tile + T::along(row, chunk)) = piece;
    }
  }
};

// A barrier after which every wave's direct loads are in LDS.
__device__ __forceinline__ void sync_tiles() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0); the other counters as they are
  __syncthreads();
}

// The lane 32 away.
__device__ __forceinline__ float other_half(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t other = (threadIdx.x % kWave) < 32 ? r[1] : r[0];
  return __builtin_bit_cast(float, other);
}

// Workgroups (2^31 - 1 at most, as checked before a launch; divisions of 64 bits
// would cost a short block a tenth) go to the 8 XCDs in turn; this gives each XCD one contiguous
// part of the work, whose neighbours share what they read through its L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t id, uint32_t n) {
  const uint32_t per = n / 8, rest = n % 8, x = id % 8, at = id / 8;
  return x * per + (x < rest ? x : rest) + at;
}

// How equal blocks of work are cut over `slots` workgroups that run at once:
// the first `whole` run as they are, each of the rest in `parts`, so that the
// last round does not leave most of the chip waiting for a few blocks.
struct TailCut {
  int64_t whole, rest;
  int32_t parts;
  __host__ __device__ __forceinline__ int64_t items() const { return whole + rest * parts; }
};

// The launch that joins one part a slot takes 5 to 8 us, a tile 1 to 3, the most in
// float32: 128 bfloat16 key blocks are not worth two parts each (a backward pass of
// 2 x 1,000 tokens of 8 heads of 128: 92 us, 80 whole).  For float32 it says little: 45
// key blocks (3 x 517 tokens of 6 heads of 64) take 73 us in five parts, and 70 with
// joining held to cost nothing.
inline double join_cost(bool float32) { return float32 ? 2.0 : 6.0; }

// Costs in tiles, of which a block has `tiles`: a part more for its start and
// its sums, `join` as above by their number; a part has two at least.
inline TailCut cut_tail(int64_t blocks, int64_t slots, int64_t tiles, double join) {
  constexpr double kPart = 0.75;
  const int64_t rest = blocks % slots;
  TailCut cut{blocks, 0, 1};
  double best = static_cast<double>(tiles);
  for (int64_t p = 2; 2 * p <= tiles && p <= 16 && rest > 0; ++p) {
    const double rounds = static_cast<double>((rest * p + slots - 1) / slots);
    const double cost = rounds * (static_cast<double>((tiles + p - 1) / p) + kPart) +
                        join * (0.5 + 0.5 * static_cast<double>(rest * p) / slots);
    if (cost < best) {
      best = cost;
      cut = TailCut{blocks - rest, rest, static_cast<int32_t>(p)};
    }
  }
  return cut;
}

// Which block and part of it a workgroup takes; the whole ones in XCD order.
struct CutItem {
  uint32_t block;
  int32_t part, parts;
  int64_t slot;  // of its sums in scratch, -1 for a whole block
  __device__ __forceinline__ CutItem(const TailCut &cut, uint32_t id) {
    const uint32_t whole = static_cast<uint32_t>(cut.whole);
    if (id < whole) {
      block = xcd_order(id, whole);
      part = 0;
      parts = 1;
      slot = -1;
    } else {
      const uint32_t at = id - whole, of = static_cast<uint32_t>(cut.parts);
      slot = at;
      block = whole + at / of;
      part = static_cast<int32_t>(at % of);
      parts = cut.parts;
    }
  }
  // The part's first tile of `tiles` (2^26 at most, in 16 parts at most).
  __device__ __forceinline__ int32_t first(int32_t tiles, int32_t more = 0) const {
    return parts == 1 ? tiles * more : tiles * (part + more) / parts;
  }
};

}  // namespace msx
