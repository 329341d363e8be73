// distill.hip - distillation from a teacher's top logits, the rows of a CSR
// matrix: per-row losses and the gradient in the student's logits.
//
// With z = logits / T, q = softmax(z) over the row and p = softmax(kept / T)
// over the row's kept logits:
//   loss = T^2 sum_r p_r (ln p_r - ln q_r),  ln q_r = z_r - lse
//   grad = weight T (q - p)
// One workgroup a row: a pass over the row for its maximum and the sum of
// exponentials, and for the gradient a second one, over what the first kept in
// registers.  The columns of kept logits are written last, each by the thread
// that holds it, q - p rounded once.
//
// Memory bounds it: the logits read and the gradient written once, 2.1 GB for
// 4,096 rows of 131,072 bfloat16, take 430 us (5.0 TB/s, what a copy reaches, over
// one matrix again and again as over five in turn; 470 with the row read twice), the
// gradient alone 397; 2,000 rows of 50,257 take 71 us (90), 65 of 1,009 float32 6.0.
// The loss alone reads 2,049 rows of 50,001 float16 in 41 us (5.0 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "msx_device.h"
#include "msx_internal.h"
#include "msx_window.h"
#include "msx_window_check.h"
#include "msx_window_mfma.h"

#pragma clang fp contract(fast)

namespace msx {
namespace {

struct DistillArgs {
  int64_t n_cols, ld, ld_grad, nnz;
  const void *logits;
  const void *data, *indices, *indptr;
  int32_t teacher_vtype, index64;
  const float *weights;
  int64_t weights_stride;
  float scale;        // log2(e) / T: scaled logits are kept in base 2
  float temperature;  // T^2 of a loss and T of a gradient come from it

  // A row's first entry, as far as there are any.
  __device__ inline int64_t offset(int64_t r) const {
    const int64_t p = index64 ? static_cast<const int64_t *>(indptr)[r]
                              : static_cast<const int32_t *>(indptr)[r];
    return p < 0 ? 0 : p > nnz ? nnz : p;
  }
  // Column of entry e, or -1 outside the matrix.
  __device__ inline int64_t column(int64_t e) const {
    const int64_t c = index64 ? static_cast<const int64_t *>(indices)[e]
                              : static_cast<const int32_t *>(indices)[e];
    return c < 0 || c >= n_cols ? -1 : c;
  }
  __device__ inline float kept(int64_t e) const {
    if (teacher_vtype == MSX_F32) return static_cast<const float *>(data)[e] * scale;
    const uint16_t bits = static_cast<const uint16_t *>(data)[e];
    return (teacher_vtype == MSX_F16 ? half_bits_to_float(bits) : bf16_bits_to_float(bits)) * scale;
  }
  __device__ inline float weight(int64_t r) const {
    return weights == nullptr ? 1.0f : weights[r * weights_stride];
  }
};

// Maximum and sum of exponentials of what has been seen, base 2.
struct Stat {
  float top, sum;
  __device__ inline float base() const { return top == -INFINITY ? 0.0f : top; }
  __device__ inline float log_sum() const { return base() + log2_fast(sum); }
  template <int N>
  __device__ inline void add(const float (&x)[N]) {
    float t = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) t = fmaxf(t, x[j]);
    if (t > top) {
      sum *= exp2_fast(top - t);
      top = t;
    }
    const float b = base();
#pragma unroll
    for (int j = 0; j < N; ++j) sum += exp2_fast(x[j] - b);
  }
  __device__ inline void merge(Stat o) {
    const float t = fmaxf(top, o.top);
    const float b = t == -INFINITY ? 0.0f : t;
    sum = sum * exp2_fast(top - b) + o.sum * exp2_fast(o.top - b);
    top = t;
  }
  __device__ inline void merge_wave() {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) merge({__shfl_xor(top, d), __shfl_xor(sum, d)});
  }
};

// A row as sixteen-byte pieces at sixteen-byte addresses, and up to seven
// values before and after them, one a thread.
template <class V>
struct RowPieces {
  using S = typename V::Storage;
  static constexpr int kPer = 16 / sizeof(S);
  int64_t n;
  int32_t head;
  int64_t pieces;
  __device__ inline RowPieces(const S *row, int64_t columns) : n(columns) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(S));
    const int lead = off == 0 ? 0 : kPer - off;
    head = static_cast<int32_t>(lead < n ? lead : n);
    pieces = (n - head) / kPer;
  }
  // The column of this thread's single value, or -1.
  __device__ inline int64_t single() const {
    const int64_t tail = head + pieces * kPer, t = threadIdx.x;
    if (t < head) return t;
    return tail + (t - head) < n ? tail + (t - head) : -1;
  }
  __device__ static inline void widen(v4u piece, float scale, float (&x)[kPer]) {
    const v4f values = __builtin_bit_cast(v4f, piece);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kPer == 4) {
        x[j] = values[j] * scale;
      } else {
        x[2 * j] = V::widen(static_cast<uint16_t>(piece[j])) * scale;
        x[2 * j + 1] = V::widen(static_cast<uint16_t>(piece[j] >> 16)) * scale;
      }
    }
  }
};

// q factor of a piece, rounded.
template <class V>
__device__ inline v4u softmax_piece(v4u piece, float scale, float total, float factor) {
  constexpr int kPer = RowPieces<V>::kPer;
  float x[kPer];
  RowPieces<V>::widen(piece, scale, x);
#pragma unroll
  for (int j = 0; j < kPer; ++j) x[j] = exp2_fast(x[j] - total) * factor;
  v4u out;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (kPer == 4)
      out[j] = __builtin_bit_cast(uint32_t, x[j]);
    else
      out[j] = Mfma<V>::pack(x[2 * j], x[2 * j + 1]);
  }
  return out;
}

// A piece to where the gradient's rows lie, which may start elsewhere in
// their sixteen bytes than the logits'.  It is not read again here.
template <class S>
__device__ inline void store_piece(v4u piece, S *to) {
  if (reinterpret_cast<uintptr_t>(to) % 16 == 0) {
    __builtin_nontemporal_store(piece, reinterpret_cast<v4u *>(to));
  } else {
    S v[16 / sizeof(S)];
    __builtin_memcpy(v, &piece, 16);
#pragma unroll
    for (int j = 0; j < static_cast<int>(16 / sizeof(S)); ++j) to[j] = v[j];
  }
}

// Which of a row's kept columns are stored more than once, and their sums of p,
// where the row is out of order (as a teacher's largest logits by value are).
// A bit a column tells whether any is, 128 columns a thread at a time (4,096 rows
// of 131,072 with 1,000 kept by value: 565 us, 550 by column; 3,391 with each
// entry looking through its row); only then sums are made, two columns a thread at a time, of integers: p 2^52, which add up
// the same in any order and are as good as a float32 p down to 2^-28.
template <int kThreads>
struct Columns {
  static constexpr int64_t kMarks = kThreads * 128, kSums = kThreads * 2;
  union {
    uint32_t marks[kThreads * 4];
    unsigned long long sums[kThreads * 2];
  };
  int twice;

  __device__ inline void clear() {
    for (int i = threadIdx.x; i < kThreads * 4; i += kThreads) marks[i] = 0;
    if (threadIdx.x == 0) twice = 0;
  }
  __device__ inline void mark(int64_t c) {
    const uint32_t bit = 1u << (c % 32);
    if (atomicOr(&marks[c / 32], bit) & bit) twice = 1;
  }
  __device__ inline void add(int64_t c, float p) {
    atomicAdd(&sums[c], static_cast<unsigned long long>(p * 0x1p52f));
  }
  __device__ inline float sum(int64_t c) const { return static_cast<float>(sums[c]) * 0x1p-52f; }
};

// kLoss: losses (and lse where asked); kGrad: the gradient, from `lse_in` or
// from the row's own pass.
// kHold: pieces a thread keeps in registers between the two passes.
template <class V, bool kLoss, bool kGrad, int kThreads, int kHold>
__global__ __launch_bounds__(kThreads, kHold > 0 ? 4 : 8) void distill_rows(DistillArgs a, int64_t first_row,
                                                         float *losses, float *lse,
                                                         const float *lse_in,
                                                         typename V::Storage *grad) {
  using S = typename V::Storage;
  using Row = RowPieces<V>;
  constexpr int kPer = Row::kPer, kWaves = kThreads / kWave, kAhead = 4;
  __shared__ Stat kept_lds[kWaves], stat_lds[kWaves];
  __shared__ float part_lds[kWaves];
  __shared__ int ascending_lds[kWaves];
  __shared__ Columns<kGrad ? kThreads : 1> columns_lds;
  const int wave = threadIdx.x / kWave;
  const int64_t row = first_row + blockIdx.x;
  const S *z = static_cast<const S *>(a.logits) + row * a.ld;
  S *g = kGrad ? grad + row * a.ld_grad : nullptr;
  const int64_t begin = a.offset(row), end = a.offset(row + 1);
  const float weight = kGrad ? a.weight(row) : 0.0f;

  // the thread's first kept logit stays at hand; ascending: none is there twice
  Stat kept{-INFINITY, 0.0f};
  int64_t column = -1;
  float mine = -INFINITY, mine_z = 0.0f;
  int ascending = 1;
  for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
    const int64_t c = a.column(e);
    const float t = c >= 0 ? a.kept(e) : -INFINITY;
    kept.add<1>({t});
    if (e + 1 < end && a.column(e + 1) <= c) ascending = 0;
    if (e == begin + threadIdx.x && c >= 0) {
      column = c;
      mine = t;
      mine_z = V::widen(z[c]) * a.scale;
    }
  }
  kept.merge_wave();
  ascending = __all(ascending);

  const Row r(z, a.n_cols);
  const v4u *pieces = reinterpret_cast<const v4u *>(z + r.head);
  const int64_t single = r.single();
  Stat s{-INFINITY, 0.0f};
  v4u held[kHold > 0 ? kHold : 1];
  if (kLoss && begin < end) {
    int64_t c = threadIdx.x;
    if constexpr (kHold > 0) {
      if (r.pieces > 0) {
#pragma unroll
        for (int k = 0; k < kHold; ++k) held[k] = pieces[c + k * kThreads < r.pieces ? c + k * kThreads : r.pieces - 1];
      }
#pragma unroll
      for (int k = 0; k < kHold; ++k)
        if (c + k * kThreads < r.pieces) {
          float x[kPer];
          Row::widen(held[k], a.scale, x);
          s.add<kPer>(x);
        }
      c += kHold * kThreads;
    }
    for (; c + (kAhead - 1) * kThreads < r.pieces; c += kAhead * kThreads) {
      v4u w[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) w[k] = pieces[c + k * kThreads];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        float x[kPer];
        Row::widen(w[k], a.scale, x);
        s.add<kPer>(x);
      }
    }
    for (; c < r.pieces; c += kThreads) {
      float x[kPer];
      Row::widen(pieces[c], a.scale, x);
      s.add<kPer>(x);
    }
    if (single >= 0) s.add<1>({V::widen(z[single]) * a.scale});
    s.merge_wave();
  }
  if (threadIdx.x % kWave == 0) {
    kept_lds[wave] = kept;
    stat_lds[wave] = s;
    ascending_lds[wave] = ascending;
  }
  __syncthreads();
  kept = kept_lds[0];
  s = stat_lds[0];
  ascending = ascending_lds[0];
  for (int w = 1; w < kWaves; ++w) {
    kept.merge(kept_lds[w]);
    if (kLoss) s.merge(stat_lds[w]);
    ascending &= ascending_lds[w];
  }

  const bool target = !(kept.sum == 0.0f);  // NaN is one
  const bool wanted = kGrad && target && weight != 0.0f;
  const float kept_base = kept.base(), kept_inv = 1.0f / kept.sum, kept_lse = kept.log_sum();
  const float total = !kLoss ? (wanted ? lse_in[row] : 0.0f) : s.log_sum();
  if (kLoss) {
    float part = 0.0f;
    if (target)
      for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
        const bool first = e == begin + threadIdx.x;
        const int64_t c = first ? column : a.column(e);
        if (c < 0) continue;
        const float t = first ? mine : a.kept(e);
        const float x = first ? mine_z : V::widen(z[c]) * a.scale;
        const float p = exp2_fast(t - kept_base) * kept_inv;
        if (p != 0.0f) part += p * ((t - kept_lse) - (x - total));
      }
    part = wave_sum(part);
    if (threadIdx.x % kWave == 0) part_lds[wave] = part;
  }
  if (kGrad) {
    if (wanted) {
      const float factor = weight * a.temperature;
      int64_t c = threadIdx.x;
      if constexpr (kHold > 0) {
#pragma unroll
        for (int k = 0; k < kHold; ++k)
          if (c + k * kThreads < r.pieces)
            store_piece(softmax_piece<V>(held[k], a.scale, total, factor),
                        g + r.head + (c + k * kThreads) * kPer);
        c += kHold * kThreads;
      }
      for (; c + (kAhead - 1) * kThreads < r.pieces; c += kAhead * kThreads) {
        v4u w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) w[k] = pieces[c + k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          store_piece(softmax_piece<V>(w[k], a.scale, total, factor),
                      g + r.head + (c + k * kThreads) * kPer);
      }
      for (; c < r.pieces; c += kThreads)
        store_piece(softmax_piece<V>(pieces[c], a.scale, total, factor), g + r.head + c * kPer);
      if (single >= 0)
        g[single] = V::narrow(exp2_fast(V::widen(z[single]) * a.scale - total) * factor);
    } else {
      const v4u none = {0, 0, 0, 0};
      for (int64_t c = threadIdx.x; c < r.pieces; c += kThreads)
        store_piece(none, g + r.head + c * kPer);
      if (single >= 0) g[single] = 0;
    }
  }
  if (kLoss || wanted) __syncthreads();
  if (kLoss && threadIdx.x == 0) {
    float part = part_lds[0];
    for (int w = 1; w < kWaves; ++w) part += part_lds[w];
    losses[row] = target ? part * kLn2 * a.temperature * a.temperature : 0.0f;
    if (lse != nullptr) lse[row] = target ? total : 0.0f;
  }
  if constexpr (kGrad) {
    if (!wanted) return;
    const float factor = weight * a.temperature;
    // fn(column, whether it is the thread's first entry, entry) for those in [low, high)
    const auto each = [&](int64_t low, int64_t high, const auto &fn) {
      for (int64_t e = begin + threadIdx.x; e < end; e += kThreads) {
        const bool first = e == begin + threadIdx.x;
        const int64_t c = first ? column : a.column(e);
        if (c >= low && c < high) fn(c, first, e);
      }
    };
    const auto p_of = [&](bool first, int64_t e) {
      return exp2_fast((first ? mine : a.kept(e)) - kept_base) * kept_inv;
    };
    const auto store = [&](int64_t c, bool first, float p) {
      const float x = first ? mine_z : V::widen(z[c]) * a.scale;
      g[c] = V::narrow((exp2_fast(x - total) - p) * factor);
    };
    // (a teacher that is not finite: every p is NaN, and so is each sum of them)
    if (ascending || !(kept_inv == kept_inv)) {
      each(0, a.n_cols, [&](int64_t c, bool first, int64_t e) { store(c, first, p_of(first, e)); });
      return;
    }
    using C = Columns<kThreads>;
    C &columns = columns_lds;
    for (int64_t low = 0; low < a.n_cols; low += C::kMarks) {
      const int64_t high = min(low + C::kMarks, a.n_cols);
      columns.clear();
      __syncthreads();
      each(low, high, [&](int64_t c, bool, int64_t) { columns.mark(c - low); });
      __syncthreads();
      if (columns.twice == 0) {
        each(low, high, [&](int64_t c, bool first, int64_t e) { store(c, first, p_of(first, e)); });
      } else {
        for (int64_t from = low; from < high; from += C::kSums) {
          const int64_t to = min(from + C::kSums, high);
          __syncthreads();
          columns.sums[threadIdx.x] = columns.sums[threadIdx.x + kThreads] = 0;
          __syncthreads();
          each(from, to, [&](int64_t c, bool first, int64_t e) { columns.add(c - from, p_of(first, e)); });
          __syncthreads();
          each(from, to, [&](int64_t c, bool first, int64_t) { store(c, first, columns.sum(c - from)); });
        }
      }
      __syncthreads();  // before the marks are cleared again
    }
  }
}

DistillArgs args_of(const msx_distill_desc &d, int64_t ld_grad) {
  DistillArgs a{};
  a.n_cols = d.n_cols;
  a.ld = d.ld;
  a.ld_grad = ld_grad;
  a.nnz = d.nnz;
  a.logits = d.logits;
  a.data = d.data;
  a.indices = d.indices;
  a.indptr = d.indptr;
  a.teacher_vtype = d.teacher_vtype;
  a.index64 = d.itype == MSX_I64;
  a.weights = d.weights;
  a.weights_stride = d.weights_stride;
  a.scale = static_cast<float>(1.44269504088896340736 / d.temperature);
  a.temperature = static_cast<float>(d.temperature);
  return a;
}

template <bool kLoss, bool kGrad>
msx_status launch(const msx_distill_desc &d, float *losses, float *lse, const float *lse_in,
                  void *grad, int64_t ld_grad, void *stream) {
  const DistillArgs a = args_of(d, ld_grad);
  const auto run = [&](auto v) {
    using V = decltype(v);
    using S = typename V::Storage;
    const auto st = static_cast<hipStream_t>(stream);
    const int64_t kb = (d.n_cols * static_cast<int64_t>(sizeof(S)) + 1023) / 1024;
    const auto with = [&](auto kernel, unsigned threads) {
      for (int64_t first = 0; first < d.n_rows; first += max_blocks(threads)) {
        const auto blocks = static_cast<unsigned>(std::min(d.n_rows - first, max_blocks(threads)));
        kernel<<<blocks, threads, 0, st>>>(a, first, losses, lse, lse_in, static_cast<S *>(grad));
      }
    };
    if constexpr (kLoss && kGrad) {
      // 256 bytes of the row a thread, in its registers, so that it is read
      // once; what is beyond 256 KB is read twice
      if (kb <= 4) with(distill_rows<V, true, true, 64, 4>, 64);
      else if (kb <= 16) with(distill_rows<V, true, true, 64, 16>, 64);
      else if (kb <= 32) with(distill_rows<V, true, true, 128, 16>, 128);
      else if (kb <= 64) with(distill_rows<V, true, true, 256, 16>, 256);
      else if (kb <= 128) with(distill_rows<V, true, true, 512, 16>, 512);
      else with(distill_rows<V, true, true, 1024, 16>, 1024);
    } else if constexpr (kLoss) {
      // small enough workgroups that one's start and end run beside others'
      // passes (2,049 rows of 50,001 float16: 58 us with 1024, 40 with 512)
      if (kb <= 4) with(distill_rows<V, true, false, 64, 0>, 64);
      else if (kb <= 64) with(distill_rows<V, true, false, 256, 0>, 256);
      else with(distill_rows<V, true, false, 512, 0>, 512);
    } else {
      if (kb <= 4) with(distill_rows<V, false, true, 64, 0>, 64);
      else if (kb <= 64) with(distill_rows<V, false, true, 256, 0>, 256);
      else with(distill_rows<V, false, true, 1024, 0>, 1024);
    }
  };
  switch (d.vtype) {
  case MSX_F32: run(F32{}); break;
  case MSX_F16: run(F16{}); break;
  default: run(BF16{}); break;
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSX_OK : hip_fail(e, "distill");
}

msx_status check_grad(const char *op, const msx_distill_desc *d, const void *grad,
                      int64_t ld_grad) {
  if (d->n_rows > 0 && d->n_cols > 0 && grad == nullptr)
    return fail(MSX_EINVAL, std::string(op) + " grad is NULL.");
  if (ld_grad < d->n_cols)
    return fail(MSX_EINVAL, std::string(op) + " leading dimension must be at least the column count.");
  return MSX_OK;
}

}  // namespace
}  // namespace msx

using namespace msx;

extern "C" msx_status msx_distill_loss(const msx_distill_desc *desc, float *losses, float *lse,
                                       void *stream) {
  clear_error();
  if (msx_status st = check_distill("distill_loss", desc); st != MSX_OK) return st;
  if (desc->n_rows == 0) return MSX_OK;
  if (losses == nullptr) return fail(MSX_EINVAL, "distill_loss losses is NULL.");
  return launch<true, false>(*desc, losses, lse, nullptr, nullptr, 0, stream);
}

extern "C" msx_status msx_distill_grad(const msx_distill_desc *desc, const float *lse, void *grad,
                                       int64_t ld_grad, void *stream) {
  clear_error();
  if (msx_status st = check_distill("distill_grad", desc); st != MSX_OK) return st;
  if (msx_status st = check_grad("distill_grad", desc, grad, ld_grad); st != MSX_OK) return st;
  if (desc->n_rows == 0 || desc->n_cols == 0) return MSX_OK;
  if (lse == nullptr) return fail(MSX_EINVAL, "distill_grad lse is NULL.");
  return launch<false, true>(*desc, nullptr, nullptr, lse, grad, ld_grad, stream);
}

extern "C" msx_status msx_distill_loss_grad(const msx_distill_desc *desc, float *losses,
                                            void *grad, int64_t ld_grad, void *stream) {
  clear_error();
  if (msx_status st = check_distill("distill_loss_grad", desc); st != MSX_OK) return st;
  if (msx_status st = check_grad("distill_loss_grad", desc, grad, ld_grad); st != MSX_OK) return st;
  if (desc->n_rows == 0) return MSX_OK;
  if (losses == nullptr) return fail(MSX_EINVAL, "distill_loss_grad losses is NULL.");
  return launch<true, true>(*desc, losses, nullptr, nullptr, grad, ld_grad, stream);
}
