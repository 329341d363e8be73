// distill.h - C++ primitive layer of distillation from a teacher's top logits.
#pragma once

#include "common/array_view.h"
#include "msx_sparse.h"

namespace msx {

// logits (n_rows, n_cols) with adjacent columns; the teacher's CSR buffers;
// weights (n_rows) float32, or one for all rows, or null.
msx_distill_desc distill_desc(const ArrayView &logits, const ArrayView &data,
                              const ArrayView &indices, const ArrayView &indptr,
                              const ArrayView *weights, double temperature);

// losses (n_rows) float32; lse (n_rows) float32, or null.
void distill_loss(const msx_distill_desc &desc, const ArrayView &losses, float *lse,
                  const ExecContext &ctx);
// grad as logits, contiguous; lse from distill_loss.
void distill_grad(const msx_distill_desc &desc, const float *lse, const ArrayView &grad,
                  const ExecContext &ctx);
void distill_loss_grad(const msx_distill_desc &desc, const ArrayView &losses, float *lse,
                       const ArrayView &grad, const ExecContext &ctx);

}  // namespace msx
