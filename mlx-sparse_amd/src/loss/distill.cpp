// distill.cpp - C++ primitive layer of distillation: checks the operands,
// then calls the C ABI (device operands: the HIP entry point on ctx.stream;
// host operands: the native CPU entry point).
#include "loss/distill.h"

#include <string>

#include "common/validate.h"

namespace msx {
namespace {

void require_real(const ArrayView &a, const std::string &name) {
  if (a.dtype != DType::Float32 && a.dtype != DType::Float16 && a.dtype != DType::BFloat16)
    throw std::invalid_argument(name + " must have dtype float32, float16 or bfloat16, got " +
                                a.dtype_name + ".");
}

}  // namespace

msx_distill_desc distill_desc(const ArrayView &logits, const ArrayView &data,
                              const ArrayView &indices, const ArrayView &indptr,
                              const ArrayView *weights, double temperature) {
  require_rank(logits, 2, "distill logits");
  require_real(logits, "distill logits");
  require_rank(data, 1, "distill teacher data");
  require_real(data, "distill teacher data");
  require_rank(indices, 1, "distill teacher indices");
  require_rank(indptr, 1, "distill teacher indptr");
  require_same_index_dtype(indices, indptr, "distill teacher indices", "distill teacher indptr");
  require_size(indptr, logits.shape[0] + 1, "distill teacher indptr");
  require_size(indices, data.size(), "distill teacher indices");
  for (const ArrayView *a : {&data, &indices, &indptr})
    require_contiguous(*a, "distill teacher buffer");
  if (logits.shape[1] > 1 && logits.strides[1] != 1)
    throw std::invalid_argument("distill logits must have adjacent columns.");
  require_same_device({&logits, &data, &indices, &indptr}, "distill");
  msx_distill_desc d{};
  d.vtype = to_vtype(logits.dtype);
  d.teacher_vtype = to_vtype(data.dtype);
  d.itype = to_itype(indices.dtype);
  d.n_rows = logits.shape[0];
  d.n_cols = logits.shape[1];
  d.nnz = data.size();
  // a matrix of one row has no stride of its own
  d.ld = logits.shape[0] > 1 ? logits.strides[0] : logits.shape[1];
  d.temperature = temperature;
  d.logits = logits.ptr;
  d.data = data.ptr;
  d.indices = indices.ptr;
  d.indptr = indptr.ptr;
  if (weights != nullptr) {
    if (weights->dtype != DType::Float32)
      throw std::invalid_argument("distill weights must have dtype float32, got " +
                                  weights->dtype_name + ".");
    require_rank(*weights, 1, "distill weights");
    require_size(*weights, logits.shape[0], "distill weights");
    require_same_device({&logits, weights}, "distill");
    d.weights = static_cast<const float *>(weights->ptr);
    d.weights_stride = weights->strides[0];
  }
  return d;
}

void distill_loss(const msx_distill_desc &desc, const ArrayView &losses, float *lse,
                  const ExecContext &ctx) {
  check_status(losses.device >= 0
                   ? msx_distill_loss(&desc, static_cast<float *>(losses.ptr), lse, ctx.stream)
                   : msx_distill_loss_cpu(&desc, static_cast<float *>(losses.ptr), lse,
                                          ctx.n_threads),
               "distill_loss");
}

void distill_grad(const msx_distill_desc &desc, const float *lse, const ArrayView &grad,
                  const ExecContext &ctx) {
  require_contiguous(grad, "distill_grad output");
  check_status(grad.device >= 0
                   ? msx_distill_grad(&desc, lse, grad.ptr, desc.n_cols, ctx.stream)
                   : msx_distill_grad_cpu(&desc, lse, grad.ptr, desc.n_cols, ctx.n_threads),
               "distill_grad");
}

void distill_loss_grad(const msx_distill_desc &desc, const ArrayView &losses, float *lse,
                       const ArrayView &grad, const ExecContext &ctx) {
  require_contiguous(grad, "distill_loss_grad output");
  if (grad.device < 0) {  // the host path is two passes in any case
    distill_loss(desc, losses, lse, ctx);
    distill_grad(desc, lse, grad, ctx);
    return;
  }
  check_status(msx_distill_loss_grad(&desc, static_cast<float *>(losses.ptr), grad.ptr,
                                     desc.n_cols, ctx.stream),
               "distill_loss_grad");
}

}  // namespace msx
