// bindings_operators.cpp - window attention and distillation in the Python
// module: operands read in place as torch tensors, their derivatives as torch
// autograd nodes.
//
// The `*_plain` entry points take calls whose operands need nothing done to
// them (tensors on the selected device, of one dtype, adjacent values, shapes
// that fit) and return None for any other, whose errors and conversions are
// Python's: checked there, a small call spent as long on its operands as on
// its kernels.  Their backward passes run without the interpreter.
#include "bindings_operators.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "attention/window_attention.h"
#include "bindings_operands.h"
#include "loss/distill.h"
#include "msx_sparse.h"

namespace py = pybind11;
using msx::aligned_rows;
using msx::ArrayView;
using msx::direct;
using msx::DType;
using msx::for_tiles;
using msx::kStepDim;
using msx::kTilesDim;
using msx::made_direct;
using msx::new_tensor;
using msx::on_device;
using msx::optional_tensor;
using msx::OptionalView;
using msx::present;
using msx::real_type;
using msx::require_writable;
using msx::run_op;
using msx::tensor_of;
using msx::usable;
using msx::usable_counts;
using msx::view_of;
using msx::wrap;
using msx::written;
using at::Tensor;

namespace {

// The head dimension that those kernels take for `t`'s: whole sixteen bytes, as
// long as zeros are a third of it at most.
int64_t padded_dim(const Tensor &t) {
  const int64_t dim = t.size(-1), per = 16 / static_cast<int64_t>(t.element_size());
  const int64_t padded = (dim + per - 1) / per * per;
  return t.is_cuda() && padded <= kTilesDim && 2 * padded <= 3 * dim ? padded : dim;
}
// An operand of attention, with zeros beyond its heads' values (scores and
// gradients do not see them) or at an address where either is all it lacks.
Tensor attention_operand(const Tensor &t, int64_t padded) {
  return padded == t.size(-1) ? for_tiles(t, kTilesDim)
                              : at::constant_pad_nd(t, {0, padded - t.size(-1)});
}
Tensor without_padding(const Tensor &t, int64_t dim) {
  return t.size(-1) == dim ? t : t.narrow(-1, 0, dim).contiguous();
}

struct Pattern {
  int64_t window, sinks;
  double scale;
};

struct Attended {
  Tensor out, lse, low;  // low: of 16-bit outputs, what rounding left of them
};

// With `with_lse` what the backward pass reads: lse and low.
Attended attention(const Tensor &q_in, const Tensor &k_in, const Tensor &v_in,
                   const Tensor &lengths_t, Pattern p, bool with_lse) {
  const int64_t dim = padded_dim(q_in);
  const Tensor q_t = attention_operand(q_in, dim), k_t = attention_operand(k_in, dim),
               v_t = attention_operand(v_in, dim);
  const ArrayView q = view_of(q_t), k = view_of(k_t), v = view_of(v_t);
  const OptionalView lengths(lengths_t);
  auto desc = msx::window_attention_desc(q, k, v, lengths.get, p.window, p.sinks, p.scale);
  const Tensor out = new_tensor(q_t, {desc.batch, desc.lq, desc.heads, desc.dim}, q_t.scalar_type());
  Tensor lse, low;
  if (with_lse) lse = new_tensor(q_t, {desc.batch, desc.heads, desc.lq}, at::kFloat);
  if (with_lse && q_t.scalar_type() != at::kFloat) {
    low = new_tensor(q_t, {desc.batch, desc.heads, (desc.lq + 31) / 32 * 32, (desc.dim + 7) / 8 * 8},
                     q_t.scalar_type());
    desc.out_low = low.data_ptr();
  }
  const ArrayView vo = view_of(out);
  float *l = with_lse ? lse.data_ptr<float>() : nullptr;
  msx::ExecContext ctx = msx::context_for(q, 0);
  Tensor scratch;
  if (q.device >= 0) scratch = msx::scratch_for(ctx, q_t, msx_window_attention_scratch(&desc));
  run_op(q, [&] { msx::window_attention(desc, vo, l, ctx); });
  return {without_padding(out, q_in.size(-1)), lse, low};
}

std::tuple<Tensor, Tensor, Tensor> attention_gradients(const Tensor &q_in, const Tensor &k_in,
                                                       const Tensor &v_in, const Tensor &lengths_t,
                                                       const Tensor &out_in, const Tensor &lse_t,
                                                       const Tensor &low_t, const Tensor &grad_in,
                                                       Pattern p) {
  const int64_t dim = padded_dim(q_in);
  const Tensor q_t = attention_operand(q_in, dim), k_t = attention_operand(k_in, dim),
               v_t = attention_operand(v_in, dim), out_t = attention_operand(out_in, dim),
               grad_t = attention_operand(grad_in, dim);
  const ArrayView q = view_of(q_t), k = view_of(k_t), v = view_of(v_t), out = view_of(out_t),
                  lse = view_of(lse_t), grad = view_of(grad_t);
  const OptionalView lengths(lengths_t);
  auto desc = msx::window_attention_desc(q, k, v, lengths.get, p.window, p.sinks, p.scale);
  if (low_t.defined()) {
    const ArrayView low = view_of(low_t);
    msx::require_size(low, desc.batch * desc.heads * ((desc.lq + 31) / 32 * 32) * ((desc.dim + 7) / 8 * 8),
                      "window_attention_backward low");
    msx::require_contiguous(low, "window_attention_backward low");
    msx::require_same_device({&q, &low}, "window_attention_backward");
    if (low.dtype != q.dtype || q.dtype == DType::Float32)
      throw std::invalid_argument("window_attention_backward low must have the queries' 16-bit dtype.");
    desc.out_low = low.ptr;
  }
  if (lse.dtype != DType::Float32)
    throw std::invalid_argument("window_attention_backward lse must have dtype float32.");
  msx::require_size(lse, desc.batch * desc.heads * desc.lq, "window_attention_backward lse");
  msx::require_contiguous(lse, "window_attention_backward lse");
  msx::require_same_device({&q, &out, &lse, &grad}, "window_attention_backward");
  const at::ScalarType type = q_t.scalar_type();
  const Tensor dq = new_tensor(q_t, {desc.batch, desc.lq, desc.heads, desc.dim}, type);
  const Tensor dk = new_tensor(q_t, {desc.batch, desc.lk, desc.kv_heads, desc.dim}, type);
  const Tensor dv = new_tensor(q_t, {desc.batch, desc.lk, desc.kv_heads, desc.dim}, type);
  const ArrayView vq = view_of(dq), vk = view_of(dk), vv = view_of(dv);
  msx::ExecContext ctx = msx::context_for(q, 0);
  Tensor scratch;
  if (q.device >= 0)
    scratch = msx::scratch_for(ctx, q_t, msx_window_attention_backward_scratch(&desc));
  run_op(q, [&] {
    msx::window_attention_backward(desc, out, static_cast<const float *>(lse.ptr), grad, vq, vk,
                                   vv, ctx);
  });
  const int64_t given = q_in.size(-1);
  return {without_padding(dq, given), without_padding(dk, given), without_padding(dv, given)};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The gradients of a node whose own graph is asked for (create_graph): first
// derivatives, and an error where theirs are used.
struct AttentionGradients : torch::autograd::Function<AttentionGradients> {
  static variable_list forward(AutogradContext *, Tensor q, Tensor k, Tensor v,
                               std::optional<Tensor> lengths, Tensor out, Tensor lse,
                               std::optional<Tensor> low, Tensor grad, int64_t window, int64_t sinks, double scale) {
    const auto [dq, dk, dv] = attention_gradients(q, k, v, lengths.value_or(Tensor()), out, lse,
                                                  low.value_or(Tensor()), grad, {window, sinks, scale});
    return {dq, dk, dv};
  }
  static variable_list backward(AutogradContext *, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(
        false, "second-order derivatives of window_attention are not supported.");
  }
};

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext *ctx, Tensor q, Tensor k, Tensor v,
                        std::optional<Tensor> lengths_o, int64_t window, int64_t sinks,
                        double scale) {
    const Tensor lengths = lengths_o.value_or(Tensor());
    const auto [out, lse, low] = attention(q, k, v, lengths, {window, sinks, scale}, true);
    ctx->save_for_backward({q, k, v, lengths, out, lse, low});
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list result(7);
    if (!grads[0].defined()) return result;
    const variable_list s = ctx->get_saved_variables();
    const Pattern p{ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt(),
                    ctx->saved_data["scale"].toDouble()};
    const Tensor grad = made_direct(grads[0]);
    if (at::GradMode::is_enabled()) {
      const variable_list got = AttentionGradients::apply(s[0], s[1], s[2], present(s[3]), s[4],
                                                          s[5], present(s[6]), grad, p.window, p.sinks, p.scale);
      std::copy(got.begin(), got.end(), result.begin());
    } else {
      std::tie(result[0], result[1], result[2]) =
          attention_gradients(s[0], s[1], s[2], s[3], s[4], s[5], s[6], grad, p);
    }
    return result;
  }
};

// A span given as plain integers in range.
bool plain_span(py::handle window, py::handle sinks, Pattern &p) {
  if (!PyLong_CheckExact(window.ptr()) || !PyLong_CheckExact(sinks.ptr())) return false;
  int over_w = 0, over_s = 0;
  p.window = PyLong_AsLongLongAndOverflow(window.ptr(), &over_w);
  p.sinks = PyLong_AsLongLongAndOverflow(sinks.ptr(), &over_s);
  // 2^40 at most, to which the checks in Python lower wider ones
  return !over_w && !over_s && p.window >= 1 && p.sinks >= 0 && p.window <= (int64_t{1} << 40) &&
         p.sinks <= (int64_t{1} << 40);
}

bool plain_scale(py::handle scale, int64_t dim, Pattern &p) {
  if (scale.is_none()) p.scale = 1.0 / std::sqrt(static_cast<double>(dim));
  else if (PyFloat_CheckExact(scale.ptr())) p.scale = PyFloat_AS_DOUBLE(scale.ptr());
  else return false;
  return true;
}

bool plain_heads(int64_t heads, int64_t kv_heads, int64_t dim) {
  return kv_heads >= 1 && heads >= 1 && heads % kv_heads == 0 && dim >= 1 && dim <= 256;
}

py::object window_attention_plain(py::handle q_o, py::handle k_o, py::handle v_o,
                                  py::handle lengths_o, py::handle window, py::handle sinks,
                                  py::handle scale, int64_t device) {
  for (py::handle h : {q_o, k_o, v_o})
    if (!THPVariable_Check(h.ptr())) return py::none();
  if (!lengths_o.is_none() && !THPVariable_Check(lengths_o.ptr())) return py::none();
  const Tensor &q = tensor_of(q_o), &k = tensor_of(k_o), &v = tensor_of(v_o);
  Pattern p;
  if (q.dim() != 4 || k.dim() != 4 || v.sizes() != k.sizes() || q.size(0) != k.size(0) ||
      q.size(3) != k.size(3) || !plain_heads(q.size(2), k.size(2), q.size(3)) ||
      !plain_span(window, sinks, p) || !plain_scale(scale, q.size(3), p))
    return py::none();
  const at::ScalarType type = q.scalar_type();
  const Tensor lengths = optional_tensor(lengths_o);
  if (!real_type(type) || !usable(q, type, device) || !usable(k, type, device) ||
      !usable(v, type, device) || (lengths.defined() && !usable_counts(lengths, q.size(0), device)))
    return py::none();
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return wrap(Attention::apply(q, k, v, present(lengths), p.window, p.sinks, p.scale));
  return wrap(attention(q, k, v, lengths, p, false).out);
}

py::tuple window_attention(py::handle q, py::handle k, py::handle v, py::handle lengths,
                           int64_t window, int64_t sinks, double scale, bool with_lse) {
  const auto [out, lse, low] = attention(tensor_of(q), tensor_of(k), tensor_of(v),
                                         optional_tensor(lengths), {window, sinks, scale}, with_lse);
  return py::make_tuple(wrap(out), wrap(lse), wrap(low));
}

py::tuple window_attention_backward(py::handle q, py::handle k, py::handle v, py::handle lengths,
                                    py::handle out, py::handle lse, py::handle low,
                                    py::handle grad, int64_t window, int64_t sinks, double scale) {
  const auto [dq, dk, dv] =
      attention_gradients(tensor_of(q), tensor_of(k), tensor_of(v), optional_tensor(lengths),
                          tensor_of(out), tensor_of(lse), optional_tensor(low), tensor_of(grad),
                          {window, sinks, scale});
  return py::make_tuple(wrap(dq), wrap(dk), wrap(dv));
}

// ---------------------------------------------------------------------------
// Single-token step.

Tensor step(const Tensor &q_in, const Tensor &k_in, const Tensor &v_in, const Tensor &ck_t,
            const Tensor &cv_t, const Tensor &lengths_t, Pattern p) {
  // (caches are written in place, so none is copied)
  const bool caches = aligned_rows(ck_t) && aligned_rows(cv_t);
  const Tensor q_t = caches ? for_tiles(q_in, kStepDim) : q_in,
               k_t = caches ? for_tiles(k_in, kStepDim) : k_in,
               v_t = caches ? for_tiles(v_in, kStepDim) : v_in;
  const ArrayView q = view_of(q_t), k = view_of(k_t), v = view_of(v_t), ck = view_of(ck_t),
                  cv = view_of(cv_t), lengths = view_of(lengths_t);
  require_writable(ck_t, "window_attention_step cache_k");
  require_writable(cv_t, "window_attention_step cache_v");
  const auto desc = msx::window_step_desc(q, k, v, ck, cv, lengths, p.window, p.sinks, p.scale);
  const Tensor out = new_tensor(q_t, {desc.batch, desc.heads, desc.dim}, q_t.scalar_type());
  const ArrayView vo = view_of(out);
  msx::ExecContext ctx = msx::context_for(q, 0);
  Tensor scratch;
  if (q.device >= 0) scratch = msx::scratch_for(ctx, q_t, msx_window_attention_step_scratch(&desc));
  run_op(q, [&] { msx::window_attention_step(desc, vo, ctx); });
  written(ck_t);
  written(cv_t);
  return out;
}

py::object window_attention_step_plain(py::handle q_o, py::handle k_o, py::handle v_o,
                                       py::handle ck_o, py::handle cv_o, py::handle lengths_o,
                                       py::handle window, py::handle sinks, py::handle scale,
                                       int64_t device) {
  for (py::handle h : {q_o, k_o, v_o, ck_o, cv_o, lengths_o})
    if (!THPVariable_Check(h.ptr())) return py::none();
  const Tensor &q = tensor_of(q_o), &k = tensor_of(k_o), &v = tensor_of(v_o), &ck = tensor_of(ck_o),
               &cv = tensor_of(cv_o), &lengths = tensor_of(lengths_o);
  Pattern p;
  if (q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() || ck.dim() != 4 ||
      cv.sizes() != ck.sizes() || !plain_heads(q.size(1), k.size(1), q.size(2)) ||
      !plain_span(window, sinks, p) || !plain_scale(scale, q.size(2), p) ||
      p.window + p.sinks > ck.size(1))
    return py::none();
  const at::ScalarType type = q.scalar_type();
  if (!real_type(type) || !usable_counts(lengths, q.size(0), device) || ck.requires_grad() ||
      cv.requires_grad())
    return py::none();
  for (const Tensor *t : {&q, &k, &v, &ck, &cv})
    if (!usable(*t, type, device)) return py::none();
  return wrap(step(q, k, v, ck, cv, lengths, p));
}

py::object window_attention_step(py::handle q, py::handle k, py::handle v, py::handle ck,
                                 py::handle cv, py::handle lengths, int64_t window, int64_t sinks,
                                 double scale) {
  return wrap(step(tensor_of(q), tensor_of(k), tensor_of(v), tensor_of(ck), tensor_of(cv),
                   tensor_of(lengths), {window, sinks, scale}));
}

void window_cache_store(py::handle k_o, py::handle v_o, py::handle cache_k_o, py::handle cache_v_o,
                        py::handle starts_o, py::handle lengths_o, int64_t sinks) {
  const ArrayView k = view_of(k_o), v = view_of(v_o), ck = view_of(cache_k_o),
                  cv = view_of(cache_v_o);
  const OptionalView starts(optional_tensor(starts_o)), lengths(optional_tensor(lengths_o));
  require_writable(tensor_of(cache_k_o), "window_cache_store cache_k");
  require_writable(tensor_of(cache_v_o), "window_cache_store cache_v");
  const msx::ExecContext ctx = msx::context_for(k, 0);
  run_op(k, [&] { msx::window_cache_store(k, v, ck, cv, starts.get, lengths.get, sinks, ctx); });
  written(tensor_of(cache_k_o));
  written(tensor_of(cache_v_o));
}

// ---------------------------------------------------------------------------
// Distillation.

struct Teacher {
  Tensor data, indices, indptr;
};

std::tuple<Tensor, Tensor> losses_of(const Tensor &logits_t, const Teacher &t, double temperature,
                                     bool with_lse) {
  const ArrayView logits = view_of(logits_t);
  const auto desc = msx::distill_desc(logits, view_of(t.data), view_of(t.indices),
                                      view_of(t.indptr), nullptr, temperature);
  const Tensor losses = new_tensor(logits_t, {desc.n_rows}, at::kFloat);
  Tensor lse;
  if (with_lse) lse = new_tensor(logits_t, {desc.n_rows}, at::kFloat);
  const ArrayView vl = view_of(losses);
  float *l = with_lse ? lse.data_ptr<float>() : nullptr;
  const msx::ExecContext ctx = msx::context_for(logits, 0);
  run_op(logits, [&] { msx::distill_loss(desc, vl, l, ctx); });
  return {losses, lse};
}

Tensor gradient_of(const Tensor &logits_t, const Teacher &t, const Tensor &weights_t,
                   const Tensor &lse_t, double temperature) {
  const ArrayView logits = view_of(logits_t), lse = view_of(lse_t);
  const OptionalView weights(weights_t);
  const auto desc = msx::distill_desc(logits, view_of(t.data), view_of(t.indices),
                                      view_of(t.indptr), weights.get, temperature);
  if (lse.dtype != DType::Float32)
    throw std::invalid_argument("distill_grad lse must have dtype float32.");
  msx::require_size(lse, desc.n_rows, "distill_grad lse");
  msx::require_contiguous(lse, "distill_grad lse");
  msx::require_same_device({&logits, &lse}, "distill_grad");
  const Tensor grad = new_tensor(logits_t, {desc.n_rows, desc.n_cols}, logits_t.scalar_type());
  const ArrayView vg = view_of(grad);
  const msx::ExecContext ctx = msx::context_for(logits, 0);
  run_op(logits, [&] { msx::distill_grad(desc, static_cast<const float *>(lse.ptr), vg, ctx); });
  return grad;
}

std::tuple<Tensor, Tensor> losses_and_gradient(const Tensor &logits_t, const Teacher &t,
                                               const Tensor &weights_t, double temperature) {
  const ArrayView logits = view_of(logits_t);
  const OptionalView weights(weights_t);
  const auto desc = msx::distill_desc(logits, view_of(t.data), view_of(t.indices),
                                      view_of(t.indptr), weights.get, temperature);
  const Tensor losses = new_tensor(logits_t, {desc.n_rows}, at::kFloat);
  const Tensor grad = new_tensor(logits_t, {desc.n_rows, desc.n_cols}, logits_t.scalar_type());
  Tensor lse;
  if (logits.device < 0) lse = new_tensor(logits_t, {desc.n_rows}, at::kFloat);
  const ArrayView vl = view_of(losses), vg = view_of(grad);
  float *l = lse.defined() ? lse.data_ptr<float>() : nullptr;
  const msx::ExecContext ctx = msx::context_for(logits, 0);
  run_op(logits, [&] { msx::distill_loss_grad(desc, vl, l, vg, ctx); });
  return {losses, grad};
}

struct DistillGradient : torch::autograd::Function<DistillGradient> {
  static Tensor forward(AutogradContext *, Tensor logits, Tensor data, Tensor indices,
                        Tensor indptr, Tensor weights, Tensor lse, double temperature) {
    return gradient_of(logits, {data, indices, indptr}, weights, lse, temperature);
  }
  static variable_list backward(AutogradContext *, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false,
                                "second-order derivatives of distill_loss are not supported.");
  }
};

struct Distill : torch::autograd::Function<Distill> {
  static Tensor forward(AutogradContext *ctx, Tensor logits, Tensor data, Tensor indices,
                        Tensor indptr, double temperature) {
    const auto [losses, lse] = losses_of(logits, {data, indices, indptr}, temperature, true);
    ctx->save_for_backward({logits, data, indices, indptr, lse});
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    return losses;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list result(5);
    if (!grads[0].defined()) return result;
    const variable_list s = ctx->get_saved_variables();
    const double t = ctx->saved_data["temperature"].toDouble();
    const Tensor weights = grads[0].is_neg() ? grads[0].resolve_neg() : grads[0];
    result[0] = at::GradMode::is_enabled()
                    ? DistillGradient::apply(s[0], s[1], s[2], s[3], weights, s[4], t)
                    : gradient_of(s[0], {s[1], s[2], s[3]}, weights, s[4], t);
    return result;
  }
};

bool direct_rows(const Tensor &t) {
  return direct(t) && (t.size(0) < 2 || t.stride(0) >= t.size(1));
}

// The operands of a distillation of rank-2 logits, where nothing is to be
// done to them.
bool plain_distill(py::handle logits_o, py::handle data_o, py::handle indices_o,
                   py::handle indptr_o, int64_t n_rows, int64_t n_cols, int64_t device) {
  for (py::handle h : {logits_o, data_o, indices_o, indptr_o})
    if (!THPVariable_Check(h.ptr())) return false;
  const Tensor &z = tensor_of(logits_o), &data = tensor_of(data_o), &indices = tensor_of(indices_o),
               &indptr = tensor_of(indptr_o);
  const auto index = indices.scalar_type();
  return z.dim() == 2 && z.size(0) == n_rows && z.size(1) == n_cols && real_type(z.scalar_type()) &&
         on_device(z, device) && direct_rows(z) && data.dim() == 1 &&
         real_type(data.scalar_type()) && !data.requires_grad() && !data.is_neg() &&
         (index == at::kInt || index == at::kLong) && indptr.scalar_type() == index &&
         indices.dim() == 1 && indices.size(0) == data.size(0) && indptr.dim() == 1 &&
         indptr.size(0) == n_rows + 1 && on_device(data, device) && on_device(indices, device) &&
         on_device(indptr, device) && data.is_contiguous() && indices.is_contiguous() &&
         indptr.is_contiguous();
}

bool plain_temperature(py::handle o, double &t) {
  if (!PyFloat_CheckExact(o.ptr())) return false;
  t = PyFloat_AS_DOUBLE(o.ptr());
  return t > 0.0 && std::isnormal(static_cast<float>(t * t));
}

py::object distill_loss_plain(py::handle logits, py::handle data, py::handle indices,
                              py::handle indptr, int64_t n_rows, int64_t n_cols,
                              py::handle temperature, int64_t device) {
  double t = 0.0;
  if (!plain_temperature(temperature, t) ||
      !plain_distill(logits, data, indices, indptr, n_rows, n_cols, device))
    return py::none();
  const Tensor &z = tensor_of(logits);
  const Teacher teacher{tensor_of(data), tensor_of(indices), tensor_of(indptr)};
  if (at::GradMode::is_enabled() && z.requires_grad())
    return wrap(Distill::apply(z, teacher.data, teacher.indices, teacher.indptr, t));
  return wrap(std::get<0>(losses_of(z, teacher, t, false)));
}

py::object distill_loss_grad_plain(py::handle logits, py::handle data, py::handle indices,
                                   py::handle indptr, py::handle weights_o, int64_t n_rows,
                                   int64_t n_cols, py::handle temperature, int64_t device) {
  double t = 0.0;
  if (!plain_temperature(temperature, t) ||
      !plain_distill(logits, data, indices, indptr, n_rows, n_cols, device) ||
      (!weights_o.is_none() && !THPVariable_Check(weights_o.ptr())))
    return py::none();
  const Tensor weights = optional_tensor(weights_o);
  if (weights.defined() && (weights.scalar_type() != at::kFloat || weights.dim() != 1 ||
                            weights.size(0) != n_rows || !on_device(weights, device) ||
                            weights.is_neg()))
    return py::none();
  const auto [losses, grad] = losses_and_gradient(
      tensor_of(logits), {tensor_of(data), tensor_of(indices), tensor_of(indptr)}, weights, t);
  return py::make_tuple(wrap(losses), wrap(grad));
}

py::tuple distill_loss(py::handle logits, py::handle data, py::handle indices, py::handle indptr,
                       double temperature, bool with_lse) {
  const auto [losses, lse] =
      losses_of(tensor_of(logits), {tensor_of(data), tensor_of(indices), tensor_of(indptr)},
                temperature, with_lse);
  return py::make_tuple(wrap(losses), wrap(lse));
}

py::object distill_grad(py::handle logits, py::handle data, py::handle indices, py::handle indptr,
                        py::handle weights, py::handle lse, double temperature) {
  return wrap(gradient_of(tensor_of(logits),
                          {tensor_of(data), tensor_of(indices), tensor_of(indptr)},
                          optional_tensor(weights), tensor_of(lse), temperature));
}

py::tuple distill_loss_grad(py::handle logits, py::handle data, py::handle indices,
                            py::handle indptr, py::handle weights, double temperature) {
  const auto [losses, grad] = losses_and_gradient(
      tensor_of(logits), {tensor_of(data), tensor_of(indices), tensor_of(indptr)},
      optional_tensor(weights), temperature);
  return py::make_tuple(wrap(losses), wrap(grad));
}

}  // namespace

void bind_operators(py::module_ &m) {
  m.def("window_attention_plain", &window_attention_plain, py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("lengths"), py::arg("window"), py::arg("sinks"), py::arg("scale"),
        py::arg("device"), "window_attention where nothing is to be done to the operands, else None.");
  m.def("window_attention", &window_attention, py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("lengths"), py::arg("window"), py::arg("sinks"), py::arg("scale"),
        py::arg("with_lse"),
        "(out, lse, low) of attention over the last window and the first sinks keys.");
  m.def("window_attention_backward", &window_attention_backward, py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("lengths"), py::arg("out"), py::arg("lse"), py::arg("low"),
        py::arg("grad"),
        py::arg("window"), py::arg("sinks"), py::arg("scale"),
        "(dq, dk, dv) of window_attention.");
  m.def("window_attention_step_plain", &window_attention_step_plain, py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("cache_k"), py::arg("cache_v"), py::arg("lengths"),
        py::arg("window"), py::arg("sinks"), py::arg("scale"), py::arg("device"),
        "window_attention_step where nothing is to be done to the operands, else None.");
  m.def("window_attention_step", &window_attention_step, py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("cache_k"), py::arg("cache_v"), py::arg("lengths"), py::arg("window"),
        py::arg("sinks"), py::arg("scale"),
        "One token of every sequence: into its ring cache, and its attention over it.");
  m.def("window_cache_store", &window_cache_store, py::arg("k"), py::arg("v"), py::arg("cache_k"),
        py::arg("cache_v"), py::arg("starts"), py::arg("lengths"), py::arg("sinks"),
        "A prompt's keys and values into ring caches.");
  m.def("distill_loss_plain", &distill_loss_plain, py::arg("logits"), py::arg("data"),
        py::arg("indices"), py::arg("indptr"), py::arg("n_rows"), py::arg("n_cols"),
        py::arg("temperature"), py::arg("device"),
        "distill_loss where nothing is to be done to the operands, else None.");
  m.def("distill_loss_grad_plain", &distill_loss_grad_plain, py::arg("logits"), py::arg("data"),
        py::arg("indices"), py::arg("indptr"), py::arg("weights"), py::arg("n_rows"),
        py::arg("n_cols"), py::arg("temperature"), py::arg("device"),
        "distill_value_and_grad where nothing is to be done to the operands, else None.");
  m.def("distill_loss", &distill_loss, py::arg("logits"), py::arg("data"), py::arg("indices"),
        py::arg("indptr"), py::arg("temperature"), py::arg("with_lse"),
        "(losses, lse) of distillation from a CSR teacher's logits.");
  m.def("distill_grad", &distill_grad, py::arg("logits"), py::arg("data"), py::arg("indices"),
        py::arg("indptr"), py::arg("weights"), py::arg("lse"), py::arg("temperature"),
        "Gradient of the weighted losses in the logits.");
  m.def("distill_loss_grad", &distill_loss_grad, py::arg("logits"), py::arg("data"),
        py::arg("indices"), py::arg("indptr"), py::arg("weights"), py::arg("temperature"),
        "(losses, gradient of the weighted losses) in one call.");
}
