// bindings_paged.cpp - rotary positions, paged caches and the attention over them in
// the Python module.  As in bindings_operators.cpp the `*_plain` entry points take
// calls whose operands need nothing done to them and return None for any other.
#include "bindings_operators.h"

#include <cmath>
#include <optional>
#include <string>

#include "attention/paged_attention.h"
#include "bindings_operands.h"
#include "msx_sparse.h"

namespace py = pybind11;
using namespace msx;

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Rotation {
  Tensor turns;  // undefined: none
  int64_t dim;
  bool interleaved;
  double magnitude;
};

// `rotation` as Python hands it on: None, or (turns, dim, interleaved, magnitude).
Rotation rotation_from(py::handle o) {
  if (o.is_none()) return {Tensor(), 0, false, 1.0};
  const auto t = py::cast<py::tuple>(o);
  return {tensor_of(t[0]), py::cast<int64_t>(t[1]), py::cast<bool>(t[2]), py::cast<double>(t[3])};
}

Tensor rotated(const Tensor &x_t, const Tensor &starts_t, const Tensor &positions_t,
               const Rotation &r, bool inverse) {
  const ArrayView x = view_of(x_t);
  const OptionalView starts(starts_t), positions(positions_t), turns(r.turns);
  if (x.ndim != 4) throw std::invalid_argument("rotary x must be rank-4.");
  const Tensor out = new_tensor(x_t, {x.shape[0], x.shape[1], x.shape[2], x.shape[3]}, x_t.scalar_type());
  const ArrayView vo = view_of(out);
  const ExecContext ctx = context_for(x, 0);
  const RotationView how{r.dim, r.interleaved, inverse, r.magnitude, turns.get};
  run_op(x, [&] { rotary(x, starts.get, positions.get, how, vo, ctx); });
  return out;
}

// A rotation's derivative is the rotation back, of any order.
struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext *ctx, Tensor x, std::optional<Tensor> starts,
                        std::optional<Tensor> positions, Tensor turns, int64_t dim,
                        bool interleaved, double magnitude, bool inverse) {
    ctx->save_for_backward({starts.value_or(Tensor()), positions.value_or(Tensor()), turns});
    ctx->saved_data["dim"] = dim;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["inverse"] = inverse;
    ctx->set_materialize_grads(false);
    return rotated(x, starts.value_or(Tensor()), positions.value_or(Tensor()),
                   {turns, dim, interleaved, magnitude}, inverse);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    variable_list result(8);
    if (!grads[0].defined()) return result;
    const variable_list s = ctx->get_saved_variables();
    const Rotation r{s[2], ctx->saved_data["dim"].toInt(), ctx->saved_data["interleaved"].toBool(),
                     ctx->saved_data["magnitude"].toDouble()};
    const bool inverse = !ctx->saved_data["inverse"].toBool();
    const Tensor grad = made_direct(grads[0]);
    result[0] = at::GradMode::is_enabled()
                    ? Rotary::apply(grad, present(s[0]), present(s[1]), r.turns, r.dim, r.interleaved,
                                    r.magnitude, inverse)
                    : rotated(grad, s[0], s[1], r, inverse);
    return result;
  }
};

bool usable_positions(const Tensor &t, const Tensor &x, int64_t device) {
  return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 2 &&
         t.size(0) == x.size(0) && t.size(1) == x.size(1) && on_device(t, device) && !t.is_neg();
}

bool absent_or_tensor(py::handle h) { return h.is_none() || THPVariable_Check(h.ptr()); }

py::object rotary_plain(py::handle x_o, py::handle starts_o, py::handle positions_o,
                        py::handle rotation, int64_t device) {
  if (!THPVariable_Check(x_o.ptr()) || !absent_or_tensor(starts_o) || !absent_or_tensor(positions_o))
    return py::none();
  const Tensor &x = tensor_of(x_o);
  const Tensor starts = optional_tensor(starts_o), positions = optional_tensor(positions_o);
  const Rotation r = rotation_from(rotation);
  if (x.dim() != 4 || !real_type(x.scalar_type()) || !usable(x, x.scalar_type(), device) ||
      x.size(3) > 256 || x.size(3) < r.dim || (starts.defined() && positions.defined()) ||
      (starts.defined() && !usable_counts(starts, x.size(0), device)) ||
      (positions.defined() && !usable_positions(positions, x, device)))
    return py::none();
  if (at::GradMode::is_enabled() && x.requires_grad())
    return wrap(Rotary::apply(x, present(starts), present(positions), r.turns, r.dim, r.interleaved,
                              r.magnitude, false));
  return wrap(rotated(x, starts, positions, r, false));
}

py::object rotary_call(py::handle x, py::handle starts, py::handle positions, py::handle rotation,
                       bool inverse) {
  return wrap(rotated(tensor_of(x), optional_tensor(starts), optional_tensor(positions),
                      rotation_from(rotation), inverse));
}

// ---------------------------------------------------------------------------
// Paged caches.

Tensor append(const Tensor &k_t, const Tensor &v_t, const Tensor &ck_t, const Tensor &cv_t,
              const Tensor &pages_t, const Tensor &starts_t, const Tensor &lengths_t,
              const Rotation &r, const Tensor &q_t) {
  const ArrayView k = view_of(k_t), v = view_of(v_t), ck = view_of(ck_t), cv = view_of(cv_t),
                  pages = view_of(pages_t);
  const OptionalView starts(starts_t), lengths(lengths_t), turns(r.turns), q(q_t);
  require_writable(ck_t, "paged_cache_append cache_k");
  require_writable(cv_t, "paged_cache_append cache_v");
  Tensor out;
  if (q_t.defined()) {
    if (q_t.dim() != 4) throw std::invalid_argument("paged_cache_append q must be rank-4.");
    out = new_tensor(q_t, {q_t.size(0), q_t.size(1), q_t.size(2), q_t.size(3)}, q_t.scalar_type());
  }
  const OptionalView vo(out);
  const ExecContext ctx = context_for(k, 0);
  const RotationView how{r.dim, r.interleaved, false, r.magnitude, turns.get};
  run_op(k, [&] {
    paged_cache_append(k, v, {ck, cv, pages}, starts.get, lengths.get, how, q.get, vo.get, ctx);
  });
  written(ck_t);
  written(cv_t);
  return out;
}

bool usable_table(const Tensor &t, int64_t batch, int64_t device) {
  return (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.dim() == 2 &&
         t.size(0) == batch && on_device(t, device) && direct(t);
}

// Caches that a call on `like` (batch, tokens, heads, dim) takes as they are.
bool usable_caches(const Tensor &like, const Tensor &ck, const Tensor &cv, const Tensor &pages,
                   int64_t device) {
  const at::ScalarType type = like.scalar_type();
  return like.dim() == 4 && real_type(type) && ck.dim() == 4 && cv.sizes() == ck.sizes() &&
         ck.size(3) == like.size(3) && ck.size(1) >= 1 && usable(ck, type, device) &&
         usable(cv, type, device) && !ck.requires_grad() && !cv.requires_grad() &&
         usable(like, type, device) && usable_table(pages, like.size(0), device);
}

bool usable_starts(const Tensor &starts, const Tensor &lengths, int64_t batch, int64_t device) {
  for (const Tensor *t : {&starts, &lengths})
    if (t->defined() && !usable_counts(*t, batch, device)) return false;
  return !starts.defined() || !lengths.defined() || starts.scalar_type() == lengths.scalar_type();
}

// (done, queries): done false where Python's checks are wanted.
py::object paged_cache_append_plain(py::handle k_o, py::handle v_o, py::handle ck_o,
                                    py::handle cv_o, py::handle pages_o, py::handle starts_o,
                                    py::handle lengths_o, py::handle rotation, py::handle q_o,
                                    int64_t device) {
  for (py::handle h : {k_o, v_o, ck_o, cv_o, pages_o})
    if (!THPVariable_Check(h.ptr())) return py::none();
  for (py::handle h : {starts_o, lengths_o, q_o})
    if (!absent_or_tensor(h)) return py::none();
  const Tensor &k = tensor_of(k_o), &v = tensor_of(v_o), &ck = tensor_of(ck_o), &cv = tensor_of(cv_o),
               &pages = tensor_of(pages_o);
  const Tensor starts = optional_tensor(starts_o), lengths = optional_tensor(lengths_o),
               q = optional_tensor(q_o);
  const Rotation r = rotation_from(rotation);
  if (!usable_caches(k, ck, cv, pages, device) || k.size(2) != ck.size(2) || v.sizes() != k.sizes() ||
      !usable(v, k.scalar_type(), device) || !usable_starts(starts, lengths, k.size(0), device) ||
      k.size(3) < r.dim)
    return py::none();
  if (q.defined() && (q.dim() != 4 || q.size(0) != k.size(0) || q.size(1) != k.size(1) ||
                      q.size(3) != k.size(3) || !usable(q, k.scalar_type(), device) || !r.turns.defined()))
    return py::none();
  return py::make_tuple(wrap(append(k, v, ck, cv, pages, starts, lengths, r, q)));
}

py::object paged_cache_append_call(py::handle k, py::handle v, py::handle ck, py::handle cv,
                                   py::handle pages, py::handle starts, py::handle lengths,
                                   py::handle rotation, py::handle q) {
  return wrap(append(tensor_of(k), tensor_of(v), tensor_of(ck), tensor_of(cv), tensor_of(pages),
                     optional_tensor(starts), optional_tensor(lengths), rotation_from(rotation),
                     optional_tensor(q)));
}

struct Seen {
  int64_t window, sinks, shared_pages;
  double scale;
};

Tensor attend(const Tensor &q_in, const Tensor &ck_t, const Tensor &cv_t, const Tensor &pages_t,
              const Tensor &starts_t, const Tensor &lengths_t, const Seen &s) {
  // (caches are never copied)
  const Tensor q_t = aligned_rows(ck_t) && aligned_rows(cv_t) ? for_tiles(q_in, kStepDim) : q_in;
  const ArrayView q = view_of(q_t), ck = view_of(ck_t), cv = view_of(cv_t), pages = view_of(pages_t);
  const OptionalView starts(starts_t), lengths(lengths_t);
  const auto desc = paged_attention_desc(q, {ck, cv, pages}, starts.get, lengths.get, s.window,
                                         s.sinks, s.scale, s.shared_pages);
  const Tensor out = new_tensor(q_t, {desc.batch, desc.tokens, desc.heads, desc.cache.dim}, q_t.scalar_type());
  const ArrayView vo = view_of(out);
  ExecContext ctx = context_for(q, 0);
  Tensor scratch;
  if (q.device >= 0) scratch = scratch_for(ctx, q_t, msx_paged_attention_scratch(&desc));
  run_op(q, [&] { paged_attention(desc, vo, ctx); });
  return out;
}

bool plain_int(py::handle o, int64_t least, int64_t &value) {
  if (!PyLong_CheckExact(o.ptr())) return false;
  int over = 0;
  value = PyLong_AsLongLongAndOverflow(o.ptr(), &over);
  // 2^40 at most, to which the checks in Python lower wider spans
  return !over && value >= least && value <= (int64_t{1} << 40);
}

py::object paged_attention_plain(py::handle q_o, py::handle ck_o, py::handle cv_o,
                                 py::handle pages_o, py::handle starts_o, py::handle lengths_o,
                                 py::handle window, py::handle sinks, py::handle scale,
                                 py::handle shared_pages, int64_t device) {
  for (py::handle h : {q_o, ck_o, cv_o, pages_o})
    if (!THPVariable_Check(h.ptr())) return py::none();
  if (!absent_or_tensor(starts_o) || !absent_or_tensor(lengths_o)) return py::none();
  const Tensor &q = tensor_of(q_o), &ck = tensor_of(ck_o), &cv = tensor_of(cv_o),
               &pages = tensor_of(pages_o);
  const Tensor starts = optional_tensor(starts_o), lengths = optional_tensor(lengths_o);
  Seen s{};
  if (!usable_caches(q, ck, cv, pages, device) || !usable_starts(starts, lengths, q.size(0), device))
    return py::none();
  const int64_t heads = q.size(2), kv_heads = ck.size(2), dim = q.size(3);
  if (kv_heads < 1 || heads < 1 || heads % kv_heads != 0 || dim < 1 || dim > 256) return py::none();
  if (window.is_none()) s.window = int64_t{1} << 40;
  else if (!plain_int(window, 1, s.window)) return py::none();
  if (!plain_int(sinks, 0, s.sinks) || !plain_int(shared_pages, 0, s.shared_pages) ||
      s.shared_pages > pages.size(1))
    return py::none();
  if (scale.is_none()) s.scale = 1.0 / std::sqrt(static_cast<double>(dim));
  else if (PyFloat_CheckExact(scale.ptr())) s.scale = PyFloat_AS_DOUBLE(scale.ptr());
  else return py::none();
  return wrap(attend(q, ck, cv, pages, starts, lengths, s));
}

py::object paged_attention_call(py::handle q, py::handle ck, py::handle cv, py::handle pages,
                                py::handle starts, py::handle lengths, int64_t window,
                                int64_t sinks, double scale, int64_t shared_pages) {
  return wrap(attend(tensor_of(q), tensor_of(ck), tensor_of(cv), tensor_of(pages),
                     optional_tensor(starts), optional_tensor(lengths),
                     {window, sinks, shared_pages, scale}));
}

}  // namespace

void bind_paged(py::module_ &m) {
  m.def("rotary_plain", &rotary_plain, py::arg("x"), py::arg("starts"), py::arg("positions"),
        py::arg("rotation"), py::arg("device"),
        "rotary where nothing is to be done to the operands, else None.");
  m.def("rotary", &rotary_call, py::arg("x"), py::arg("starts"), py::arg("positions"),
        py::arg("rotation"), py::arg("inverse"), "Heads rotated by their positions, or back.");
  m.def("paged_cache_append_plain", &paged_cache_append_plain, py::arg("k"), py::arg("v"),
        py::arg("cache_k"), py::arg("cache_v"), py::arg("pages"), py::arg("starts"),
        py::arg("lengths"), py::arg("rotation"), py::arg("q"), py::arg("device"),
        "(queries,) of paged_cache_append where nothing is to be done to the operands, else None.");
  m.def("paged_cache_append", &paged_cache_append_call, py::arg("k"), py::arg("v"),
        py::arg("cache_k"), py::arg("cache_v"), py::arg("pages"), py::arg("starts"),
        py::arg("lengths"), py::arg("rotation"), py::arg("q"),
        "Keys and values into a paged cache; the queries rotated, or None.");
  m.def("paged_attention_plain", &paged_attention_plain, py::arg("q"), py::arg("cache_k"),
        py::arg("cache_v"), py::arg("pages"), py::arg("starts"), py::arg("lengths"),
        py::arg("window"), py::arg("sinks"), py::arg("scale"), py::arg("shared_pages"),
        py::arg("device"),
        "paged_attention where nothing is to be done to the operands, else None.");
  m.def("paged_attention", &paged_attention_call, py::arg("q"), py::arg("cache_k"),
        py::arg("cache_v"), py::arg("pages"), py::arg("starts"), py::arg("lengths"),
        py::arg("window"), py::arg("sinks"), py::arg("scale"), py::arg("shared_pages"),
        "Attention of every sequence's last tokens over its pages.");
}
