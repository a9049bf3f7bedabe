// Autograd nodes of the norms, the embedding and the distillation loss.
//
// The Python layer checks a call and hands it over here: outputs and workspaces are
// allocated, the C ABI is called on the current stream, and what a backward pass needs
// is saved, all without the interpreter.  A call whose operands are all of the ordinary
// kind takes one step less: the usual_* functions make the same checks here and run it,
// and answer None to any other, which then goes through the Python layer's checks, for
// its conversions and its errors (norm of 64 x 1024: 5.2 us -> 4.1; a loss of 4 x 1000
// with weights: 8.3 -> 4.2, with its gradient 9.4 -> 5.3).  A backward pass runs in the engine's own
// thread; one written in Python has to be handed the interpreter's lock there first
// and finds its caches cold.  Host time of a layer norm of 64 x 1024, forward and
// backward, with the nodes in Python: 130 us; here: 42.
//
// The C ABI's addresses come from the Python layer, which has loaded the library: this
// module links to none of it.
#include <Python.h>
#include <limits.h>

#include <cmath>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/mfattn.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using MaybeTensor = std::optional<Tensor>;

// ---------------------------------------------------------------------------
// The C ABI
// ---------------------------------------------------------------------------

#define MF_FUNCTIONS(F)                                                                 \
  F(mf_norm) F(mf_norm_bwd) F(mf_norm_bwd_workspace_bytes) F(mf_embed) F(mf_embed_bwd)  \
  F(mf_embed_bwd_workspace_bytes) F(mf_distill) F(mf_distill_bwd)                       \
  F(mf_distill_stats_bytes) F(mf_last_error)

struct Library {
#define MF_MEMBER(name) decltype(&::name) name = nullptr;
  MF_FUNCTIONS(MF_MEMBER)
#undef MF_MEMBER
} lib;

PyObject* error_class = nullptr;        // of the library's refusals: a ValueError
PyObject* launch_error_class = nullptr;  // of failed launches

// A call that the library refused; the caller of a forward pass sees the Python layer's own
// exception for it.
struct Refused {
  int code;
  std::string message;
};

void check(int code) {
  if (code != MF_OK) throw Refused{code, lib.mf_last_error()};
}

int code_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? MF_DTYPE_F32 : MF_DTYPE_BF16; }

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T* data_as(const Tensor& t) {
  return static_cast<T*>(data(t));
}

// Elements between the rows of x [..., D], which the Python layer has found evenly spaced.
long long row_step(const Tensor& x) {
  const int64_t d = x.size(-1);
  if (x.is_contiguous()) return d;
  for (int64_t i = x.dim() - 2; i >= 0; --i)
    if (x.size(i) > 1) return x.stride(i);
  return d;
}

// Whether the rows of x are evenly spaced, do not overlap, and are dense themselves.
bool rows_even(const Tensor& x) {
  if (x.is_contiguous()) return true;
  const int64_t d = x.size(-1);
  if (d > 1 && x.stride(-1) != 1) return false;
  int64_t step = -1, rows = 1;  // between rows, and rows of the dimensions behind
  for (int64_t i = x.dim() - 2; i >= 0; --i) {
    if (x.size(i) <= 1) continue;
    if (step < 0) {
      step = x.stride(i);
      if (step < d) return false;
    } else if (x.stride(i) != step * rows) {
      return false;
    }
    rows *= x.size(i);
  }
  return true;
}

// The kernels read memory: a view whose sign stands beside it (of a conjugate's imaginary part,
// say) is written out.
Tensor dense(const Tensor& x) { return x.resolve_neg().contiguous(); }
Tensor even(const Tensor& x) { return rows_even(x) ? x.resolve_neg() : dense(x); }

// The C ABI takes its sizes as int.
void fit(std::initializer_list<int64_t> sizes) {
  for (int64_t n : sizes)
    if (n > INT_MAX) throw Refused{MF_ERR_SHAPE, "sizes must be below 2^31"};
}

Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte));
}

void refuse_second_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              " is differentiable once: its backward pass records no graph (create_graph=True)");
}

// What was saved goes through the caller's hooks (torch.autograd.graph.saved_tensors_hooks),
// which may lay it out anew but have to give it back.
void restored(bool same) {
  TORCH_CHECK(same, "a tensor saved for the backward pass came back with another shape, dtype "
                    "or device");
}

bool on(const Tensor& t, const Tensor& like, int64_t numel) {
  return t.device() == like.device() && t.numel() == numel;
}

// A library's refusal inside the engine's thread.
template <typename F>
void in_backward(F&& f) {
  try {
    f();
  } catch (const Refused& r) {
    TORCH_CHECK(false, r.message);
  }
}

// ---------------------------------------------------------------------------
// Norms
// ---------------------------------------------------------------------------

Tensor norm(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, bool center,
            Tensor* stats) {
  const int64_t d = x.size(-1), rows = x.numel() / d;
  fit({rows, d});
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  if (stats) *stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  if (rows)
    check(lib.mf_norm(data(x), row_step(x), data(weight), data(bias), code_of(x), code_of(weight),
                      (int)rows, (int)d, center, (float)eps, data(y),
                      stats ? data_as<float>(*stats) : nullptr, stream_of(x)));
  return y;
}

struct Norm : public Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const MaybeTensor& maybe_bias, double eps, bool center) {
    const Tensor bias = maybe_bias.value_or(Tensor());
    Tensor stats, y = norm(x, weight, bias, eps, center, &stats);
    ctx->save_for_backward({x, weight, stats});
    ctx->saved_data["center"] = center;
    ctx->saved_data["bias"] = bias.defined();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_second_order("the norm");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor x = even(saved[0]), weight = dense(saved[1]), stats = dense(saved[2]);
    const bool center = ctx->saved_data["center"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
               need_b = ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(2);
    const int64_t d = x.size(-1), rows = x.numel() / d;
    const auto param = weight.scalar_type();
    restored(x.sizes() == grads[0].sizes() && on(x, grads[0], grads[0].numel()) &&
             x.scalar_type() == grads[0].scalar_type() && on(weight, x, d) &&
             (param == x.scalar_type() || param == at::kFloat) && on(stats, x, 2 * rows) &&
             stats.scalar_type() == at::kFloat);
    c10::DeviceGuard guard(x.device());
    Tensor dx, dw, db, ws;
    if (rows == 0) {
      if (need_x) dx = at::zeros_like(x);
      if (need_w) dw = at::zeros_like(weight);
      if (need_b) db = at::zeros_like(weight);
      return {dx, dw, db, Tensor(), Tensor()};
    }
    const Tensor dy = even(grads[0]);
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_w) dw = at::empty({d}, weight.options());
    if (need_b) db = at::empty({d}, weight.options());
    size_t need = 0;
    if (need_w || need_b) {
      need = lib.mf_norm_bwd_workspace_bytes((int)rows, (int)d, code_of(x));
      if (need) ws = bytes(need, x);
    }
    in_backward([&] {
      check(lib.mf_norm_bwd(data(x), row_step(x), data(weight), data_as<float>(stats), data(dy),
                            row_step(dy), code_of(x), code_of(weight), (int)rows, (int)d, center,
                            data(dx), data(dw), data(db), data(ws), need, stream_of(x)));
    });
    return {dx, dw, db, Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------

Tensor embed(const Tensor& ids, const Tensor& table, double scale, int64_t padding) {
  const int64_t v = table.size(0), d = table.size(1), n = ids.numel();
  fit({v, d, n});
  c10::DeviceGuard guard(table.device());
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(d);
  Tensor out = at::empty(shape, table.options());
  if (n)
    check(lib.mf_embed(data(ids), (int)ids.element_size(), data(table), row_step(table),
                       code_of(table), (int)n, (int)v, (int)d, padding, (float)scale, data(out),
                       stream_of(table)));
  return out;
}

Tensor embed_gradient(const Tensor& grad, const Tensor& ids, int64_t v, double scale,
                      int64_t padding) {
  const int64_t d = grad.size(-1), n = ids.numel();
  restored(on(ids, grad, grad.numel() / d) &&
           (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong));
  c10::DeviceGuard guard(grad.device());
  if (n == 0) return at::zeros({v, d}, grad.options());
  const Tensor dout = even(grad);
  Tensor dtable = at::empty({v, d}, dout.options());
  const size_t need = lib.mf_embed_bwd_workspace_bytes((int)n, (int)v, (int)d);
  const Tensor ws = bytes(need, dout);
  check(lib.mf_embed_bwd(data(ids), (int)ids.element_size(), data(dout), row_step(dout),
                         code_of(dout), (int)n, (int)v, (int)d, padding, (float)scale, data(dtable),
                         data(ws), need, stream_of(dout)));
  return dtable;
}

// The lookup and its gradient are linear and each other's transpose: differentiable as
// often as asked.
struct Embed : public Function<Embed> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& table, double scale,
                        int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["v"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed(ids, table, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads);
};

struct EmbedGradient : public Function<EmbedGradient> {
  static Tensor forward(AutogradContext* ctx, const Tensor& grad, const Tensor& ids, int64_t v,
                        double scale, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    return embed_gradient(grad, ids, v, scale, padding);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor ids = dense(ctx->get_saved_variables()[0]), g = even(grads[0]);
    restored(ids.device() == g.device() &&
             (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong));
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t padding = ctx->saved_data["padding"].toInt();
    Tensor out;
    in_backward([&] {
      out = at::GradMode::is_enabled() ? Embed::apply(ids, g, scale, padding)
                                       : embed(ids, g, scale, padding);
    });
    return {out, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

variable_list Embed::backward(AutogradContext* ctx, variable_list grads) {
  const Tensor ids = dense(ctx->get_saved_variables()[0]);
  const int64_t v = ctx->saved_data["v"].toInt(), padding = ctx->saved_data["padding"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  Tensor dtable;
  in_backward([&] {
    dtable = at::GradMode::is_enabled() ? EmbedGradient::apply(grads[0], ids, v, scale, padding)
                                        : embed_gradient(grads[0], ids, v, scale, padding);
  });
  return {Tensor(), dtable, Tensor(), Tensor()};
}

// ---------------------------------------------------------------------------
// Distillation
// ---------------------------------------------------------------------------

Tensor distill(const Tensor& logits, const Tensor& teacher, const Tensor& ids, const Tensor& total,
               const Tensor& weights, double temperature, Tensor* stats, const Tensor& grad) {
  const int64_t v = logits.size(-1), k = ids.size(-1), rows = logits.numel() / v;
  fit({v, k, rows});
  c10::DeviceGuard guard(logits.device());
  Tensor loss = at::empty(logits.sizes().slice(0, logits.dim() - 1),
                          logits.options().dtype(at::kFloat));
  size_t nbytes = 0;
  if (stats) {
    nbytes = lib.mf_distill_stats_bytes((int)rows, (int)k);
    *stats = at::empty({(int64_t)nbytes / 4}, loss.options());
  }
  if (rows)
    check(lib.mf_distill(data(logits), row_step(logits), data(teacher), code_of(teacher), data(ids),
                         (int)ids.element_size(), data_as<float>(total), data_as<float>(weights),
                         code_of(logits), (int)rows, (int)v, (int)k, temperature,
                         data_as<float>(loss), stats ? data_as<float>(*stats) : nullptr, nbytes,
                         data(grad), grad.defined() ? row_step(grad) : 0, stream_of(logits)));
  return loss;
}

struct TopLogitsLoss : public Function<TopLogitsLoss> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& teacher,
                        const Tensor& ids, const MaybeTensor& total,
                        const MaybeTensor& maybe_weights, double temperature) {
    const Tensor weights = maybe_weights.value_or(Tensor());
    Tensor stats, loss = distill(logits, teacher, ids, total.value_or(Tensor()), weights,
                                 temperature, &stats, Tensor());
    ctx->save_for_backward({logits, ids, weights, stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["dtype"] = logits.scalar_type();
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_second_order("the loss");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor logits = even(saved[0]), ids = dense(saved[1]),
                 weights = saved[2].defined() ? dense(saved[2]) : saved[2],
                 stats = dense(saved[3]);
    const int64_t v = logits.size(-1), k = ids.size(-1), rows = grads[0].numel();
    restored(on(logits, grads[0], rows * v) && logits.dim() == grads[0].dim() + 1 &&
             logits.scalar_type() == ctx->saved_data["dtype"].toScalarType() &&
             on(ids, logits, rows * k) &&
             (ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong) &&
             (!weights.defined() ||
              (on(weights, logits, rows) && weights.scalar_type() == at::kFloat)) &&
             on(stats, logits, rows * (k + 4)) && stats.scalar_type() == at::kFloat);
    c10::DeviceGuard guard(logits.device());
    const Tensor grad = at::empty(logits.sizes(), logits.options());
    const Tensor dloss = dense(grads[0]);
    in_backward([&] {
      if (rows)
        check(lib.mf_distill_bwd(data(logits), row_step(logits), data(ids), (int)ids.element_size(),
                                 data_as<float>(weights), data_as<float>(stats),
                                 4 * (size_t)stats.numel(), data_as<float>(dloss), code_of(logits),
                                 (int)rows, (int)v, (int)k,
                                 ctx->saved_data["temperature"].toDouble(), data(grad), v,
                                 stream_of(logits)));
    });
    return {grad, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ---------------------------------------------------------------------------
// Python's side
// ---------------------------------------------------------------------------

Tensor unpack(PyObject* o) {
  if (o == Py_None) return Tensor();
  TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a tensor or None");
  return THPVariable_Unpack(o);
}

MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : std::nullopt; }

double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return x;
}

int64_t integer(PyObject* o) {
  const int64_t x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}

// Runs f, a tensor's worth of work, with the interpreter's lock released.
template <typename F>
PyObject* tensor_of(F&& f) {
  Tensor out;
  try {
    pybind11::gil_scoped_release no_gil;
    out = f();
  } catch (const Refused& r) {
    PyObject* type = r.code == MF_ERR_HIP ? launch_error_class : error_class;
    PyObject* args = Py_BuildValue("(is)", r.code, r.message.c_str());
    if (args) {
      PyErr_SetObject(type, args);
      Py_DECREF(args);
    }
    throw python_error();
  }
  return THPVariable_Wrap(std::move(out));
}

void expect(Py_ssize_t got, Py_ssize_t want) {
  TORCH_CHECK_TYPE(got == want, "expected ", want, " arguments, got ", got);
}

// init({name: address}, refusal class, launch error class)
PyObject* py_init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 3);
#define MF_TAKE(f)                                                          \
  {                                                                         \
    PyObject* address = PyDict_GetItemString(a[0], #f);                     \
    TORCH_CHECK_VALUE(address, "no address of " #f);                        \
    lib.f = reinterpret_cast<decltype(lib.f)>(PyLong_AsVoidPtr(address));   \
    TORCH_CHECK_VALUE(lib.f, "no address of " #f);                          \
  }
  MF_FUNCTIONS(MF_TAKE)
#undef MF_TAKE
  Py_INCREF(a[1]);
  Py_INCREF(a[2]);
  error_class = a[1];
  launch_error_class = a[2];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// norm(x, weight, bias, eps, center, record)
PyObject* py_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 6);
  const Tensor x = unpack(a[0]), w = unpack(a[1]), b = unpack(a[2]);
  const double eps = number(a[3]);
  const bool center = a[4] == Py_True, record = a[5] == Py_True;
  return tensor_of([&] {
    return record ? Norm::apply(x, w, maybe(b), eps, center) : norm(x, w, b, eps, center, nullptr);
  });
  END_HANDLE_TH_ERRORS
}

// embed(ids, table, scale, padding, record)
PyObject* py_embed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  const Tensor ids = unpack(a[0]), table = unpack(a[1]);
  const double scale = number(a[2]);
  const int64_t padding = integer(a[3]);
  const bool record = a[4] == Py_True;
  return tensor_of([&] {
    return record ? Embed::apply(ids, table, scale, padding) : embed(ids, table, scale, padding);
  });
  END_HANDLE_TH_ERRORS
}

// distill(logits, teacher, ids, total, weights, temperature, record, gradient)
PyObject* py_distill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 8);
  const Tensor z = unpack(a[0]), t = unpack(a[1]), ids = unpack(a[2]), total = unpack(a[3]),
               weights = unpack(a[4]), grad = unpack(a[7]);
  const double temperature = number(a[5]);
  const bool record = a[6] == Py_True;
  return tensor_of([&] {
    return record ? TopLogitsLoss::apply(z, t, ids, maybe(total), maybe(weights), temperature)
                  : distill(z, t, ids, total, weights, temperature, nullptr, grad);
  });
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------------
// Ordinary calls
// ---------------------------------------------------------------------------

// A device tensor of a dtype that the kernels have, without a tangent and its memory what it
// holds; one of `like`'s device.
bool usual(const Tensor& t, const Tensor& like) {
  const auto dtype = t.scalar_type();
  return t.is_cuda() && (dtype == at::kFloat || dtype == at::kBFloat16) &&
         t.device() == like.device() && !t.is_neg() && !t._fw_grad(0).defined();
}

bool usual_ids(const Tensor& t, const Tensor& like) {
  return t.is_cuda() && (t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) &&
         t.device() == like.device() && t.is_contiguous() && !t.is_neg();
}

// None or a tensor; false: neither.
bool take(PyObject* o, Tensor& t) {
  if (o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  t = THPVariable_Unpack(o);
  return true;
}

bool take_tensor(PyObject* o, Tensor& t) { return take(o, t) && t.defined(); }

bool records(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// usual_norm(x, weight, bias, eps, center)
PyObject* py_usual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 5);
  Tensor x, w, b;
  if (!take_tensor(a[0], x) || !take_tensor(a[1], w) || !take(a[2], b) || !PyFloat_Check(a[3]))
    Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(a[3]);
  const bool center = a[4] == Py_True;
  auto parameter = [&](const Tensor& p) {
    return usual(p, x) && p.dim() == 1 && p.size(0) == x.size(-1) && p.is_contiguous() &&
           p.scalar_type() == w.scalar_type();
  };
  if (!usual(x, x) || x.dim() == 0 || x.size(-1) == 0 || !rows_even(x) || !parameter(w) ||
      (w.scalar_type() != x.scalar_type() && w.scalar_type() != at::kFloat) ||
      (b.defined() && !parameter(b)) || !(eps >= 0 && std::isfinite(eps)))
    Py_RETURN_NONE;
  const bool record = records({&x, &w, &b});
  return tensor_of([&] {
    return record ? Norm::apply(x, w, maybe(b), eps, center) : norm(x, w, b, eps, center, nullptr);
  });
  END_HANDLE_TH_ERRORS
}

// usual_embed(ids, table, scale, padding)
PyObject* py_usual_embed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  Tensor ids, table;
  if (!take_tensor(a[0], ids) || !take_tensor(a[1], table) || !PyFloat_Check(a[2]))
    Py_RETURN_NONE;
  const double scale = PyFloat_AS_DOUBLE(a[2]);
  int64_t padding = -1;
  if (a[3] != Py_None) {
    if (!PyLong_CheckExact(a[3])) Py_RETURN_NONE;
    int overflow = 0;
    padding = PyLong_AsLongLongAndOverflow(a[3], &overflow);
    if (overflow) Py_RETURN_NONE;
  }
  if (!usual(table, table) || table.dim() != 2 || table.numel() == 0 || !rows_even(table) ||
      !usual_ids(ids, table) || !std::isfinite(scale))
    Py_RETURN_NONE;
  const bool record = records({&table});
  return tensor_of([&] {
    return record ? Embed::apply(ids, table, scale, padding) : embed(ids, table, scale, padding);
  });
  END_HANDLE_TH_ERRORS
}

// usual_distill(logits, teacher, ids, total, weights, temperature, both): the loss, or the loss
// and the gradient
PyObject* py_usual_distill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  Tensor z, t, ids, total, weights;
  if (!take_tensor(a[0], z) || !take_tensor(a[1], t) || !take_tensor(a[2], ids) ||
      !take(a[3], total) || !take(a[4], weights) || !PyFloat_Check(a[5]))
    Py_RETURN_NONE;
  const double temperature = PyFloat_AS_DOUBLE(a[5]);
  auto lead = [&] { return z.sizes().slice(0, z.dim() - 1); };
  auto per_row = [&](const Tensor& r) {
    return usual(r, z) && r.scalar_type() == at::kFloat && r.is_contiguous() && r.sizes() == lead();
  };
  if (!usual(z, z) || z.dim() == 0 || z.size(-1) == 0 || !rows_even(z) || !usual_ids(ids, z) ||
      ids.dim() != z.dim() || ids.size(-1) == 0 || ids.sizes().slice(0, z.dim() - 1) != lead() ||
      !usual(t, z) || t.sizes() != ids.sizes() || !t.is_contiguous() ||
      (total.defined() && !per_row(total)) || (weights.defined() && !per_row(weights)) ||
      !(temperature >= 1e-6 && temperature <= 1e6) || records({&t, &total, &weights}))
    Py_RETURN_NONE;
  const bool record = records({&z});
  if (a[6] == Py_True) {
    if (record) Py_RETURN_NONE;
    Tensor grad;
    PyObject* loss = tensor_of([&] {
      c10::DeviceGuard guard(z.device());
      grad = at::empty(z.sizes(), z.options());
      return distill(z, t, ids, total, weights, temperature, nullptr, grad);
    });
    if (!loss) return nullptr;
    PyObject* dz = THPVariable_Wrap(std::move(grad));
    PyObject* pair = dz ? PyTuple_Pack(2, loss, dz) : nullptr;
    Py_DECREF(loss);
    Py_XDECREF(dz);
    return pair;
  }
  return tensor_of([&] {
    return record ? TopLogitsLoss::apply(z, t, ids, maybe(total), maybe(weights), temperature)
                  : distill(z, t, ids, total, weights, temperature, nullptr, Tensor());
  });
  END_HANDLE_TH_ERRORS
}

// rows_even(x)
PyObject* py_rows_even(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 1);
  return PyBool_FromLong(rows_even(unpack(a[0])));
  END_HANDLE_TH_ERRORS
}

#define MF_METHOD(name)                                                                   \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##name)), METH_FASTCALL, \
   nullptr}
PyMethodDef methods[] = {MF_METHOD(init),          MF_METHOD(norm),
                         MF_METHOD(embed),         MF_METHOD(distill),
                         MF_METHOD(usual_norm),    MF_METHOD(usual_embed),
                         MF_METHOD(usual_distill), MF_METHOD(rows_even),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mfnodes", "Autograd nodes over the C ABI.", -1,
                      methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__mfnodes() { return PyModule_Create(&module); }
