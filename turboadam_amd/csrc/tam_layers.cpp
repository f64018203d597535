// tam_layers.cpp -- linear and layer_norm for torch: argument checks, outputs and
// workspaces, and the autograd nodes of their backward passes (part of the torch
// extension module _tam_host).
//
// A layer's host work in Python (two ctypes structures and an autograd.Function)
// took 140 us for a layer norm's forward and backward pass, several times its
// kernels' time at GPT-2's size; here it is a few microseconds a call.  The
// kernels are reached through the library's C entries, whose addresses
// turboadam_amd.layers hands over once (bind_layers): the library stays the one
// that the rest of the package has loaded.
#include "tam_layers.h"

namespace {

using namespace tam;

constexpr int64_t kMostNorm = 32768;               // elements of a layer norm's row

// ------------------------------------------------------------------ linear
struct LinearCall {
  TamLinear d = {};
  Tensor x, w;  // what d points at
  bool in_out;

  LinearCall(const Tensor& x0, const Tensor& weight, int64_t activation) {
    int64_t ldx, ldw;
    x = rows_of(x0, weight.size(1), ldx);
    w = weight_of(weight, ldw, in_out);
    d.x = x.data_ptr();
    d.w = w.data_ptr();
    d.rows = x.size(0);
    d.inputs = x.size(1);
    d.outputs = w.size(0);
    d.ldx = ldx;
    d.ldw = ldw;
    d.w_in_out = in_out;
    d.dtype = dtype_of(x);
    d.activation = (uint32_t)activation;
  }

  void run(bool backward) {
    const char* what = backward ? "tam_linear_backward" : "tam_linear";
    size_t need = 0;
    check(lib.linear_workspace(&d, backward, &need), what);
    const Tensor ws = workspace(need, x);
    check((backward ? lib.linear_backward : lib.linear)(&d, ptr(ws), need, stream_of(x)), what);
  }
};

Tensor linear_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual,
                      int64_t activation, Tensor* z) {
  const c10::DeviceGuard guard(x.device());
  LinearCall c(x, weight, activation);
  auto sizes = x.sizes().vec();
  sizes.back() = weight.size(0);
  const Tensor y = at::empty(sizes, x.options().requires_grad(false)), b = plain(bias), r = plain(residual);
  if (z && activation) *z = at::empty(sizes, y.options());
  c.d.bias = ptr(b);
  c.d.residual = ptr(r);
  c.d.y = y.data_ptr();
  c.d.z = z ? ptr(*z) : nullptr;
  c.run(false);
  return y;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const OptTensor& bias, const OptTensor& residual, int64_t activation) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor b = given(bias), r = given(residual);
    // the activation's argument is kept unless only the residual's gradient is wanted
    const bool keep = wants_gradient(x) || wants_gradient(weight) || wants_gradient(b);
    Tensor z;
    const Tensor y = linear_forward(x, weight, b, r, activation, keep ? &z : nullptr);
    ctx->save_for_backward({x, weight, z});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["wants"] = (int64_t)((wants_gradient(x) ? 1 : 0) | (wants_gradient(weight) ? 2 : 0) |
                                         (wants_gradient(b) ? 4 : 0) | (wants_gradient(r) ? 8 : 0));
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    not_twice("linear");
    refuse_recording("linear");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &z = saved[2], dy = grads[0];
    refuse_tangents("linear", {&dy});
    const int64_t wants = ctx->saved_data["wants"].toInt();
    Tensor dx, dw, db;
    if (dy.defined() && (wants & 7)) {
      const c10::DeviceGuard guard(x.device());
      LinearCall c(x, weight, ctx->saved_data["activation"].toInt());
      const Tensor g = plain(dy);
      const auto options = x.options().requires_grad(false);
      const int64_t outputs = weight.size(0), inputs = weight.size(1);
      if (wants & 1) dx = at::empty(x.sizes(), options);
      if (wants & 2)  // laid out as the weight
        dw = c.in_out ? at::empty({inputs, outputs}, options) : at::empty({outputs, inputs}, options);
      if (wants & 4) db = at::empty({outputs}, options);
      c.d.dy = g.data_ptr();
      c.d.z = ptr(z);
      c.d.dx = ptr(dx);
      c.d.dw = ptr(dw);
      c.d.db = ptr(db);
      c.run(true);
      if (dw.defined() && c.in_out) dw = dw.t();
    }
    return {dx, dw, db, wants & 8 ? dy : Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
              int64_t activation) {
  check_first("linear", x);
  refuse_recording("linear");
  check_other("linear", "weight", weight, x);
  if (weight.dim() != 2 || x.dim() < 1 || x.size(-1) != weight.size(1))
    refuse_value(c10::str("linear: x ", shape(x), " and weight ", shape(weight),
                          " are not (..., inputs) and (outputs, inputs)"));
  if (bias) {
    check_other("linear", "bias", *bias, x);
    if (bias->dim() != 1 || bias->size(0) != weight.size(0))
      refuse_value(c10::str("linear: bias must have shape (", weight.size(0), ",), got ", shape(*bias)));
  }
  if (residual) {
    check_other("linear", "residual", *residual, x);
    auto sizes = x.sizes().vec();
    sizes.back() = weight.size(0);
    if (residual->sizes() != at::IntArrayRef(sizes))
      refuse_value(c10::str("linear: residual must have the result's shape (", at::IntArrayRef(sizes), "), got ",
                            shape(*residual)));
  }
  const Tensor b = given(bias), r = given(residual);
  refuse_tangents("linear", {&x, &weight, &b, &r});
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() ||
                                     (bias && bias->requires_grad()) || (residual && residual->requires_grad())))
    return Linear::apply(x, weight, bias, residual, activation);
  return linear_forward(x, weight, b, r, activation, nullptr);
}

// -------------------------------------------------------------- layer norm
struct NormCall {
  TamNorm d = {};
  Tensor x, w, b;  // what d points at

  NormCall(const Tensor& x0, const Tensor& weight, const Tensor& bias, double eps) {
    int64_t ld;
    x = rows_of(x0, x0.size(-1), ld);
    w = plain(weight);
    b = plain(bias);
    d.x = x.data_ptr();
    d.w = ptr(w);
    d.b = ptr(b);
    d.rows = x.size(0);
    d.n = x.size(1);
    d.ldx = ld;
    d.dtype = dtype_of(x);
    d.eps = (float)eps;
  }
};

Tensor norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, double eps, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  NormCall c(x, weight, bias, eps);
  const Tensor y = at::empty(x.sizes(), x.options().requires_grad(false));
  if (stats) *stats = at::empty({(int64_t)c.d.rows, 2}, y.options().dtype(at::kFloat));
  c.d.y = y.data_ptr();
  c.d.stats = stats ? static_cast<float*>(stats->data_ptr()) : nullptr;
  check(lib.norm(&c.d, stream_of(x)), "tam_norm");
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const OptTensor& weight,
                        const OptTensor& bias, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor w = given(weight), b = given(bias);
    Tensor stats;
    const Tensor y = norm_forward(x, w, b, eps, &stats);
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["wants"] =
        (int64_t)((wants_gradient(x) ? 1 : 0) | (wants_gradient(w) ? 2 : 0) | (wants_gradient(b) ? 4 : 0));
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    not_twice("layer_norm");
    refuse_recording("layer_norm");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], dy = grads[0];
    refuse_tangents("layer_norm", {&dy});
    const int64_t wants = ctx->saved_data["wants"].toInt();
    Tensor dx, dw, db;
    if (dy.defined() && wants) {
      const c10::DeviceGuard guard(x.device());
      NormCall c(x, saved[1], Tensor(), ctx->saved_data["eps"].toDouble());
      const Tensor g = plain(dy);
      const auto options = x.options().requires_grad(false);
      if (wants & 1) dx = at::empty(x.sizes(), options);
      if (wants & 2) dw = at::empty({(int64_t)c.d.n}, options);
      if (wants & 4) db = at::empty({(int64_t)c.d.n}, options);
      c.d.dy = g.data_ptr();
      c.d.stats = static_cast<float*>(saved[2].data_ptr());
      c.d.dx = ptr(dx);
      c.d.dw = ptr(dw);
      c.d.db = ptr(db);
      size_t need = 0;
      check(lib.norm_workspace(&c.d, 1, &need), "tam_norm_backward");
      const Tensor ws = workspace(need, x);
      check(lib.norm_backward(&c.d, ptr(ws), need, stream_of(x)), "tam_norm_backward");
    }
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  check_first("layer_norm", x);
  refuse_recording("layer_norm");
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > kMostNorm)
    refuse_value(c10::str("layer_norm: x must have rows of 1 to ", kMostNorm, " elements, got ", shape(x)));
  if (!(eps >= 0)) refuse_value(c10::str("layer_norm: eps must be 0 or more, got ", eps));
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor&>("weight", weight), {"bias", bias}})
    if (t) {
      check_other("layer_norm", name, *t, x);
      if (t->dim() != 1 || t->size(0) != x.size(-1))
        refuse_value(c10::str("layer_norm: ", name, " must have shape (", x.size(-1), ",), got ", shape(*t)));
    }
  const Tensor w = given(weight), b = given(bias);
  refuse_tangents("layer_norm", {&x, &w, &b});
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
    return LayerNorm::apply(x, weight, bias, eps);
  return norm_forward(x, w, b, eps, nullptr);
}

// The same checks for an entry whose host work is in Python.
void check_call(const std::string& what, const Tensor& t) {
  refuse_recording(what.c_str());
  refuse_tangents(what.c_str(), {&t});
}

template <typename F>
void take(const py::dict& at, const char* name, F& f) {
  f = reinterpret_cast<F>(at[name].cast<uintptr_t>());
}

}  // namespace

void tam_register_layers(py::module_& m) {
  m.def("bind_layers", [](const py::dict& at) {
    take(at, "tam_linear_workspace", lib.linear_workspace);
    take(at, "tam_linear", lib.linear);
    take(at, "tam_linear_backward", lib.linear_backward);
    take(at, "tam_norm_workspace", lib.norm_workspace);
    take(at, "tam_norm", lib.norm);
    take(at, "tam_norm_backward", lib.norm_backward);
    take(at, "tam_gated_kept", lib.gated_kept);
    take(at, "tam_gated_workspace", lib.gated_workspace);
    take(at, "tam_gated", lib.gated);
    take(at, "tam_gated_backward", lib.gated_backward);
    take(at, "tam_cross_kept", lib.cross_kept);
    take(at, "tam_cross_reads_x", lib.cross_reads_x);
    take(at, "tam_cross_workspace", lib.cross_workspace);
    take(at, "tam_cross", lib.cross);
    take(at, "tam_cross_backward", lib.cross_backward);
    take(at, "tam_rotary_workspace", lib.rotary_workspace);
    take(at, "tam_rotary", lib.rotary);
    take(at, "tam_rotary_backward", lib.rotary_backward);
    take(at, "tam_last_error", lib.last_error);
  }, py::arg("addresses"));
  m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("residual"),
        py::arg("activation"));
  m.def("check_call", &check_call, py::arg("what"), py::arg("tensor"));
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
}
