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
#include <torch/extension.h>

#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <string>

#include "../../include/turboadam_amd.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Library {
  decltype(&tam_linear_workspace) linear_workspace = nullptr;
  decltype(&tam_linear) linear = nullptr;
  decltype(&tam_linear_backward) linear_backward = nullptr;
  decltype(&tam_norm_workspace) norm_workspace = nullptr;
  decltype(&tam_norm) norm = nullptr;
  decltype(&tam_norm_backward) norm_backward = nullptr;
  decltype(&tam_last_error) last_error = nullptr;
};
Library lib;

constexpr int64_t kMostStride = int64_t(1) << 21;  // elements of a row stride the kernels take
constexpr int64_t kMostNorm = 32768;               // elements of a layer norm's row

[[noreturn]] void refuse(const std::string& what) { throw std::runtime_error("turboadam_amd." + what); }
[[noreturn]] void refuse_value(const std::string& what) { throw py::value_error("turboadam_amd." + what); }

void check(int rc, const char* what) {
  if (rc != TAM_OK)
    throw std::runtime_error("turboadam_amd: " + std::string(what) + " failed (code " + std::to_string(rc) +
                             "): " + lib.last_error());
}

std::string shape(const Tensor& t) { return c10::str("(", t.sizes(), ")"); }

int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TAM_DTYPE_F32;
    case at::kBFloat16: return TAM_DTYPE_BF16;
    case at::kHalf: return TAM_DTYPE_F16;
    default: return -1;
  }
}

void check_first(const char* what, const Tensor& x) {
  if (!x.is_cuda())
    refuse(c10::str(what, ": tensors must be on an MI355X (HIP) device, got ", x.device()));
  if (x.layout() != at::kStrided) refuse(c10::str(what, ": x must be dense, got ", x.layout()));
  if (dtype_of(x) < 0)
    refuse_value(c10::str(what, ": x must be float32, bfloat16 or float16, got ", x.scalar_type()));
}

void check_other(const char* what, const char* name, const Tensor& t, const Tensor& x) {
  if (t.device() != x.device() || t.layout() != at::kStrided)
    refuse(c10::str(what, ": ", name, " must be dense on ", x.device(), " with x, got ", t.layout(), " on ", t.device()));
  if (t.scalar_type() != x.scalar_type())
    refuse_value(c10::str(what, ": ", name, " must be ", x.scalar_type(), " as x is, got ", t.scalar_type()));
}

Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// t as memory holds it: its negative bit resolved, and zeros where it is one of
// autograd's zero tensors, which have no memory (a null address means "not given" to the
// kernels, and a missing weight is ones).
Tensor solid(const Tensor& t) {
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}

Tensor plain(const Tensor& t) { return t.defined() ? solid(t).contiguous() : t; }

// t as rows of `width` contiguous elements, and the stride between them.
Tensor rows_of(const Tensor& t, int64_t width, int64_t& ld) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  Tensor r = solid(t);
  if (r.dim() != 2) r = r.reshape({n, width});
  if ((width != 1 && r.stride(1) != 1) || (n > 1 && (r.stride(0) < width || r.stride(0) >= kMostStride)))
    r = r.contiguous();
  ld = n > 1 ? r.stride(0) : std::max<int64_t>(width, 1);
  return r;
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

bool wants_gradient(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A recorder of torch operations (torch.jit.trace, make_fx) would see the allocation of
// the output and not the kernel that fills it: its graph returns memory as it finds it.
void refuse_recording(const char* what) {
  if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(at::DispatchKey::PreDispatch) ||
      c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value())
    refuse(c10::str(what, ": cannot be recorded by torch.jit.trace or make_fx"));
}

// What the kernels write has no tangent: a dual tensor's would be lost, and everything
// behind the result would see a zero derivative. (Also under no_grad, where forward
// mode stays on, and in a backward pass whose gradient is dual.)
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(0).defined())
      refuse(c10::str(what, ": has no forward-mode derivative, and an argument is a dual tensor"));
}

// The results of these backward passes come from raw memory: they have no graph.
void not_twice(const char* what) {
  if (at::GradMode::is_enabled())
    refuse(c10::str(what, ": its gradients cannot be differentiated again (create_graph=True)"));
}

// ------------------------------------------------------------------ linear
// The weight, its row stride, and whether its rows are the inputs: a weight stored
// as (inputs, outputs) and passed as its transpose stays where it is.
Tensor weight_of(const Tensor& weight, int64_t& ld, bool& in_out) {
  Tensor w = solid(weight);
  const int64_t outputs = w.size(0), inputs = w.size(1);
  in_out = false;
  if ((inputs == 1 || w.stride(1) == 1) &&
      (outputs == 1 || (w.stride(0) >= inputs && w.stride(0) < kMostStride))) {
    ld = outputs > 1 ? w.stride(0) : std::max<int64_t>(inputs, 1);
    return w;
  }
  if ((outputs == 1 || w.stride(0) == 1) &&
      (inputs == 1 || (w.stride(1) >= outputs && w.stride(1) < kMostStride))) {
    in_out = true;
    ld = inputs > 1 ? w.stride(1) : std::max<int64_t>(outputs, 1);
    return w;
  }
  ld = std::max<int64_t>(inputs, 1);
  return w.contiguous();
}

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
    take(at, "tam_last_error", lib.last_error);
  }, py::arg("addresses"));
  m.def("linear", &linear, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("residual"),
        py::arg("activation"));
  m.def("check_call", &check_call, py::arg("what"), py::arg("tensor"));
  m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"));
}
