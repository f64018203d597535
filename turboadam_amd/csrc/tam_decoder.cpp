// tam_decoder.cpp -- gated_linear, linear_cross_entropy and rotary for torch: argument
// checks, outputs and workspaces, and the autograd nodes of their backward passes (part of
// the torch extension module _tam_host).
#include "tam_layers.h"

#include <cfloat>

namespace {

using namespace tam;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool any_gradient(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (wants_gradient(*t)) return true;
  return false;
}

// ------------------------------------------------------------ gated linear
struct GatedCall {
  TamGated d = {};
  Tensor x, gate, up;  // what d points at
  bool in_out;

  GatedCall(const Tensor& x0, const Tensor& gate0, const Tensor& up0, int64_t activation) {
    int64_t ldx, ldw, ldu;
    bool up_in_out;
    x = rows_of(x0, gate0.size(1), ldx);
    gate = weight_of(gate0, ldw, in_out);
    up = weight_of(up0, ldu, up_in_out);
    if (in_out != up_in_out || ldw != ldu) {  // the kernels take both laid out the same way
      gate = plain(gate0);
      up = plain(up0);
      in_out = false;
      ldw = std::max<int64_t>(gate.size(1), 1);
    }
    d.x = x.data_ptr();
    d.gate = gate.data_ptr();
    d.up = up.data_ptr();
    d.rows = x.size(0);
    d.inputs = x.size(1);
    d.outputs = gate.size(0);
    d.ldx = ldx;
    d.ldw = ldw;
    d.w_in_out = in_out;
    d.dtype = dtype_of(x);
    d.activation = (uint32_t)activation;
  }

  void run(bool backward) {
    const char* what = backward ? "tam_gated_backward" : "tam_gated";
    size_t need = 0;
    check(lib.gated_workspace(&d, backward, &need), what);
    const Tensor ws = workspace(need, x);
    check((backward ? lib.gated_backward : lib.gated)(&d, ptr(ws), need, stream_of(x)), what);
  }
};

Tensor gated_forward(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation, Tensor* kept) {
  const c10::DeviceGuard guard(x.device());
  GatedCall c(x, gate, up, activation);
  auto sizes = x.sizes().vec();
  sizes.back() = gate.size(0);
  const Tensor h = at::empty(sizes, x.options().requires_grad(false));
  if (kept) {
    *kept = workspace(lib.gated_kept(c.d.rows, c.d.outputs, c.d.dtype), x);
    c.d.kept = ptr(*kept);
  }
  c.d.h = h.data_ptr();
  c.run(false);
  return h;
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation) {
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor kept;
    const Tensor h = gated_forward(x, gate, up, activation, &kept);
    ctx->save_for_backward({x, gate, up, kept});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["wants"] =
        (int64_t)((wants_gradient(x) ? 1 : 0) | (wants_gradient(gate) ? 2 : 0) | (wants_gradient(up) ? 4 : 0));
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_twice("gated_linear");
    refuse_recording("gated_linear");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], dh = grads[0];
    refuse_tangents("gated_linear", {&dh});
    const int64_t wants = ctx->saved_data["wants"].toInt();
    Tensor dx, dgate, dup;
    if (dh.defined() && wants) {
      const c10::DeviceGuard guard(x.device());
      GatedCall c(x, saved[1], saved[2], ctx->saved_data["activation"].toInt());
      const Tensor d = plain(dh);
      const auto options = x.options().requires_grad(false);
      const int64_t outputs = saved[1].size(0), inputs = saved[1].size(1);
      auto weight = [&] {  // laid out as the weights
        return c.in_out ? at::empty({inputs, outputs}, options) : at::empty({outputs, inputs}, options);
      };
      if (wants & 1) dx = at::empty(x.sizes(), options);
      if (wants & 2) dgate = weight();
      if (wants & 4) dup = weight();
      c.d.dh = d.data_ptr();
      c.d.kept = ptr(saved[3]);
      c.d.dx = ptr(dx);
      c.d.dgate = ptr(dgate);
      c.d.dup = ptr(dup);
      c.run(true);
      if (c.in_out) {
        if (dgate.defined()) dgate = dgate.t();
        if (dup.defined()) dup = dup.t();
      }
    }
    return {dx, dgate, dup, Tensor()};
  }
};

Tensor gated_linear(const Tensor& x, const Tensor& gate, const Tensor& up, int64_t activation) {
  check_first("gated_linear", x);
  refuse_recording("gated_linear");
  check_other("gated_linear", "gate", gate, x);
  check_other("gated_linear", "up", up, x);
  if (gate.dim() != 2 || x.dim() < 1 || x.size(-1) != gate.size(1))
    refuse_value(c10::str("gated_linear: x ", shape(x), " and gate ", shape(gate),
                          " are not (..., inputs) and (outputs, inputs)"));
  if (up.sizes() != gate.sizes())
    refuse_value(c10::str("gated_linear: up must have gate's shape ", shape(gate), ", got ", shape(up)));
  refuse_tangents("gated_linear", {&x, &gate, &up});
  if (any_gradient({&x, &gate, &up})) return GatedLinear::apply(x, gate, up, activation);
  return gated_forward(x, gate, up, activation, nullptr);
}

// --------------------------------------------- projection and cross entropy
struct CrossCall {
  TamCross d = {};
  Tensor x, w;  // what d points at

  // x0: of `rows` rows, or undefined (a backward pass that does not read it)
  CrossCall(const Tensor& x0, const Tensor& weight, int64_t rows, int64_t reduction, int64_t ignored) {
    int64_t ldx = std::max<int64_t>(weight.size(1), 1), ldw;
    if (x0.defined()) x = rows_of(x0, x0.size(-1), ldx);
    w = rows_of(weight, weight.size(1), ldw);
    d.x = ptr(x);
    d.w = w.data_ptr();
    d.rows = rows;
    d.inputs = weight.size(1);
    d.vocabulary = w.size(0);
    d.ldx = ldx;
    d.ldw = ldw;
    d.ignored = ignored;
    d.dtype = dtype_of(w);
    d.reduction = (uint32_t)reduction;
  }

  void run(bool backward) {
    const char* what = backward ? "tam_cross_backward" : "tam_cross";
    size_t need = 0;
    check(lib.cross_workspace(&d, backward, &need), what);
    const Tensor ws = workspace(need, w);
    check((backward ? lib.cross_backward : lib.cross)(&d, ptr(ws), need, stream_of(w)), what);
  }
};

Tensor cross_forward(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t reduction, int64_t ignored,
                     Tensor* kept, bool* reads_x) {
  const c10::DeviceGuard guard(x.device());
  CrossCall c(x, weight, target.numel(), reduction, ignored);
  const auto options = x.options().requires_grad(false).dtype(at::kFloat);
  const Tensor loss = reduction == TAM_CROSS_NONE ? at::empty(target.sizes(), options) : at::empty({}, options);
  const Tensor t = plain(target);
  if (kept) {
    *kept = workspace(lib.cross_kept(&c.d), x);
    *reads_x = lib.cross_reads_x(&c.d) != 0;
    c.d.kept = kept->data_ptr();
  }
  c.d.target = static_cast<const int64_t*>(t.data_ptr());
  c.d.loss = static_cast<float*>(loss.data_ptr());
  c.run(false);
  return loss;
}

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& target, int64_t reduction,
                        int64_t ignored) {
    at::AutoDispatchBelowADInplaceOrView below;
    Tensor kept;
    bool reads_x = false;
    const Tensor loss = cross_forward(x, weight, target, reduction, ignored, &kept, &reads_x);
    // otherwise what is kept holds its rows that count
    ctx->save_for_backward({reads_x ? x : Tensor(), weight, kept});
    ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["ignored"] = ignored;
    ctx->saved_data["wants"] = (int64_t)((wants_gradient(x) ? 1 : 0) | (wants_gradient(weight) ? 2 : 0));
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_twice("linear_cross_entropy");
    refuse_recording("linear_cross_entropy");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], dloss = grads[0];
    refuse_tangents("linear_cross_entropy", {&dloss});
    const int64_t wants = ctx->saved_data["wants"].toInt();
    Tensor dx, dw;
    if (dloss.defined() && wants) {
      const c10::DeviceGuard guard(weight.device());
      const auto sizes = ctx->saved_data["sizes"].toIntVector();
      int64_t rows = 1;
      for (size_t i = 0; i + 1 < sizes.size(); ++i) rows *= sizes[i];
      CrossCall c(x, weight, rows, ctx->saved_data["reduction"].toInt(), ctx->saved_data["ignored"].toInt());
      const auto options = weight.options().requires_grad(false);
      Tensor d = solid(dloss);
      // a gradient of one number for all rows (that of a sum) is read as it is
      bool one = d.dim() > 0 && d.numel() > 0;
      for (int64_t i = 0; i < d.dim(); ++i) one = one && (d.size(i) == 1 || d.stride(i) == 0);
      if (!one) d = d.contiguous();
      if (wants & 1) dx = at::empty(sizes, options);
      if (wants & 2) dw = at::empty(weight.sizes(), options);
      c.d.kept = saved[2].data_ptr();
      c.d.dloss = static_cast<const float*>(d.data_ptr());
      c.d.dloss_stride = one ? 0 : 1;
      c.d.dx = ptr(dx);
      c.d.dw = ptr(dw);
      c.run(true);
    }
    return {dx, dw, Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& target, int64_t reduction, int64_t ignored) {
  const char* me = "linear_cross_entropy";
  check_first(me, x);
  refuse_recording(me);
  check_other(me, "weight", weight, x);
  if (weight.dim() != 2 || x.dim() < 1 || x.size(-1) != weight.size(1))
    refuse_value(c10::str(me, ": x ", shape(x), " and weight ", shape(weight), " are not (..., inputs) and (vocabulary, inputs)"));
  if (target.device() != x.device() || target.layout() != at::kStrided)
    refuse(c10::str(me, ": target must be dense on ", x.device(), " with x, got ", target.layout(), " on ", target.device()));
  if (target.scalar_type() != at::kLong) refuse_value(c10::str(me, ": target must be int64, got ", target.scalar_type()));
  if (target.sizes() != x.sizes().slice(0, x.dim() - 1))
    refuse_value(c10::str(me, ": target must have shape (", x.sizes().slice(0, x.dim() - 1), "), got ", shape(target)));
  if (weight.size(0) == 0 && target.numel()) refuse_value(c10::str(me, ": the vocabulary is empty"));
  refuse_tangents(me, {&x, &weight});
  if (any_gradient({&x, &weight})) return CrossEntropy::apply(x, weight, target, reduction, ignored);
  return cross_forward(x, weight, target, reduction, ignored, nullptr, nullptr);
}

// ------------------------------------------------------------------ rotary
struct Turn {
  bool interleaved;
  double magnitude, eps;
};

// Elements between two heads that the kernels' 32-bit offsets do not reach: 2^31 bytes for the heads that a
// wave of 64 lanes takes at once, of a lane to 16 elements.
int64_t too_far(const Tensor& like, int64_t rotated) {
  const int64_t units = (rotated / 2 + 7) / 8 + (like.size(-1) - rotated + 15) / 16;
  int64_t lanes = 1;
  while (lanes < units && lanes < 64) lanes *= 2;
  return (int64_t(1) << 31) / like.element_size() / (64 / lanes);
}

// t as (batch, tokens, heads, dim) with contiguous heads, in place where its strides allow.
Tensor heads_of(const Tensor& t0, int64_t far) {
  Tensor t = solid(t0);
  const int64_t n = t.dim();
  if (n == 3) t = t.unsqueeze(0);
  if (n > 4) {
    int64_t batch = 1;
    for (int64_t i = 0; i + 3 < n; ++i) batch *= t.size(i);
    t = t.reshape({batch, t.size(n - 3), t.size(n - 2), t.size(n - 1)});
  }
  return (t.size(3) > 1 && t.stride(3) != 1) || (t.size(2) > 1 && t.stride(2) >= far) ? t.contiguous() : t;
}

// A tensor for results in t's order of dimensions (in place of a slice: without its gaps).
Tensor result_of(const Tensor& t) {
  const auto options = t.options().requires_grad(false);
  const Tensor y = at::empty_like(t, options, at::MemoryFormat::Preserve);
  return y.size(-1) > 1 && y.stride(-1) != 1 ? at::empty(t.sizes(), options) : y;
}

struct RotaryCall {
  TamRotary d = {};
  std::vector<Tensor> held;  // what d points at
  int64_t far;

  RotaryCall(const Tensor& like, const Tensor& positions, const Tensor& frequencies, const Turn& turn) {
    const int64_t n = like.dim();
    d.tokens = like.size(n - 3);
    d.batch = 1;
    for (int64_t i = 0; i + 3 < n; ++i) d.batch *= like.size(i);
    d.dim = like.size(n - 1);
    d.rotated = 2 * frequencies.size(0);
    far = too_far(like, (int64_t)d.rotated);
    d.dtype = dtype_of(like);
    d.interleaved = turn.interleaved;
    d.magnitude = (float)turn.magnitude;
    d.eps = (float)turn.eps;
    Tensor p = positions.expand(like.sizes().slice(0, n - 2));
    if (n == 3) p = p.unsqueeze(0);
    if (n > 4) p = p.reshape({(int64_t)d.batch, (int64_t)d.tokens});
    d.positions = p.data_ptr();
    d.positions64 = p.scalar_type() == at::kLong;
    d.pos_b = p.stride(0);
    d.pos_t = p.stride(1);
    const Tensor f = frequencies.contiguous();
    d.frequencies = static_cast<const double*>(f.data_ptr());
    held = {p, f};
  }

  void input(TamHeads& h, const Tensor& x) {
    const Tensor t = heads_of(x, far);
    h.heads = t.size(2);
    h.x = t.data_ptr();
    h.x_b = t.stride(0);
    h.x_t = t.stride(1);
    h.x_h = t.size(2) > 1 ? t.stride(2) : 0;
    held.push_back(t);
  }
  void gradient(TamHeads& h, const Tensor& dy) {
    const Tensor t = heads_of(dy, far);
    h.heads = t.size(2);
    h.dy = t.data_ptr();
    h.dy_b = t.stride(0);
    h.dy_t = t.stride(1);
    h.dy_h = t.size(2) > 1 ? t.stride(2) : 0;
    held.push_back(t);
  }
  void weight(TamHeads& h, const Tensor& w) {
    if (!w.defined()) return;
    const Tensor t = plain(w);
    h.w = t.data_ptr();
    held.push_back(t);
  }
  Tensor output(TamHeads& h, const Tensor& like) {
    Tensor y = result_of(like);
    if (!y.is_contiguous() && (y.dim() > 4 || y.stride(-2) >= far)) y = at::empty(like.sizes(), y.options());
    const Tensor t = heads_of(y, far);
    h.y = t.data_ptr();
    h.y_b = t.stride(0);
    h.y_t = t.stride(1);
    h.y_h = t.size(2) > 1 ? t.stride(2) : 0;
    return y;
  }
};

variable_list rotary_forward(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& frequencies,
                             const Tensor& q_weight, const Tensor& k_weight, const Turn& turn) {
  const c10::DeviceGuard guard(q.device());
  RotaryCall c(q, positions, frequencies, turn);
  variable_list out;
  c.input(c.d.q, q);
  c.weight(c.d.q, q_weight);
  out.push_back(c.output(c.d.q, q));
  if (k.defined()) {
    c.input(c.d.k, k);
    c.weight(c.d.k, k_weight);
    out.push_back(c.output(c.d.k, k));
  }
  check(lib.rotary(&c.d, stream_of(q)), "tam_rotary");
  return out;
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions,
                               const Tensor& frequencies, const OptTensor& q_weight, const OptTensor& k_weight,
                               bool interleaved, double magnitude, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->set_materialize_grads(false);
    const Tensor key = given(k), wq = given(q_weight), wk = given(k_weight);
    auto out = rotary_forward(q, key, positions, frequencies, wq, wk, Turn{interleaved, magnitude, eps});
    // heads without a norm are only turned back
    ctx->save_for_backward({wq.defined() ? q : Tensor(), wk.defined() ? key : Tensor(), positions, frequencies, wq, wk});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["wants"] = (int64_t)((wants_gradient(q) ? 1 : 0) | (wants_gradient(key) ? 2 : 0) |
                                         (wants_gradient(wq) ? 4 : 0) | (wants_gradient(wk) ? 8 : 0));
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_twice("rotary");
    refuse_recording("rotary");
    const auto saved = ctx->get_saved_variables();
    const int64_t wants = ctx->saved_data["wants"].toInt();
    const Tensor none, &dq = grads[0], &dk = grads.size() > 1 ? grads[1] : none;
    refuse_tangents("rotary", {&dq, &dk});
    Tensor d[2], dw[2];
    const bool with[2] = {dq.defined() && (wants & 5), dk.defined() && (wants & 10)};
    if (with[0] || with[1]) {
      const Tensor& like = with[0] ? dq : dk;
      const c10::DeviceGuard guard(like.device());
      RotaryCall c(like, saved[2], saved[3], Turn{ctx->saved_data["interleaved"].toBool(), ctx->saved_data["magnitude"].toDouble(),
                                                  ctx->saved_data["eps"].toDouble()});
      for (int i = 0; i < 2; ++i) {
        if (!with[i]) continue;
        TamHeads& h = i ? c.d.k : c.d.q;
        const Tensor &x = saved[i], &w = saved[4 + i], &dy = i ? dk : dq;
        c.gradient(h, dy);
        if (w.defined()) c.input(h, x);
        c.weight(h, w);
        d[i] = c.output(h, w.defined() ? x : dy);
        if (wants & (4 << i)) {
          dw[i] = at::empty(w.sizes(), w.options().requires_grad(false));
          h.dw = dw[i].data_ptr();
        }
      }
      size_t need = 0;
      check(lib.rotary_workspace(&c.d, 1, &need), "tam_rotary_backward");
      const Tensor ws = workspace(need, like);
      check(lib.rotary_backward(&c.d, ptr(ws), need, stream_of(like)), "tam_rotary_backward");
    }
    return {wants & 1 ? d[0] : none, wants & 2 ? d[1] : none, none, none, dw[0], dw[1], none, none, none};
  }
};

variable_list rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& frequencies, bool interleaved,
                     double magnitude, const OptTensor& q_weight, const OptTensor& k_weight, double eps) {
  check_first("rotary", q);
  refuse_recording("rotary");
  const int64_t n = q.dim();
  if (n < 3 || q.size(n - 1) < 1)
    refuse_value(c10::str("rotary: q must be (..., tokens, heads, dim), got ", shape(q)));
  if (k) {
    check_other("rotary", "k", *k, q);
    auto sizes = q.sizes().vec();
    if (k->dim() == n) sizes[n - 2] = k->size(n - 2);
    if (k->sizes() != at::IntArrayRef(sizes))
      refuse_value(c10::str("rotary: k must have q's shape ", shape(q), " but for its heads, got ", shape(*k)));
  }
  for (const auto& [name, t] : {std::pair<const char*, const Tensor*>("positions", &positions), {"frequencies", &frequencies}})
    if (t->device() != q.device() || t->layout() != at::kStrided)
      refuse(c10::str("rotary: ", name, " must be dense on ", q.device(), " with q, got ", t->layout(), " on ", t->device()));
  if (positions.scalar_type() != at::kLong && positions.scalar_type() != at::kInt)
    refuse_value(c10::str("rotary: positions must be int64 or int32, got ", positions.scalar_type()));
  bool fits = positions.dim() <= n - 2;
  for (int64_t i = 1; fits && i <= positions.dim(); ++i)
    fits = positions.size(-i) == 1 || positions.size(-i) == q.size(n - 2 - i);
  if (!fits)
    refuse_value(c10::str("rotary: positions must broadcast to (", q.sizes().slice(0, n - 2), "), got ", shape(positions)));
  if (frequencies.scalar_type() != at::kDouble || frequencies.dim() != 1 || 2 * frequencies.size(0) > q.size(n - 1))
    refuse_value(c10::str("rotary: frequencies must be float64 (pairs,) with at most ", q.size(n - 1) / 2, " pairs, got ",
                          frequencies.scalar_type(), " ", shape(frequencies)));
  if (frequencies.requires_grad() && at::GradMode::is_enabled()) refuse("rotary: frequencies have no gradient");
  const float eps32 = (float)eps;  // as the kernels take it
  if (!(eps == 0 || (eps32 >= FLT_MIN && eps32 <= FLT_MAX)))
    refuse_value(c10::str("rotary: eps must be 0 or in float32's normal numbers, got ", eps));
  if (k_weight && !k) refuse_value("rotary: k_weight without k");
  for (const auto& [name, t] : {std::pair<const char*, const OptTensor&>("q_weight", q_weight), {"k_weight", k_weight}})
    if (t) {
      check_other("rotary", name, *t, q);
      if (t->dim() != 1 || t->size(0) != q.size(n - 1))
        refuse_value(c10::str("rotary: ", name, " must have shape (", q.size(n - 1), ",), got ", shape(*t)));
    }
  const Tensor key = given(k), wq = given(q_weight), wk = given(k_weight);
  refuse_tangents("rotary", {&q, &key, &wq, &wk, &frequencies});
  if (any_gradient({&q, &key, &wq, &wk}))
    return Rotary::apply(q, k, positions, frequencies, q_weight, k_weight, interleaved, magnitude, eps);
  return rotary_forward(q, key, positions, frequencies, wq, wk, Turn{interleaved, magnitude, eps});
}

}  // namespace

void tam_register_decoder(py::module_& m) {
  m.def("gated_linear", &gated_linear, py::arg("x"), py::arg("gate"), py::arg("up"), py::arg("activation"));
  m.def("linear_cross_entropy", &linear_cross_entropy, py::arg("x"), py::arg("weight"), py::arg("target"),
        py::arg("reduction"), py::arg("ignored"));
  m.def("rotary", &rotary, py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("frequencies"), py::arg("interleaved"),
        py::arg("magnitude"), py::arg("q_weight"), py::arg("k_weight"), py::arg("eps"));
}
