// tam_layers.h -- what the layers' host sources (tam_layers.cpp, tam_decoder.cpp) share:
// the library's entries, checks of arguments, and tensors as the kernels take them.
#ifndef TAM_LAYERS_H
#define TAM_LAYERS_H

#include <torch/extension.h>

#include <ATen/TracerMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>

#include <string>

#include "../../include/turboadam_amd.h"

namespace py = pybind11;

namespace tam {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Library {
  decltype(&tam_linear_workspace) linear_workspace = nullptr;
  decltype(&tam_linear) linear = nullptr;
  decltype(&tam_linear_backward) linear_backward = nullptr;
  decltype(&tam_norm_workspace) norm_workspace = nullptr;
  decltype(&tam_norm) norm = nullptr;
  decltype(&tam_norm_backward) norm_backward = nullptr;
  decltype(&tam_gated_kept) gated_kept = nullptr;
  decltype(&tam_gated_workspace) gated_workspace = nullptr;
  decltype(&tam_gated) gated = nullptr;
  decltype(&tam_gated_backward) gated_backward = nullptr;
  decltype(&tam_cross_kept) cross_kept = nullptr;
  decltype(&tam_cross_reads_x) cross_reads_x = nullptr;
  decltype(&tam_cross_workspace) cross_workspace = nullptr;
  decltype(&tam_cross) cross = nullptr;
  decltype(&tam_cross_backward) cross_backward = nullptr;
  decltype(&tam_rotary_workspace) rotary_workspace = nullptr;
  decltype(&tam_rotary) rotary = nullptr;
  decltype(&tam_rotary_backward) rotary_backward = nullptr;
  decltype(&tam_last_error) last_error = nullptr;
};
inline Library lib;

constexpr int64_t kMostStride = int64_t(1) << 21;  // elements of a row stride the kernels take

[[noreturn]] inline void refuse(const std::string& what) { throw std::runtime_error("turboadam_amd." + what); }
[[noreturn]] inline void refuse_value(const std::string& what) { throw py::value_error("turboadam_amd." + what); }

inline void check(int rc, const char* what) {
  if (rc != TAM_OK)
    throw std::runtime_error("turboadam_amd: " + std::string(what) + " failed (code " + std::to_string(rc) +
                             "): " + lib.last_error());
}

inline std::string shape(const Tensor& t) { return c10::str("(", t.sizes(), ")"); }

inline int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TAM_DTYPE_F32;
    case at::kBFloat16: return TAM_DTYPE_BF16;
    case at::kHalf: return TAM_DTYPE_F16;
    default: return -1;
  }
}

inline void check_first(const char* what, const Tensor& x) {
  if (!x.is_cuda())
    refuse(c10::str(what, ": tensors must be on an MI355X (HIP) device, got ", x.device()));
  if (x.layout() != at::kStrided) refuse(c10::str(what, ": x must be dense, got ", x.layout()));
  if (dtype_of(x) < 0)
    refuse_value(c10::str(what, ": x must be float32, bfloat16 or float16, got ", x.scalar_type()));
}

inline void check_other(const char* what, const char* name, const Tensor& t, const Tensor& x) {
  if (t.device() != x.device() || t.layout() != at::kStrided)
    refuse(c10::str(what, ": ", name, " must be dense on ", x.device(), " with x, got ", t.layout(), " on ", t.device()));
  if (t.scalar_type() != x.scalar_type())
    refuse_value(c10::str(what, ": ", name, " must be ", x.scalar_type(), " as x is, got ", t.scalar_type()));
}

inline Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// t as memory holds it: its negative bit resolved, and zeros where it is one of
// autograd's zero tensors, which have no memory (a null address means "not given" to the
// kernels, and a missing weight is ones).
inline Tensor solid(const Tensor& t) {
  if (t._is_zerotensor()) return at::zeros(t.sizes(), t.options());
  return t.is_neg() ? t.resolve_neg() : t;
}

inline Tensor plain(const Tensor& t) { return t.defined() ? solid(t).contiguous() : t; }

// t as rows of `width` contiguous elements, and the stride between them.
inline Tensor rows_of(const Tensor& t, int64_t width, int64_t& ld) {
  int64_t n = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) n *= t.size(i);
  Tensor r = solid(t);
  if (r.dim() != 2) r = r.reshape({n, width});
  if ((width != 1 && r.stride(1) != 1) || (n > 1 && (r.stride(0) < width || r.stride(0) >= kMostStride)))
    r = r.contiguous();
  ld = n > 1 ? r.stride(0) : std::max<int64_t>(width, 1);
  return r;
}

inline Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

inline void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline bool wants_gradient(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A recorder of torch operations (torch.jit.trace, make_fx) would see the allocation of
// the output and not the kernel that fills it: its graph returns memory as it finds it.
inline void refuse_recording(const char* what) {
  if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(at::DispatchKey::PreDispatch) ||
      c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value())
    refuse(c10::str(what, ": cannot be recorded by torch.jit.trace or make_fx"));
}

// What the kernels write has no tangent: a dual tensor's would be lost, and everything
// behind the result would see a zero derivative. (Also under no_grad, where forward
// mode stays on, and in a backward pass whose gradient is dual.)
inline void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(0).defined())
      refuse(c10::str(what, ": has no forward-mode derivative, and an argument is a dual tensor"));
}

// The results of these backward passes come from raw memory: they have no graph.
inline void not_twice(const char* what) {
  if (at::GradMode::is_enabled())
    refuse(c10::str(what, ": its gradients cannot be differentiated again (create_graph=True)"));
}

// The weight, its row stride, and whether its rows are the inputs: a weight stored
// as (inputs, outputs) and passed as its transpose stays where it is.
inline Tensor weight_of(const Tensor& weight, int64_t& ld, bool& in_out) {
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

}  // namespace tam

#endif  // TAM_LAYERS_H
