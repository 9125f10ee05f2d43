// What the operators on real channels and over points have in common: checks of tensors, memory, the stream, and torch's own operations in
// their place where only those will do.
#pragma once

#include <torch/extension.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "gelib_hip.h"

namespace gelib_tensors {

namespace py = pybind11;

typedef std::optional<at::Tensor> Maybe;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

inline void done(int status) {
  if (status == GELIB_HIP_OK) return;
  std::string why = gelib_hip_strerror(status);
  if (status == GELIB_HIP_ERR_RUNTIME) why += std::string(": ") + gelib_hip_last_runtime_error();
  throw std::runtime_error("GElib error: " + why + " (status " + std::to_string(status) + ")");
}

inline int type_of(const at::Tensor &x) {
  switch (x.scalar_type()) {
    case at::kFloat: return GELIB_HIP_F32;
    case at::kBFloat16: return GELIB_HIP_BF16;
    case at::kHalf: return GELIB_HIP_F16;
    default: throw py::type_error("GElib: float32, bfloat16 and float16 tensors are taken");
  }
}

inline void like(const at::Tensor &t, const at::Tensor &x, const char *name) {
  if (t.scalar_type() != x.scalar_type()) throw py::type_error(std::string("GElib: ") + name + " has another type than x");
  if (t.device() != x.device()) throw py::value_error(std::string("GElib: ") + name + " is on another device than x");
}

inline void on_gpu(const at::Tensor &x) {
  if (!x.is_cuda()) throw py::value_error("GElib: tensors must be on GPU: these operators have no host form in this build");
}

// t packed, and from a multiple of 16 bytes on
inline at::Tensor plain(const at::Tensor &t) {
  if (!t.is_neg() && t.is_contiguous() && (t.numel() == 0 || (uintptr_t)t.data_ptr() % 16 == 0)) return t;   // (no dispatch)
  const at::Tensor p = t.resolve_neg().contiguous();
  return p.numel() && (uintptr_t)p.data_ptr() % 16 ? p.clone() : p;
}

// Is a call left to torch's own operations?  Only they know of forward-mode derivatives, function transforms, tracing, dispatch modes
// (shapes without data, counters of operations) and batches of gradients: a kernel would read the memory below, and its result would be a constant to them.
inline bool left_to_torch(std::initializer_list<const at::Tensor *> ts) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::any_modes_set() ||
      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
    return true;
  for (const at::Tensor *t : ts)
    if (t && t->defined() && (t->_fw_grad(/*level=*/0).defined() || t->unsafeGetTensorImpl()->is_python_dispatch() || !t->has_storage())) return true;
  return false;
}
inline const at::Tensor *address(const Maybe &t) { return t ? &*t : nullptr; }

inline void *ptr(const at::Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }

struct OnDevice {
  c10::OptionalDeviceGuard guard;
  void *stream;
  explicit OnDevice(const at::Tensor &x) : guard(x.device()), stream((void *)c10::hip::getCurrentHIPStream(x.device().index()).stream()) {}
};

inline at::Tensor workspace(uint64_t bytes, const at::Tensor &x) {
  return bytes ? at::empty({(int64_t)bytes}, x.options().dtype(at::kByte)) : at::Tensor();
}

struct Rows {   // x as rows: itself where they are evenly spaced, contiguous and aligned as packed ones are, else a copy
  at::Tensor x;
  int64_t rows, stride;
  int K;
};
inline Rows rows_of(const at::Tensor &t) {
  Rows r;
  r.x = t.is_neg() ? t.resolve_neg() : t;
  const int64_t d = t.dim();
  r.K = (int)t.size(d - 1), r.rows = 1;
  bool even = t.stride(d - 1) == 1 || r.K == 1;
  int64_t step = -1;
  for (int64_t k = d - 2; k >= 0; k--) {
    if (t.size(k) != 1 && even) {
      if (step < 0) step = r.x.stride(k);
      else even = r.x.stride(k) == step * r.rows;
    }
    r.rows *= t.size(k);
  }
  const int64_t width = r.K * t.element_size() % 16 == 0 ? 16 : 1;
  if (even) even = (step < 0 || step * t.element_size() % width == 0) && (uintptr_t)r.x.data_ptr() % width == 0;
  if (!even || r.x.numel() == 0) {
    r.x = r.x.is_contiguous() ? r.x.clone() : r.x.contiguous();
    step = r.K;
  }
  r.stride = step < 0 ? r.K : step;
  return r;
}

// torch's operations in the types that are written here: under autocast a product of float32 values would be one of 16-bit values.
struct AsWritten {
  c10::impl::ExcludeDispatchKeyGuard guard{c10::autocast_dispatch_keyset};
};

// Gradients of f(tensors) for those that need one, with a graph of their own where the caller wants one.
template <typename F>
inline variable_list graph_grads(F f, const variable_list &tensors, const at::Tensor &g) {
  const bool graph = at::GradMode::is_enabled();
  AsWritten types;
  at::AutoGradMode on(true);
  variable_list views, wanted, grads(tensors.size());
  for (const at::Tensor &t : tensors) {
    views.push_back(t.defined() ? t.view_as(t) : t);   // (one tensor may stand in two places)
    if (t.defined() && t.requires_grad()) wanted.push_back(views.back());
  }
  if (wanted.empty()) return grads;
  const variable_list got = torch::autograd::grad({f(views)}, wanted, {g}, /*retain_graph=*/graph, /*create_graph=*/graph);
  size_t k = 0;
  for (size_t i = 0; i < tensors.size(); i++)
    if (tensors[i].defined() && tensors[i].requires_grad()) grads[i] = got[k++];
  return grads;
}

inline at::Tensor some(const Maybe &t) { return t ? *t : at::Tensor(); }
inline Maybe some(const at::Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }
inline bool needs(const at::Tensor &t) { return t.defined() && t.requires_grad(); }

}  // namespace gelib_tensors
