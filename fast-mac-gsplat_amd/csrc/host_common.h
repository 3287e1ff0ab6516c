// host_common.h -- what the host paths share (host.cpp, host_codes.cpp): the C
// ABI's functions, checks, streams, which tensors the C++ paths take, and the
// Python layer's timing.
#pragma once

#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/PythonDispatcherTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <atomic>

#include "../../include/gsplat_hip.h"

namespace gs_host {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The C ABI, from the library that the Python layer has loaded.
#define GS_API(F)                       \
  F(last_error)                         \
  F(bin_workspace_bytes)                \
  F(render_workspace_bytes)             \
  F(bin_render_forward)                 \
  F(render_forward_long)                \
  F(render_backward)                    \
  F(direct_workspace_bytes)             \
  F(direct_pairs)                       \
  F(direct_render)                      \
  F(tile_workspace_bytes)               \
  F(tile_render)                        \
  F(project_forward)                    \
  F(project_backward)                   \
  F(project_backward_workspace_bytes)     \
  F(lookup_forward)                       \
  F(lookup_backward_workspace_bytes)      \
  F(lookup_backward)                      \
  F(code_probs_workspace_bytes)           \
  F(code_probs_forward)                   \
  F(code_probs_backward)                  \
  F(code_balance_workspace_bytes)         \
  F(code_balance_forward)                 \
  F(code_balance_backward)                \
  F(group_codes_workspace_bytes)          \
  F(group_codes)                          \
  F(rows_by_code)                         \
  F(rows_from_codes)                      \
  F(rows_from_codes_backward)             \
  F(code_adapters_workspace_bytes)        \
  F(code_adapters_forward)                \
  F(code_adapters_backward_workspace_bytes) \
  F(code_adapters_backward)               \
  F(clip_gradients_workspace_bytes)       \
  F(clip_gradients)
struct Api {
#define GS_POINTER(name) decltype(&gsplat_hip_##name) name = nullptr;
  GS_API(GS_POINTER)
#undef GS_POINTER
};
inline Api api;

inline void check(int rc, const char* what) {
  if (rc == 0) return;
  const char* msg = api.last_error();
  TORCH_CHECK(false, what, " failed (status ", rc, "): ", msg ? msg : "");
}

inline hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

constexpr int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

inline const float* f32(const Tensor& t) { return t.data_ptr<float>(); }

// A tensor the C++ paths take: an ordinary strided tensor in device memory, of
// a type whose operations nothing intercepts.
inline bool ordinary(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage())
    return false;
  const auto ks = t.key_set();
  if (ks.has_any(c10::DispatchKeySet(
          {c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
           c10::DispatchKey::FuncTorchGradWrapper,
           c10::DispatchKey::Functionalize})) ||
      t.is_conj() || t.is_neg())
    return false;
  return !t._fw_grad(0).defined();
}

inline bool plain(PyObject* o) {
  return ordinary(o) && THPVariable_Unpack(o).scalar_type() == at::kFloat;
}

// Nothing that intercepts operations is active (modes, functorch, tracing).
inline bool plain_context() {
  return !c10::impl::dispatch_mode_enabled() &&
         c10::impl::PythonDispatcherTLS::get_state() == nullptr &&
         !c10::impl::tls_is_dispatch_key_included(
             c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
         !torch::jit::tracer::isTracing();
}

// Timing of a backward call by the Python layer (_ops.set_timing): the
// context manager _ops._timed, entered around the C-ABI call.
inline std::atomic<bool> g_timed{false};
struct Timed {
  PyObject* cm = nullptr;
  explicit Timed(const char* name) {
    if (!g_timed.load(std::memory_order_relaxed)) return;
    py::gil_scoped_acquire gil;
    py::object ops = py::module_::import("torch_gsplat_bridge_fast._ops");
    py::object c = ops.attr("_timed")(name);
    c.attr("__enter__")();
    cm = c.release().ptr();
  }
  ~Timed() {
    if (cm == nullptr) return;
    py::gil_scoped_acquire gil;
    try {
      py::object c = py::reinterpret_steal<py::object>(cm);
      c.attr("__exit__")(py::none(), py::none(), py::none());
    } catch (py::error_already_set& e) {
      e.discard_as_unraisable("gsplat timing");
    }
  }
};

inline Tensor bytes(int64_t n, const Tensor& like) {
  return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false));
}

void def_codes(py::module_& m);
void def_decoders(py::module_& m);

}  // namespace gs_host
