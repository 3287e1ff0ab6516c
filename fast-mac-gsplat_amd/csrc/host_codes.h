// host_codes.h -- what the host paths of scenes in codes and of decoders by code
// share (host_codes.cpp, host_decoders.cpp).
#pragma once

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <vector>

#include "host_common.h"

namespace gs_host {

inline int dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GSPLAT_F32;
    case at::kBFloat16: return GSPLAT_BF16;
    case at::kHalf: return GSPLAT_F16;
    default: return -1;
  }
}

inline bool codes_ok(const Tensor& t) {
  return t.scalar_type() == at::kInt || t.scalar_type() == at::kLong;
}

// Elements between the rows of x, taken as [rows, C] without a copy; -1 where
// that takes one.
inline int64_t row_stride(const Tensor& x) {
  const int64_t nd = x.dim(), C = x.size(nd - 1);
  if (C > 1 && x.stride(nd - 1) != 1) return -1;
  int64_t stride = C, below = 1;  // (of one row: any)
  for (int64_t d = nd - 2; d >= 0; --d) {
    if (x.size(d) == 1) continue;
    if (x.size(d) == 0) return C;
    if (below == 1)
      stride = x.stride(d);
    else if (x.stride(d) != stride * below)
      return -1;
    below *= x.size(d);
  }
  return stride >= C ? stride : -1;
}

// x with its row stride, copied where the rows are not a constant stride apart.
inline Tensor rows_of(const Tensor& x, int64_t& stride) {
  stride = row_stride(x);
  if (stride >= 0) return x;
  stride = x.size(x.dim() - 1);
  return x.contiguous();
}

inline void* pointer(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* f32_or_null(const Tensor& t) {
  return t.defined() ? t.data_ptr<float>() : nullptr;
}
inline int32_t* i32(const Tensor& t) { return t.data_ptr<int32_t>(); }

inline at::TensorOptions plain_options(const Tensor& like) {
  return like.options().requires_grad(false);
}

inline std::vector<int64_t> with(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> s = sizes.vec();
  s.push_back(last);
  return s;
}

// These backwards cannot be differentiated: under create_graph their results
// carry a node, between them and the inputs they depend on, that says so when
// one tries.
inline variable_list once(variable_list g, const variable_list& inputs, const char* what) {
  if (!at::GradMode::is_enabled()) return g;
  std::vector<size_t> at;
  variable_list some;
  for (size_t k = 0; k < g.size(); ++k)
    if (g[k].defined()) {
      at.push_back(k);
      some.push_back(g[k].detach().requires_grad_(true));
    }
  for (const Tensor& t : inputs)
    if (t.defined()) some.push_back(t);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + ": its gradient cannot be differentiated again", some.size());
  some = (*node)(std::move(some));
  for (size_t k = 0; k < at.size(); ++k) g[at[k]] = some[k];
  return g;
}

inline PyObject* wrap_or_none(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

inline py::tuple tuple_of(std::initializer_list<Tensor> ts) {
  py::tuple out(ts.size());
  size_t k = 0;
  for (const Tensor& t : ts) out[k++] = py::reinterpret_steal<py::object>(wrap_or_none(t));
  return out;
}

}  // namespace gs_host
