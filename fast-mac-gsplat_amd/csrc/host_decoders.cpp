// host_decoders.cpp -- the host path of decoders by code and of clipping in C++:
// argument checks, buffers, the C-ABI calls and the autograd nodes of
// group_codes, rows_by_code, rows_from_codes, code_adapters and clip_gradients.
//
// As in host_codes.cpp, what is not the plain case returns None, and the Python
// layer's operators take it, with its messages.
#include <algorithm>
#include <cmath>
#include <optional>

#include "host_codes.h"

namespace gs_host {
namespace {

constexpr int64_t kMostRows = int64_t(1) << 29;

// The groups of a call: contiguous int32 tensors on one device.
struct Groups {
  Tensor order, places, starts;
  int64_t choices() const { return places.size(places.dim() - 1); }
  at::IntArrayRef splats() const { return places.sizes().slice(0, places.dim() - 1); }
};

bool index_ok(py::handle o, const c10::Device& device) {
  if (!ordinary(o.ptr())) return false;
  const Tensor& t = THPVariable_Unpack(o.ptr());
  return t.scalar_type() == at::kInt && t.device() == device;
}

bool groups_of(py::handle order, py::handle places, py::handle starts, const c10::Device& device,
               Groups& g) {
  if (!index_ok(order, device) || !index_ok(places, device) || !index_ok(starts, device)) return false;
  const Tensor &o = THPVariable_Unpack(order.ptr()), &p = THPVariable_Unpack(places.ptr()),
               &s = THPVariable_Unpack(starts.ptr());
  if (o.dim() != 1 || p.dim() < 1 || s.dim() != 1 || s.numel() < 2) return false;
  if (o.numel() != p.numel() || p.size(p.dim() - 1) == 0 || o.numel() > kMostRows) return false;
  if (p.size(p.dim() - 1) > GSPLAT_MAX_CHOICES) return false;
  g = Groups{o.contiguous(), p.contiguous(), s.contiguous()};
  return true;
}

const int32_t* ids(const Tensor& t) { return t.data_ptr<int32_t>(); }

// ---- sorting

py::object group(py::handle codes, int64_t num_codes, bool several) {
  if (!ordinary(codes.ptr()) || !plain_context()) return py::none();
  const Tensor& given = THPVariable_Unpack(codes.ptr());
  if (!codes_ok(given) || num_codes < 1 || num_codes > GSPLAT_MAX_CODES) return py::none();
  if (given.numel() > kMostRows) return py::none();
  const int64_t nd = given.dim();
  if (several && (nd < 1 || given.size(nd - 1) == 0 || given.size(nd - 1) > GSPLAT_MAX_CHOICES))
    return py::none();
  const c10::DeviceGuard device(given.device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor c = given.contiguous();
  const auto opt = c.options().dtype(at::kInt);
  const Tensor order = at::empty({c.numel()}, opt);
  const Tensor places = at::empty(several ? c.sizes().vec() : with(c.sizes(), 1), opt);
  const Tensor starts = at::empty({num_codes + 1}, opt);
  const gsplat_group_meta meta{c.numel(), (int32_t)num_codes, (int32_t)c.element_size()};
  const size_t n = api.group_codes_workspace_bytes(&meta);
  const Tensor ws = n > 0 ? bytes((int64_t)n, c) : Tensor();
  {
    const Timed timed("group_codes");
    check(api.group_codes(&meta, c.data_ptr(), i32(order), i32(places), i32(starts), pointer(ws), n,
                          stream_of(c)),
          "gsplat_hip_group_codes");
  }
  return tuple_of({order, places, starts});
}

// ---- rows by code

gsplat_rows_meta rows_meta(const Tensor& rows, int64_t stride, const Tensor& places) {
  const int64_t S = places.size(places.dim() - 1);
  return gsplat_rows_meta{places.numel() / S, (int32_t)S, (int32_t)rows.size(rows.dim() - 1), stride,
                          dtype_of(rows)};
}

// Where the number of choices with a code stands.
const int32_t* named(const Tensor& starts) { return ids(starts) + starts.numel() - 1; }

Tensor by_code_values(const Tensor& rows, const Groups& g) {
  int64_t stride;
  const Tensor x = rows_of(rows, stride);
  const Tensor out = at::empty({g.order.numel(), x.size(x.dim() - 1)}, plain_options(x));
  const auto meta = rows_meta(x, stride, g.places);
  const Timed timed("rows_by_code");
  check(api.rows_by_code(&meta, x.data_ptr(), ids(g.order), ids(g.places), named(g.starts), nullptr,
                         out.data_ptr(), stream_of(x)),
        "gsplat_hip_rows_by_code");
  return out;
}

// (rows: [P, D] in the order of the places)
Tensor from_codes_values(const Tensor& rows, const Tensor& places, const Tensor& weights,
                         const char* name) {
  int64_t stride;
  const Tensor y = rows_of(rows, stride);
  const Tensor w = weights.defined() ? weights.contiguous() : weights;
  const Tensor out = at::empty(with(places.sizes().slice(0, places.dim() - 1), y.size(1)),
                               plain_options(y));
  const auto meta = rows_meta(y, stride, places);
  const Timed timed(name);
  check(api.rows_from_codes(&meta, y.data_ptr(), ids(places), f32_or_null(w), out.data_ptr(),
                            stream_of(y)),
        "gsplat_hip_rows_from_codes");
  return out;
}

struct ByCode : torch::autograd::Function<ByCode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& order,
                        const Tensor& places, const Tensor& starts) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({places});
    return by_code_values(rows, Groups{order, places, starts});
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined() || !ctx->needs_input_grad(0)) return out;
    const c10::DeviceGuard device(grads[0].device());
    out[0] = from_codes_values(grads[0], ctx->get_saved_variables()[0].contiguous(), Tensor(),
                               "rows_by_code_backward");
    return once(std::move(out), {grads[0]}, "rows_by_code");
  }
};

py::object by_code(py::handle rows, py::handle order, py::handle places, py::handle starts) {
  if (!ordinary(rows.ptr()) || !plain_context()) return py::none();
  const Tensor& x = THPVariable_Unpack(rows.ptr());
  Groups g;
  if (dtype_of(x) < 0 || x.dim() < 1 || !groups_of(order, places, starts, x.device(), g))
    return py::none();
  const int64_t nd = x.dim(), D = x.size(nd - 1);
  if (D == 0 || D > GSPLAT_MAX_CODE_WIDTH || x.sizes().slice(0, nd - 1) != g.splats())
    return py::none();
  const c10::DeviceGuard device(x.device());
  Tensor out;
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    out = ByCode::apply(x, g.order, g.places, g.starts);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    out = by_code_values(x, g);
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

struct FromCodes : torch::autograd::Function<FromCodes> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& order,
                        const Tensor& places, const Tensor& starts,
                        const std::optional<Tensor>& given_weights) {
    const Tensor weights = given_weights.value_or(Tensor());
    ctx->set_materialize_grads(false);
    // (the rows are for the weights' gradient only)
    const bool keep = weights.defined() && weights.requires_grad();
    ctx->save_for_backward({keep ? rows : Tensor(), order, places, starts, weights});
    return from_codes_values(rows, places, weights, "rows_from_codes");
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(5);
    const auto saved = ctx->get_saved_variables();
    const Tensor& weights = saved[4];
    const bool need_rows = ctx->needs_input_grad(0);
    const bool need_weights = weights.defined() && ctx->needs_input_grad(4);
    if (!grads[0].defined() || !(need_rows || need_weights)) return out;
    const c10::DeviceGuard device(grads[0].device());
    const Tensor g = grads[0].contiguous();
    const Tensor order = saved[1].contiguous(), places = saved[2].contiguous();
    const Tensor starts = saved[3].contiguous();
    const Tensor w = weights.defined() ? weights.contiguous() : weights;
    const int64_t D = g.size(g.dim() - 1);
    int64_t stride = D;
    const Tensor rows = need_weights ? rows_of(saved[0], stride) : Tensor();
    auto meta = rows_meta(g, stride, places);
    if (need_rows) out[0] = at::empty({order.numel(), D}, plain_options(g));
    if (need_weights) out[4] = at::empty(weights.sizes(), plain_options(g).dtype(at::kFloat));
    {
      const Timed timed("rows_from_codes_backward");
      check(api.rows_from_codes_backward(&meta, g.data_ptr(), pointer(rows), ids(order), ids(places),
                                         named(starts), f32_or_null(w), pointer(out[0]),
                                         f32_or_null(out[4]),
                                         stream_of(g)),
            "gsplat_hip_rows_from_codes_backward");
    }
    return once(std::move(out), {grads[0], saved[0], weights}, "rows_from_codes");
  }
};

py::object from_codes(py::handle rows, py::handle order, py::handle places, py::handle starts,
                      py::handle weights) {
  if (!ordinary(rows.ptr()) || !plain_context()) return py::none();
  if (!weights.is_none() && !plain(weights.ptr())) return py::none();
  const Tensor& y = THPVariable_Unpack(rows.ptr());
  const Tensor w = weights.is_none() ? Tensor() : THPVariable_Unpack(weights.ptr());
  Groups g;
  if (dtype_of(y) < 0 || y.dim() != 2 || !groups_of(order, places, starts, y.device(), g))
    return py::none();
  if (y.size(0) != g.order.numel() || y.size(1) == 0 || y.size(1) > GSPLAT_MAX_CODE_WIDTH)
    return py::none();
  if (w.defined() && (w.device() != y.device() ||
                      (w.sizes() != g.places.sizes() && (g.choices() != 1 || w.sizes() != g.splats()))))
    return py::none();
  const c10::DeviceGuard device(y.device());
  Tensor out;
  if (at::GradMode::is_enabled() && (y.requires_grad() || (w.defined() && w.requires_grad()))) {
    out = FromCodes::apply(y, g.order, g.places, g.starts,
                           w.defined() ? std::optional<Tensor>(w) : std::nullopt);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    out = from_codes_values(y, g.places, w, "rows_from_codes");
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

// ---- adapters

gsplat_adapters_meta adapters_meta(const Tensor& rows, int64_t stride, const Tensor& down,
                                   const Tensor& up, double scale, bool by_code) {
  return gsplat_adapters_meta{rows.numel() / rows.size(rows.dim() - 1),
                              (int32_t)down.size(0),
                              (int32_t)down.size(1),
                              (int32_t)down.size(2),
                              (int32_t)up.size(1),
                              stride,
                              dtype_of(rows),
                              by_code ? 1 : 0,
                              (float)scale};
}

Tensor adapters_values(const Tensor& rows, const Groups& g, const Tensor& down, const Tensor& up,
                       const Tensor& base, double scale, bool by_code, Tensor* hidden) {
  int64_t stride;
  const Tensor x = rows_of(rows, stride), dn = down.contiguous(), u = up.contiguous();
  const Tensor b = base.defined() ? base.contiguous() : base;
  const Tensor out = at::empty(with(x.sizes().slice(0, x.dim() - 1), u.size(1)), plain_options(x));
  const auto meta = adapters_meta(x, stride, dn, u, scale, by_code);
  if (hidden) *hidden = at::empty({meta.rows, meta.rank}, plain_options(x).dtype(at::kFloat));
  const size_t n = api.code_adapters_workspace_bytes(&meta);
  const Tensor ws = n > 0 ? bytes((int64_t)n, x) : Tensor();
  const Timed timed("code_adapters");
  check(api.code_adapters_forward(&meta, x.data_ptr(), ids(g.order), ids(g.places), ids(g.starts),
                                  dn.data_ptr(), u.data_ptr(), pointer(b), out.data_ptr(),
                                  hidden ? f32_or_null(*hidden) : nullptr, pointer(ws), n,
                                  stream_of(x)),
        "gsplat_hip_code_adapters_forward");
  return out;
}

struct Adapters : torch::autograd::Function<Adapters> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& order,
                        const Tensor& places, const Tensor& starts, const Tensor& down,
                        const Tensor& up, const std::optional<Tensor>& base, double scale,
                        bool by_code) {
    ctx->set_materialize_grads(false);
    Tensor hidden;
    const Tensor out = adapters_values(rows, Groups{order, places, starts}, down, up,
                                       base.value_or(Tensor()), scale, by_code, &hidden);
    ctx->save_for_backward({rows, order, places, starts, down, up, hidden});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["by_code"] = by_code;
    ctx->saved_data["base"] = base.has_value();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(9);
    const bool need_rows = ctx->needs_input_grad(0), need_down = ctx->needs_input_grad(4),
               need_up = ctx->needs_input_grad(5);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    if (need_rows || need_down || need_up) {
      int64_t stride;
      const Tensor x = rows_of(saved[0], stride), g = grads[0].contiguous();
      const Groups gr{saved[1].contiguous(), saved[2].contiguous(), saved[3].contiguous()};
      const Tensor down = saved[4].contiguous(), up = saved[5].contiguous();
      const Tensor hidden = saved[6].contiguous();
      const c10::DeviceGuard device(x.device());
      if (need_rows) out[0] = at::empty(x.sizes(), plain_options(x));
      if (need_down) out[4] = at::empty(down.sizes(), plain_options(x));
      if (need_up) out[5] = at::empty(up.sizes(), plain_options(x));
      const auto meta = adapters_meta(x, stride, down, up, ctx->saved_data["scale"].toDouble(),
                                      ctx->saved_data["by_code"].toBool());
      const size_t n = api.code_adapters_backward_workspace_bytes(&meta);
      const Tensor ws = n > 0 ? bytes((int64_t)n, x) : Tensor();
      const Timed timed("code_adapters_backward");
      check(api.code_adapters_backward(&meta, g.data_ptr(), x.data_ptr(), ids(gr.order),
                                       ids(gr.places), ids(gr.starts), down.data_ptr(),
                                       up.data_ptr(), f32(hidden), pointer(out[0]),
                                       pointer(out[4]), pointer(out[5]), pointer(ws), n,
                                       stream_of(x)),
            "gsplat_hip_code_adapters_backward");
    }
    out = once(std::move(out), {grads[0], saved[0], saved[4], saved[5]}, "code_adapters");
    // (the shared map's part is its own gradient, at any order)
    if (ctx->saved_data["base"].toBool() && ctx->needs_input_grad(6)) out[6] = grads[0];
    return out;
  }
};

py::object adapters(py::handle rows, py::handle order, py::handle places, py::handle starts,
                    py::handle down, py::handle up, py::handle base, double scale, bool by_code) {
  if (!ordinary(rows.ptr()) || !ordinary(down.ptr()) || !ordinary(up.ptr()) || !plain_context())
    return py::none();
  if (!base.is_none() && !ordinary(base.ptr())) return py::none();
  const Tensor &x = THPVariable_Unpack(rows.ptr()), &dn = THPVariable_Unpack(down.ptr()),
               &u = THPVariable_Unpack(up.ptr());
  const Tensor b = base.is_none() ? Tensor() : THPVariable_Unpack(base.ptr());
  Groups g;
  const int64_t nd = x.dim();
  if (dtype_of(x) < 0 || nd < 1 || !groups_of(order, places, starts, x.device(), g)) return py::none();
  if (dn.dim() != 3 || u.dim() != 3 || dn.numel() == 0 || u.numel() == 0) return py::none();
  if (dn.scalar_type() != x.scalar_type() || u.scalar_type() != x.scalar_type() ||
      dn.device() != x.device() || u.device() != x.device())
    return py::none();
  const int64_t K = dn.size(0), r = dn.size(1), D = dn.size(2), E = u.size(1);
  if (K != g.starts.numel() - 1 || u.size(0) != K || u.size(2) != r || x.size(nd - 1) != D)
    return py::none();
  if (r > GSPLAT_MAX_RANK || std::max(D, E) > GSPLAT_MAX_CODE_WIDTH || K > GSPLAT_MAX_CODES ||
      K * r * std::max(D, E) > (int64_t(1) << 40))
    return py::none();
  const auto lead = x.sizes().slice(0, nd - 1);
  if (by_code ? (nd != 2 || x.size(0) != g.order.numel()) : (g.choices() != 1 || lead != g.splats()))
    return py::none();
  if (b.defined() && (b.scalar_type() != x.scalar_type() || b.device() != x.device() ||
                      b.sizes() != at::IntArrayRef(with(lead, E))))
    return py::none();
  const c10::DeviceGuard device(x.device());
  Tensor out;
  if (at::GradMode::is_enabled() && (x.requires_grad() || dn.requires_grad() || u.requires_grad() ||
                                     (b.defined() && b.requires_grad()))) {
    out = Adapters::apply(x, g.order, g.places, g.starts, dn, u,
                          b.defined() ? std::optional<Tensor>(b) : std::nullopt, scale, by_code);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    out = adapters_values(x, g, dn, u, b, scale, by_code, nullptr);
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

// ---- clipping

// gradients and out: lists or tuples of tensors (out None: in place; a gradient that
// is None is left out).
py::object clip(py::handle gradients, double max_norm, py::handle out) {
  if (!plain_context() || !(max_norm >= 0.0)) return py::none();
  const bool into = !out.is_none();
  if (!(PyList_Check(gradients.ptr()) || PyTuple_Check(gradients.ptr()))) return py::none();
  if (into && !(PyList_Check(out.ptr()) || PyTuple_Check(out.ptr()))) return py::none();
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(gradients.ptr());
  if (count == 0 || count > (1 << 20)) return py::none();
  if (into && PySequence_Fast_GET_SIZE(out.ptr()) != count) return py::none();
  struct Range {
    uintptr_t from, to;
  };
  std::vector<gsplat_clip_tensor> table;
  table.reserve(count);
  std::vector<Range> written, read;
  written.reserve(count);
  if (into) read.reserve(count);
  const Tensor* first = nullptr;
  int64_t all = 0;
  for (Py_ssize_t k = 0; k < count; ++k) {
    PyObject* p = PySequence_Fast_GET_ITEM(gradients.ptr(), k);
    if (p == Py_None) continue;
    if (!ordinary(p)) return py::none();
    const Tensor& g = THPVariable_Unpack(p);
    if (first == nullptr) first = &g;
    const int dtype = dtype_of(g);
    const int64_t n = g.numel();
    if (dtype < 0 || g.device() != first->device() || g.requires_grad() ||
        !g.is_non_overlapping_and_dense() || (all += n) > (int64_t(1) << 40))
      return py::none();
    table.push_back(gsplat_clip_tensor{g.data_ptr(), g.data_ptr(), n, dtype});
    const size_t bytes = (size_t)n * g.element_size();
    const auto at = reinterpret_cast<uintptr_t>(g.data_ptr());
    if (into) {
      PyObject* q = PySequence_Fast_GET_ITEM(out.ptr(), k);
      if (!ordinary(q)) return py::none();
      const Tensor& o = THPVariable_Unpack(q);
      if (o.scalar_type() != g.scalar_type() || o.device() != g.device() || o.requires_grad() ||
          o.sizes() != g.sizes() || o.strides() != g.strides() || o.is_inference())
        return py::none();
      table.back().to = o.data_ptr();
      const auto to = reinterpret_cast<uintptr_t>(o.data_ptr());
      if (bytes == 0) continue;
      written.push_back({to, to + bytes});
      if (to != at) read.push_back({at, at + bytes});
    } else {
      if (g.is_inference()) return py::none();
      if (bytes > 0) written.push_back({at, at + bytes});
    }
  }
  if (first == nullptr) return py::none();
  // What is written must be nobody else's, read or written.
  const auto before = [](const Range& a, const Range& b) { return a.from < b.from; };
  std::sort(written.begin(), written.end(), before);
  for (size_t k = 1; k < written.size(); ++k)
    if (written[k].from < written[k - 1].to) return py::none();
  std::sort(read.begin(), read.end(), before);
  size_t w = 0;
  for (const Range& r : read) {
    while (w < written.size() && written[w].to <= r.from) ++w;
    if (w < written.size() && written[w].from < r.to) return py::none();
  }
  const c10::DeviceGuard device(first->device());
  at::AutoDispatchBelowADInplaceOrView below;
  const Tensor norm = at::empty({}, first->options().dtype(at::kFloat));
  const size_t n = api.clip_gradients_workspace_bytes(table.data(), table.size());
  const Tensor ws = bytes((int64_t)n, *first);
  {
    const Timed timed("clip_gradients");
    check(api.clip_gradients(table.data(), table.size(), max_norm, norm.data_ptr<float>(), pointer(ws), n,
                             stream_of(*first)),
          "gsplat_hip_clip_gradients");
  }
  for (Py_ssize_t k = 0; k < count; ++k)
    if (PySequence_Fast_GET_ITEM(gradients.ptr(), k) != Py_None)
      THPVariable_Unpack(PySequence_Fast_GET_ITEM((into ? out : gradients).ptr(), k))
          .unsafeGetTensorImpl()
          ->bump_version();
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(norm));
}

}  // namespace

void def_decoders(py::module_& m) {
  m.def("group_codes", &group);
  m.def("rows_by_code", &by_code);
  m.def("rows_from_codes", &from_codes);
  m.def("code_adapters", &adapters);
  m.def("clip_gradients", &clip);
}

}  // namespace gs_host
