// host_codes.cpp -- the host path of scenes in codes in C++: argument checks,
// buffers, the C-ABI calls and the autograd nodes of lookup_codes,
// code_log_probs and code_balance.
//
// As in host.cpp, what is not the plain case returns None, and the Python
// layer's operators take it, with its messages: inputs that fail a check,
// tensors that are not plain ones, active modes and transforms.
#include <algorithm>
#include <optional>

#include "host_codes.h"

namespace gs_host {
namespace {

// ---- lookup

gsplat_lookup_meta lookup_meta(const Tensor& codes, const Tensor& book, int64_t stride,
                               double factor) {
  return gsplat_lookup_meta{codes.numel(), (int32_t)book.size(0), (int32_t)book.size(1),
                            stride,        dtype_of(book),        (int32_t)codes.element_size(),
                            (float)factor};
}

Tensor lookup_values(const Tensor& codes, const Tensor& codebook, const Tensor& scales,
                     double factor) {
  int64_t stride;
  const Tensor c = codes.contiguous(), book = rows_of(codebook, stride);
  const Tensor s = scales.defined() ? scales.contiguous() : scales;
  const Tensor out = at::empty(with(codes.sizes(), book.size(1)), plain_options(book));
  const auto meta = lookup_meta(c, book, stride, factor);
  const Timed timed("lookup_codes");
  check(api.lookup_forward(&meta, c.data_ptr(), book.data_ptr(), f32_or_null(s),
                           out.data_ptr(), stream_of(book)),
        "gsplat_hip_lookup_forward");
  return out;
}

struct Lookup : torch::autograd::Function<Lookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& codes, const Tensor& codebook,
                        const std::optional<Tensor>& given_scales, double factor) {
    const Tensor scales = given_scales.value_or(Tensor());
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({codes, codebook, scales});
    ctx->saved_data["factor"] = factor;
    return lookup_values(codes, codebook, scales, factor);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    const bool need_book = ctx->needs_input_grad(1);
    const auto saved = ctx->get_saved_variables();
    const Tensor& scales = saved[2];
    const bool need_scales = scales.defined() && ctx->needs_input_grad(2);
    if (!grads[0].defined() || !(need_book || need_scales)) return out;
    int64_t stride;
    const Tensor g = grads[0].contiguous(), c = saved[0].contiguous();
    const Tensor book = rows_of(saved[1], stride);
    const Tensor s = scales.defined() ? scales.contiguous() : scales;
    const auto opt = plain_options(book);
    const c10::DeviceGuard device(book.device());
    const auto meta = lookup_meta(c, book, stride, ctx->saved_data["factor"].toDouble());
    size_t n = 0;
    Tensor ws;
    if (need_book) {
      out[1] = at::empty(book.sizes(), opt);
      n = api.lookup_backward_workspace_bytes(&meta);
      if (n > 0) ws = bytes((int64_t)n, book);
    }
    if (need_scales) out[2] = at::empty(scales.sizes(), opt.dtype(at::kFloat));
    {
      const Timed timed("lookup_codes_backward");
      check(api.lookup_backward(&meta, g.data_ptr(), c.data_ptr(), book.data_ptr(),
                                f32_or_null(s), pointer(out[1]), f32_or_null(out[2]),
                                pointer(ws), n, stream_of(book)),
            "gsplat_hip_lookup_backward");
    }
    return once(std::move(out), {grads[0], saved[1], scales}, "lookup_codes");
  }
};

py::object lookup(py::handle codes, py::handle codebook, py::handle scales, double factor) {
  if (!ordinary(codes.ptr()) || !ordinary(codebook.ptr()) || !plain_context())
    return py::none();
  if (!scales.is_none() && !plain(scales.ptr())) return py::none();
  const Tensor &c = THPVariable_Unpack(codes.ptr()), &book = THPVariable_Unpack(codebook.ptr());
  const Tensor s = scales.is_none() ? Tensor() : THPVariable_Unpack(scales.ptr());
  if (!codes_ok(c) || dtype_of(book) < 0 || book.dim() != 2 || book.numel() == 0)
    return py::none();
  if (book.size(0) > GSPLAT_MAX_CODES || book.size(1) > GSPLAT_MAX_CODE_WIDTH)
    return py::none();
  if (c.device() != book.device()) return py::none();
  if (s.defined() && (s.device() != c.device() || s.sizes() != c.sizes())) return py::none();
  const c10::DeviceGuard device(book.device());
  Tensor out;
  if (at::GradMode::is_enabled() &&
      (book.requires_grad() || (s.defined() && s.requires_grad()))) {
    out = Lookup::apply(c, book, s.defined() ? std::optional<Tensor>(s) : std::nullopt, factor);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    out = lookup_values(c, book, s, factor);
  }
  return py::reinterpret_steal<py::object>(THPVariable_Wrap(out));
}

// ---- log probabilities

struct ProbsOut {
  Tensor log_probs, entropy, top_log_probs, top_codes, stats;
};

gsplat_probs_meta probs_meta(const Tensor& logits, int64_t stride, const Tensor& codes,
                             int64_t top, double temperature) {
  const int64_t K = logits.size(logits.dim() - 1);
  return gsplat_probs_meta{logits.numel() / K, (int32_t)K,
                           (int32_t)top,       stride,
                           dtype_of(logits),   codes.defined() ? (int32_t)codes.element_size() : 4,
                           (float)temperature};
}

ProbsOut probs_values(const Tensor& logits, const Tensor& codes, int64_t top,
                      double temperature, bool train) {
  int64_t stride;
  const Tensor x = rows_of(logits, stride);
  const Tensor c = codes.defined() ? codes.contiguous() : codes;
  const auto shape = x.sizes().slice(0, x.dim() - 1);
  const auto opt = plain_options(x).dtype(at::kFloat);
  ProbsOut r;
  if (c.defined()) r.log_probs = at::empty(shape, opt);
  r.entropy = at::empty(shape, opt);
  if (top > 0) {
    r.top_log_probs = at::empty(with(shape, top), opt);
    r.top_codes = at::empty(with(shape, top), opt.dtype(at::kInt));
  }
  if (train) r.stats = at::empty(with(shape, 2), opt);
  const auto meta = probs_meta(x, stride, c, top, temperature);
  const size_t n = api.code_probs_workspace_bytes(&meta);
  const Tensor ws = n > 0 ? bytes((int64_t)n, x) : Tensor();
  const Timed timed("code_log_probs");
  check(api.code_probs_forward(&meta, x.data_ptr(), pointer(c), f32_or_null(r.log_probs),
                               f32_or_null(r.entropy), f32_or_null(r.top_log_probs),
                               top > 0 ? i32(r.top_codes) : nullptr, f32_or_null(r.stats),
                               pointer(ws), n, stream_of(x)),
        "gsplat_hip_code_probs_forward");
  return r;
}

struct Probs : torch::autograd::Function<Probs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits,
                               const std::optional<Tensor>& given_codes, int64_t top,
                               double temperature) {
    const Tensor codes = given_codes.value_or(Tensor());
    ctx->set_materialize_grads(false);
    ProbsOut r = probs_values(logits, codes, top, temperature, true);
    ctx->save_for_backward({logits, codes, r.top_codes, r.stats, r.entropy});
    ctx->saved_data["top"] = top;
    ctx->saved_data["T"] = temperature;
    variable_list out;
    if (codes.defined()) out.push_back(r.log_probs);
    out.push_back(r.entropy);
    if (top > 0) {
      ctx->mark_non_differentiable({r.top_codes});
      out.push_back(r.top_log_probs);
      out.push_back(r.top_codes);
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t top = ctx->saved_data["top"].toInt();
    const Tensor& codes = saved[1];
    int64_t stride;
    const Tensor x = rows_of(saved[0], stride);
    const Tensor c = codes.defined() ? codes.contiguous() : codes;
    size_t k = 0;
    auto next = [&] {
      const Tensor g = grads[k++];
      return g.defined() ? g.contiguous() : g;
    };
    const Tensor gl = codes.defined() ? next() : Tensor();
    const Tensor ge = next();
    const Tensor gt = top > 0 ? next() : Tensor();
    variable_list out(4);
    if (!ctx->needs_input_grad(0) || !(gl.defined() || ge.defined() || gt.defined()))
      return out;
    const c10::DeviceGuard device(x.device());
    out[0] = at::empty(x.sizes(), plain_options(x));
    // (saved-tensor hooks may give back another layout)
    const Tensor best = top > 0 ? saved[2].contiguous() : Tensor();
    const Tensor stats = saved[3].contiguous(), entropy = saved[4].contiguous();
    const auto meta = probs_meta(x, stride, c, top, ctx->saved_data["T"].toDouble());
    {
      const Timed timed("code_log_probs_backward");
      check(api.code_probs_backward(&meta, x.data_ptr(), pointer(c),
                                    top > 0 ? i32(best) : nullptr, f32(stats),
                                    f32(entropy), f32_or_null(gl), f32_or_null(ge),
                                    f32_or_null(gt), out[0].data_ptr(), stream_of(x)),
            "gsplat_hip_code_probs_backward");
    }
    return once(std::move(out), {saved[0], gl, ge, gt}, "code_log_probs");
  }
};

// (log_probs, entropy, top_log_probs, top_codes), None for those not asked for.
py::object log_probs(py::handle logits, py::handle codes, int64_t top, double temperature) {
  if (!ordinary(logits.ptr()) || !plain_context()) return py::none();
  if (!codes.is_none() && !ordinary(codes.ptr())) return py::none();
  const Tensor& x = THPVariable_Unpack(logits.ptr());
  const Tensor c = codes.is_none() ? Tensor() : THPVariable_Unpack(codes.ptr());
  const int64_t nd = x.dim();
  if (dtype_of(x) < 0 || nd < 1 || x.size(nd - 1) == 0 || x.size(nd - 1) > GSPLAT_MAX_CODES)
    return py::none();
  if (c.defined() && (!codes_ok(c) || c.device() != x.device() ||
                      c.sizes() != x.sizes().slice(0, nd - 1)))
    return py::none();
  if (top < 0 || top > std::min<int64_t>(GSPLAT_MAX_TOP, x.size(nd - 1))) return py::none();
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return py::none();
  const c10::DeviceGuard device(x.device());
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    const variable_list r = Probs::apply(
        x, c.defined() ? std::optional<Tensor>(c) : std::nullopt, top, temperature);
    const size_t k = c.defined() ? 1 : 0;
    return tuple_of({c.defined() ? r[0] : Tensor(), r[k], top > 0 ? r[k + 1] : Tensor(),
                     top > 0 ? r[k + 2] : Tensor()});
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const ProbsOut r = probs_values(x, c, top, temperature, false);
  return tuple_of({r.log_probs, r.entropy, r.top_log_probs, r.top_codes});
}

// ---- balance

struct BalanceOut {
  Tensor loss, counts, mean, stats, totals;
};

gsplat_balance_meta balance_meta(const Tensor& x, int64_t stride, int64_t choices,
                                 int64_t code_bytes) {
  const int64_t nd = x.dim();
  return gsplat_balance_meta{x.size(nd - 2),
                             (int32_t)(nd == 3 ? x.size(0) : 1),
                             (int32_t)x.size(nd - 1),
                             (int32_t)choices,
                             dtype_of(x),
                             stride,
                             (int32_t)code_bytes};
}

BalanceOut balance_values(const Tensor& logits, const Tensor& codes) {
  int64_t stride;
  const Tensor x = rows_of(logits, stride), c = codes.contiguous();
  const int64_t nd = x.dim(), K = x.size(nd - 1);
  const auto batch = x.sizes().slice(0, nd - 2);
  const auto opt = plain_options(x).dtype(at::kFloat);
  const int64_t B = nd == 3 ? x.size(0) : 1;
  BalanceOut r;
  r.loss = at::empty(batch, opt);
  r.counts = at::empty(with(batch, K), opt.dtype(at::kInt));
  r.mean = at::empty(with(batch, K), opt);
  r.stats = at::empty(with(x.sizes().slice(0, nd - 1), 2), opt);
  r.totals = at::empty({B, 4}, opt.dtype(at::kInt));
  const auto meta = balance_meta(x, stride, c.dim() == nd ? c.size(nd - 1) : 1,
                                 (int64_t)c.element_size());
  const size_t n = api.code_balance_workspace_bytes(&meta);
  const Tensor ws = n > 0 ? bytes((int64_t)n, x) : Tensor();
  const Timed timed("code_balance");
  check(api.code_balance_forward(&meta, x.data_ptr(), c.data_ptr(), f32_or_null(r.loss),
                                 i32(r.counts), f32_or_null(r.mean), f32_or_null(r.stats),
                                 i32(r.totals), pointer(ws), n, stream_of(x)),
        "gsplat_hip_code_balance_forward");
  return r;
}

struct Balance : torch::autograd::Function<Balance> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& codes) {
    ctx->set_materialize_grads(false);
    const BalanceOut r = balance_values(logits, codes);
    ctx->mark_non_differentiable({r.counts});
    ctx->save_for_backward({logits, r.counts, r.stats, r.totals});
    return {r.loss, r.counts, r.mean};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(2);
    if (!ctx->needs_input_grad(0) || !(grads[0].defined() || grads[2].defined())) return out;
    int64_t stride;
    const Tensor x = rows_of(saved[0], stride);
    const Tensor gl = grads[0].defined() ? grads[0].contiguous() : grads[0];
    const Tensor gm = grads[2].defined() ? grads[2].contiguous() : grads[2];
    const c10::DeviceGuard device(x.device());
    out[0] = at::empty(x.sizes(), plain_options(x));
    const Tensor counts = saved[1].contiguous(), stats = saved[2].contiguous();
    const Tensor totals = saved[3].contiguous();
    const auto meta = balance_meta(x, stride, 1, 4);
    {
      const Timed timed("code_balance_backward");
      check(api.code_balance_backward(&meta, x.data_ptr(), i32(counts), f32(stats),
                                      i32(totals), f32_or_null(gl), f32_or_null(gm),
                                      out[0].data_ptr(), stream_of(x)),
            "gsplat_hip_code_balance_backward");
    }
    return once(std::move(out), {saved[0], gl, gm}, "code_balance");
  }
};

// (loss, counts, mean_probs)
py::object balance(py::handle logits, py::handle codes) {
  if (!ordinary(logits.ptr()) || !ordinary(codes.ptr()) || !plain_context()) return py::none();
  const Tensor &x = THPVariable_Unpack(logits.ptr()), &c = THPVariable_Unpack(codes.ptr());
  const int64_t nd = x.dim();
  if (dtype_of(x) < 0 || !codes_ok(c) || (nd != 2 && nd != 3) || x.size(nd - 1) == 0)
    return py::none();
  if (x.size(nd - 1) > GSPLAT_MAX_BALANCE_CODES) return py::none();
  if (nd == 3 && (x.size(0) == 0 || x.size(0) > GSPLAT_MAX_BALANCE_IMAGES)) return py::none();
  if (c.dim() == nd && c.size(nd - 1) > GSPLAT_MAX_CHOICES) return py::none();
  if (c.device() != x.device()) return py::none();
  const auto rows = x.sizes().slice(0, nd - 1);
  if (c.sizes() != rows &&
      (c.dim() != nd || c.sizes().slice(0, nd - 1) != rows || c.size(nd - 1) == 0))
    return py::none();
  const c10::DeviceGuard device(x.device());
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    const variable_list r = Balance::apply(x, c);
    return tuple_of({r[0], r[1], r[2]});
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const BalanceOut r = balance_values(x, c);
  return tuple_of({r.loss, r.counts, r.mean});
}

}  // namespace

void def_codes(py::module_& m) {
  m.def("lookup_codes", &lookup);
  m.def("code_log_probs", &log_probs);
  m.def("code_balance", &balance);
}

}  // namespace gs_host
