// code_capi.hip -- extern "C" entry points of scenes in codes, of decoders by
// code and of gradients of many tensors (the last parts of gsplat_hip.h): checks
// of the arguments before any launch, as in capi.hip.
#include <initializer_list>

#include "codes.h"
#include "gradients.h"

namespace {

int fail(const char* what, const char* why) {
  gs::set_error("%s: %s", what, why);
  return GSPLAT_ERR_INVALID_ARGUMENT;
}

int needs(std::initializer_list<const void*> ptrs, const char* what) {
  for (const void* p : ptrs)
    if (p == nullptr) return fail(what, "NULL pointer argument");
  return GSPLAT_OK;
}

bool dtype_ok(int32_t d) { return d == GSPLAT_F32 || d == GSPLAT_BF16 || d == GSPLAT_F16; }

int room(size_t need, const void* ws, size_t bytes, const char* what) {
  if (need == 0 || (ws != nullptr && bytes >= need)) return GSPLAT_OK;
  gs::set_error("%s: workspace too small (%zu < %zu)", what, ws ? bytes : 0, need);
  return GSPLAT_ERR_WORKSPACE;
}

int make(const gsplat_lookup_meta* m, const void* codes, gs::LookupParams& P,
         const char* what) {
  if (m == nullptr) return fail(what, "meta is NULL");
  if (m->rows < 0 || m->rows > (int64_t(1) << 29)) return fail(what, "rows must lie in [0, 2^29]");
  if (m->num_codes < 1 || m->num_codes > GSPLAT_MAX_CODES)
    return fail(what, "num_codes must lie in [1, 2^28]");
  if (m->width < 1 || m->width > GSPLAT_MAX_CODE_WIDTH) return fail(what, "width must lie in [1, 2^20]");
  if (m->stride < m->width || m->stride > (int64_t(1) << 40))
    return fail(what, "stride must be at least width");
  if (!dtype_ok(m->dtype)) return fail(what, "dtype must be GSPLAT_F32, _BF16 or _F16");
  if (m->code_bytes != 4 && m->code_bytes != 8) return fail(what, "code_bytes must be 4 or 8");
  P = gs::LookupParams{m->rows, m->num_codes, m->width, m->stride, m->dtype,
                       m->factor, gs::Codes{codes, m->code_bytes == 8}};
  return GSPLAT_OK;
}

int make(const gsplat_probs_meta* m, const void* codes, gs::ProbsParams& P,
         const char* what) {
  if (m == nullptr) return fail(what, "meta is NULL");
  if (m->rows < 0 || m->rows > 0x7fffffffLL) return fail(what, "rows must lie in [0, 2^31)");
  if (m->num_codes < 1 || m->num_codes > GSPLAT_MAX_CODES)
    return fail(what, "num_codes must lie in [1, 2^28]");
  if (m->top < 0 || m->top > GSPLAT_MAX_TOP || m->top > m->num_codes)
    return fail(what, "top must lie in [0, min(num_codes, 64)]");
  if (m->stride < m->num_codes || m->stride > (int64_t(1) << 40))
    return fail(what, "stride must be at least num_codes");
  if (!dtype_ok(m->dtype)) return fail(what, "dtype must be GSPLAT_F32, _BF16 or _F16");
  if (m->code_bytes != 4 && m->code_bytes != 8) return fail(what, "code_bytes must be 4 or 8");
  // (1 / T in base 2, 1.44 times that, has to be finite too)
  const float inv_t = 1.0f / m->temperature;
  if (!(m->temperature > 0.0f) || !(inv_t > 0.0f) || inv_t > 2.0e38f)
    return fail(what, "temperature must be positive and finite, twice its reciprocal too");
  P = gs::ProbsParams{m->rows, m->num_codes, m->top, m->stride, m->dtype, inv_t,
                      gs::Codes{codes, m->code_bytes == 8}};
  return GSPLAT_OK;
}

int make(const gsplat_balance_meta* m, const void* codes, gs::BalanceParams& P,
         const char* what) {
  if (m == nullptr) return fail(what, "meta is NULL");
  if (m->batch < 1 || m->batch > GSPLAT_MAX_BALANCE_IMAGES) return fail(what, "batch must lie in [1, 65535]");
  if (m->choices < 1 || m->choices > GSPLAT_MAX_CHOICES) return fail(what, "choices must lie in [1, 2^20]");
  if (m->rows < 0 || m->rows > 0x7fffffffLL / m->batch / m->choices)
    return fail(what, "batch * rows * choices must lie in [0, 2^31)");
  if (m->num_codes < 1 || m->num_codes > GSPLAT_MAX_BALANCE_CODES)
    return fail(what, "num_codes must lie in [1, 2^24]");
  if (m->stride < m->num_codes || m->stride > (int64_t(1) << 40))
    return fail(what, "stride must be at least num_codes");
  if (!dtype_ok(m->dtype)) return fail(what, "dtype must be GSPLAT_F32, _BF16 or _F16");
  if (m->code_bytes != 4 && m->code_bytes != 8) return fail(what, "code_bytes must be 4 or 8");
  P = gs::BalanceParams{m->batch, m->rows, m->num_codes, m->choices, m->stride,
                        m->dtype, gs::Codes{codes, m->code_bytes == 8}};
  return GSPLAT_OK;
}

int make(const gsplat_group_meta* m, const void* codes, gs::GroupParams& P,
         const char* what) {
  if (m == nullptr) return fail(what, "meta is NULL");
  if (m->choices < 0 || m->choices > (int64_t(1) << 29)) return fail(what, "choices must lie in [0, 2^29]");
  if (m->num_codes < 1 || m->num_codes > GSPLAT_MAX_CODES)
    return fail(what, "num_codes must lie in [1, 2^28]");
  if (m->code_bytes != 4 && m->code_bytes != 8) return fail(what, "code_bytes must be 4 or 8");
  P = gs::GroupParams{m->choices, m->num_codes, gs::Codes{codes, m->code_bytes == 8}};
  return GSPLAT_OK;
}

int make(const gsplat_rows_meta* m, gs::RowsParams& P, const char* what) {
  if (m == nullptr) return fail(what, "meta is NULL");
  if (m->choices < 1 || m->choices > GSPLAT_MAX_CHOICES) return fail(what, "choices must lie in [1, 2^20]");
  if (m->splats < 0 || m->splats > (int64_t(1) << 29) / m->choices)
    return fail(what, "splats * choices must lie in [0, 2^29]");
  if (m->width < 1 || m->width > GSPLAT_MAX_CODE_WIDTH) return fail(what, "width must lie in [1, 2^20]");
  if (m->stride < m->width || m->stride > (int64_t(1) << 40))
    return fail(what, "stride must be at least width");
  if (!dtype_ok(m->dtype)) return fail(what, "dtype must be GSPLAT_F32, _BF16 or _F16");
  P = gs::RowsParams{m->splats, m->choices, m->width, m->stride, m->dtype};
  return GSPLAT_OK;
}

int make(const gsplat_adapters_meta* m, const int32_t* order, const int32_t* places,
         const int32_t* starts, gs::AdapterParams& P, const char* what) {
  if (m == nullptr) return fail(what, "meta is NULL");
  if (m->rows < 0 || m->rows > (int64_t(1) << 29)) return fail(what, "rows must lie in [0, 2^29]");
  if (m->num_codes < 1 || m->num_codes > GSPLAT_MAX_CODES)
    return fail(what, "num_codes must lie in [1, 2^28]");
  if (m->rank < 1 || m->rank > GSPLAT_MAX_RANK) return fail(what, "rank must lie in [1, 128]");
  if (m->width_in < 1 || m->width_in > GSPLAT_MAX_CODE_WIDTH || m->width_out < 1 ||
      m->width_out > GSPLAT_MAX_CODE_WIDTH)
    return fail(what, "width_in and width_out must lie in [1, 2^20]");
  const int64_t wide = m->width_in > m->width_out ? m->width_in : m->width_out;
  if (m->num_codes > (int64_t(1) << 40) / (m->rank * wide))
    return fail(what, "num_codes * rank * width must be at most 2^40");
  if (m->stride < m->width_in || m->stride > (int64_t(1) << 40))
    return fail(what, "stride must be at least width_in");
  if (!dtype_ok(m->dtype)) return fail(what, "dtype must be GSPLAT_F32, _BF16 or _F16");
  P = gs::AdapterParams{m->rows,  m->num_codes, m->rank,         m->width_in, m->width_out,
                        m->stride, m->dtype,    m->by_code != 0, m->scale,    order,
                        places,    starts};
  return GSPLAT_OK;
}

int tensors_ok(const gsplat_clip_tensor* x, int64_t count, const char* what) {
  if (count < 0 || count > (int64_t(1) << 20)) return fail(what, "count must lie in [0, 2^20]");
  if (count > 0 && x == nullptr) return fail(what, "NULL pointer argument");
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (x[i].size < 0 || x[i].size > (int64_t(1) << 40) || (all += x[i].size) > (int64_t(1) << 40))
      return fail(what, "sizes must lie in [0, 2^40], and their sum");
    if (!dtype_ok(x[i].dtype)) return fail(what, "dtype must be GSPLAT_F32, _BF16 or _F16");
  }
  return GSPLAT_OK;
}

}  // namespace

extern "C" {

int gsplat_hip_lookup_forward(const gsplat_lookup_meta* meta, const void* codes,
                              const void* codebook, const float* scales,
                              void* out, void* stream) {
  const char* what = "gsplat_hip_lookup_forward";
  gs::LookupParams P;
  int rc = make(meta, codes, P, what);
  if (rc || P.rows == 0) return rc;
  if ((rc = needs({codes, codebook, out}, what))) return rc;
  return gs::launch_lookup_forward(P, codebook, scales, out,
                                   static_cast<hipStream_t>(stream));
}

size_t gsplat_hip_lookup_backward_workspace_bytes(const gsplat_lookup_meta* meta) {
  gs::LookupParams P;
  if (make(meta, nullptr, P, "gsplat_hip_lookup_backward_workspace_bytes")) return 0;
  return gs::lookup_backward_workspace_bytes(P);
}

int gsplat_hip_lookup_backward(const gsplat_lookup_meta* meta,
                               const void* grad_out, const void* codes,
                               const void* codebook, const float* scales,
                               void* g_codebook, float* g_scales,
                               void* workspace, size_t workspace_bytes,
                               void* stream) {
  const char* what = "gsplat_hip_lookup_backward";
  gs::LookupParams P;
  int rc = make(meta, codes, P, what);
  if (rc) return rc;
  if (P.rows > 0 && (rc = needs({grad_out, codes}, what))) return rc;
  if (P.rows > 0 && g_scales != nullptr && (rc = needs({codebook}, what))) return rc;
  if (g_codebook != nullptr &&
      (rc = room(gs::lookup_backward_workspace_bytes(P), workspace, workspace_bytes, what)))
    return rc;
  return gs::launch_lookup_backward(P, grad_out, codebook, scales, g_codebook,
                                    g_scales, workspace,
                                    static_cast<hipStream_t>(stream));
}

size_t gsplat_hip_code_probs_workspace_bytes(const gsplat_probs_meta* meta) {
  gs::ProbsParams P;
  if (make(meta, nullptr, P, "gsplat_hip_code_probs_workspace_bytes")) return 0;
  return gs::probs_workspace_bytes(P);
}

int gsplat_hip_code_probs_forward(const gsplat_probs_meta* meta,
                                  const void* logits, const void* codes,
                                  float* log_probs, float* entropy,
                                  float* top_log_probs, int32_t* top_codes,
                                  float* row_stats, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  const char* what = "gsplat_hip_code_probs_forward";
  gs::ProbsParams P;
  int rc = make(meta, codes, P, what);
  if (rc || P.rows == 0) return rc;
  if ((rc = needs({logits, entropy}, what))) return rc;
  if ((codes == nullptr) != (log_probs == nullptr))
    return fail(what, "log_probs goes with codes");
  if (P.top > 0 && (rc = needs({top_log_probs, top_codes}, what))) return rc;
  if ((rc = room(gs::probs_workspace_bytes(P), workspace, workspace_bytes, what)))
    return rc;
  return gs::launch_probs_forward(P, logits, log_probs, entropy, top_log_probs,
                                  top_codes, reinterpret_cast<float2*>(row_stats),
                                  workspace, static_cast<hipStream_t>(stream));
}

int gsplat_hip_code_probs_backward(const gsplat_probs_meta* meta,
                                   const void* logits, const void* codes,
                                   const int32_t* top_codes,
                                   const float* row_stats, const float* entropy,
                                   const float* g_log_probs,
                                   const float* g_entropy,
                                   const float* g_top_log_probs,
                                   void* g_logits, void* stream) {
  const char* what = "gsplat_hip_code_probs_backward";
  gs::ProbsParams P;
  int rc = make(meta, codes, P, what);
  if (rc || P.rows == 0) return rc;
  if ((rc = needs({logits, row_stats, entropy, g_logits}, what))) return rc;
  if (g_log_probs != nullptr && (rc = needs({codes}, what))) return rc;
  if (g_top_log_probs != nullptr && P.top > 0 && (rc = needs({top_codes}, what)))
    return rc;
  return gs::launch_probs_backward(
      P, logits, top_codes, reinterpret_cast<const float2*>(row_stats), entropy,
      g_log_probs, g_entropy, P.top > 0 ? g_top_log_probs : nullptr, g_logits,
      static_cast<hipStream_t>(stream));
}

size_t gsplat_hip_code_balance_workspace_bytes(const gsplat_balance_meta* meta) {
  gs::BalanceParams P;
  if (make(meta, nullptr, P, "gsplat_hip_code_balance_workspace_bytes")) return 0;
  return gs::balance_workspace_bytes(P);
}

int gsplat_hip_code_balance_forward(const gsplat_balance_meta* meta,
                                    const void* logits, const void* codes,
                                    float* loss, int32_t* counts,
                                    float* mean_probs, float* row_stats,
                                    int32_t* totals, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  const char* what = "gsplat_hip_code_balance_forward";
  gs::BalanceParams P;
  int rc = make(meta, codes, P, what);
  if (rc) return rc;
  if ((rc = needs({loss, counts, mean_probs, totals}, what))) return rc;
  if (P.rows > 0 && (rc = needs({logits, codes, row_stats}, what))) return rc;
  if ((rc = room(gs::balance_workspace_bytes(P), workspace, workspace_bytes, what)))
    return rc;
  return gs::launch_balance_forward(P, logits, loss, counts, mean_probs,
                                    reinterpret_cast<float2*>(row_stats), totals,
                                    workspace, static_cast<hipStream_t>(stream));
}

int gsplat_hip_code_balance_backward(const gsplat_balance_meta* meta,
                                     const void* logits, const int32_t* counts,
                                     const float* row_stats,
                                     const int32_t* totals, const float* g_loss,
                                     const float* g_mean_probs, void* g_logits,
                                     void* stream) {
  const char* what = "gsplat_hip_code_balance_backward";
  gs::BalanceParams P;
  int rc = make(meta, nullptr, P, what);
  if (rc || P.rows == 0) return rc;
  if ((rc = needs({logits, counts, row_stats, totals, g_logits}, what))) return rc;
  return gs::launch_balance_backward(P, logits, counts,
                                     reinterpret_cast<const float2*>(row_stats),
                                     totals, g_loss, g_mean_probs, g_logits,
                                     static_cast<hipStream_t>(stream));
}

size_t gsplat_hip_group_codes_workspace_bytes(const gsplat_group_meta* meta) {
  gs::GroupParams P;
  if (make(meta, nullptr, P, "gsplat_hip_group_codes_workspace_bytes")) return 0;
  return gs::group_workspace_bytes(P);
}

int gsplat_hip_group_codes(const gsplat_group_meta* meta, const void* codes,
                           int32_t* order, int32_t* places, int32_t* starts,
                           void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "gsplat_hip_group_codes";
  gs::GroupParams P;
  int rc = make(meta, codes, P, what);
  if (rc) return rc;
  if ((rc = needs({starts}, what))) return rc;
  if (P.choices > 0 && (rc = needs({codes, order, places}, what))) return rc;
  if ((rc = room(gs::group_workspace_bytes(P), workspace, workspace_bytes, what))) return rc;
  return gs::launch_group_codes(P, order, places, starts, workspace,
                                static_cast<hipStream_t>(stream));
}

int gsplat_hip_rows_by_code(const gsplat_rows_meta* meta, const void* rows,
                            const int32_t* order, const int32_t* places,
                            const int32_t* named, const float* weights, void* out,
                            void* stream) {
  const char* what = "gsplat_hip_rows_by_code";
  gs::RowsParams P;
  int rc = make(meta, P, what);
  if (rc || P.splats == 0) return rc;
  if ((rc = needs({rows, order, places, named, out}, what))) return rc;
  return gs::launch_rows_by_code(P, rows, order, places, named, weights, out,
                                 static_cast<hipStream_t>(stream));
}

int gsplat_hip_rows_from_codes(const gsplat_rows_meta* meta, const void* rows,
                               const int32_t* places, const float* weights,
                               void* out, void* stream) {
  const char* what = "gsplat_hip_rows_from_codes";
  gs::RowsParams P;
  int rc = make(meta, P, what);
  if (rc || P.splats == 0) return rc;
  if ((rc = needs({rows, places, out}, what))) return rc;
  return gs::launch_rows_from_codes(P, rows, places, weights, out,
                                    static_cast<hipStream_t>(stream));
}

int gsplat_hip_rows_from_codes_backward(const gsplat_rows_meta* meta,
                                        const void* grad, const void* rows,
                                        const int32_t* order, const int32_t* places,
                                        const int32_t* named, const float* weights,
                                        void* g_rows, float* g_weights, void* stream) {
  const char* what = "gsplat_hip_rows_from_codes_backward";
  gs::RowsParams P;
  int rc = make(meta, P, what);
  if (rc || P.splats == 0 || (g_rows == nullptr && g_weights == nullptr)) return rc;
  if ((rc = needs({grad, order, places, named}, what))) return rc;
  if (g_weights != nullptr && (rc = needs({rows, weights}, what))) return rc;
  return gs::launch_rows_from_codes_backward(P, grad, rows, order, places, named, weights,
                                             g_rows, g_weights,
                                             static_cast<hipStream_t>(stream));
}

size_t gsplat_hip_code_adapters_workspace_bytes(const gsplat_adapters_meta* meta) {
  gs::AdapterParams P;
  if (make(meta, nullptr, nullptr, nullptr, P, "gsplat_hip_code_adapters_workspace_bytes"))
    return 0;
  return gs::adapters_forward_workspace_bytes(P);
}

int gsplat_hip_code_adapters_forward(const gsplat_adapters_meta* meta,
                                     const void* rows, const int32_t* order,
                                     const int32_t* places, const int32_t* starts,
                                     const void* down, const void* up,
                                     const void* base, void* out, float* hidden,
                                     void* workspace, size_t workspace_bytes,
                                     void* stream) {
  const char* what = "gsplat_hip_code_adapters_forward";
  gs::AdapterParams P;
  int rc = make(meta, order, places, starts, P, what);
  if (rc || P.rows == 0) return rc;
  if ((rc = needs({rows, order, places, starts, down, up, out}, what))) return rc;
  if ((rc = room(gs::adapters_forward_workspace_bytes(P), workspace, workspace_bytes, what)))
    return rc;
  return gs::launch_adapters_forward(P, rows, down, up, base, out, hidden, workspace,
                                     static_cast<hipStream_t>(stream));
}

size_t gsplat_hip_code_adapters_backward_workspace_bytes(const gsplat_adapters_meta* meta) {
  gs::AdapterParams P;
  if (make(meta, nullptr, nullptr, nullptr, P,
           "gsplat_hip_code_adapters_backward_workspace_bytes"))
    return 0;
  return gs::adapters_backward_workspace_bytes(P);
}

int gsplat_hip_code_adapters_backward(const gsplat_adapters_meta* meta,
                                      const void* grad, const void* rows,
                                      const int32_t* order, const int32_t* places,
                                      const int32_t* starts, const void* down,
                                      const void* up, const float* hidden,
                                      void* g_rows, void* g_down, void* g_up,
                                      void* workspace, size_t workspace_bytes,
                                      void* stream) {
  const char* what = "gsplat_hip_code_adapters_backward";
  gs::AdapterParams P;
  int rc = make(meta, order, places, starts, P, what);
  if (rc || !(g_rows || g_down || g_up)) return rc;
  if ((rc = needs({starts}, what))) return rc;
  if (P.rows > 0 && (rc = needs({grad, rows, order, places, down, up, hidden}, what))) return rc;
  if ((rc = room(gs::adapters_backward_workspace_bytes(P), workspace, workspace_bytes, what)))
    return rc;
  return gs::launch_adapters_backward(P, grad, rows, down, up, hidden, g_rows, g_down,
                                      g_up, workspace, static_cast<hipStream_t>(stream));
}

size_t gsplat_hip_clip_gradients_workspace_bytes(const gsplat_clip_tensor* tensors,
                                                 int64_t count) {
  if (tensors_ok(tensors, count, "gsplat_hip_clip_gradients_workspace_bytes")) return 0;
  return gs::clip_workspace_bytes(tensors, count);
}

int gsplat_hip_clip_gradients(const gsplat_clip_tensor* tensors, int64_t count,
                              double max_norm, float* norm, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const char* what = "gsplat_hip_clip_gradients";
  int rc = tensors_ok(tensors, count, what);
  if (rc) return rc;
  if (!(max_norm >= 0.0)) return fail(what, "max_norm must be at least 0");
  if ((rc = needs({norm}, what))) return rc;
  for (int64_t i = 0; i < count; ++i)
    if (tensors[i].size > 0 && (rc = needs({tensors[i].from, tensors[i].to}, what))) return rc;
  if ((rc = room(gs::clip_workspace_bytes(tensors, count), workspace, workspace_bytes, what)))
    return rc;
  return gs::launch_clip(tensors, count, max_norm, norm, workspace,
                         static_cast<hipStream_t>(stream));
}

}  // extern "C"
