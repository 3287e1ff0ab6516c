// code_adapters.hip -- low-rank maps of splats' rows by code: the kernels of
// code_adapters.h by type (code_adapters_f32.hip, _bf16.hip, _f16.hip).
#include "code_adapters.h"

namespace gs {

#define GS_OF(T)                                                                      \
  extern template int adapters_forward_of<T>(const AdapterParams&, const void*,       \
                                             const void*, const void*, const void*,   \
                                             void*, float*, void*, hipStream_t);      \
  extern template int adapters_backward_of<T>(const AdapterParams&, const void*,      \
                                              const void*, const void*, const void*,  \
                                              const float*, void*, void*, void*,      \
                                              void*, hipStream_t);
GS_OF(float)
GS_OF(__bf16)
GS_OF(_Float16)
#undef GS_OF

size_t adapters_forward_workspace_bytes(const AdapterParams& P) {
  const RowsPlan L = rows_plan(P, P.D, P.E);
  return is_split(L) ? (size_t)L.splits_down * P.rows * P.r * 4 : 0;
}
size_t adapters_backward_workspace_bytes(const AdapterParams& P) {
  return backward_layout(P).total;
}

#define GS_BY_TYPE(F)                                         \
  (P.dtype == GSPLAT_F32 ? F<float> : P.dtype == GSPLAT_BF16 ? F<__bf16> : F<_Float16>)

int launch_adapters_forward(const AdapterParams& P, const void* rows,
                            const void* down, const void* up, const void* base,
                            void* out, float* hidden, void* workspace,
                            hipStream_t stream) {
  return GS_BY_TYPE(adapters_forward_of)(P, rows, down, up, base, out, hidden, workspace, stream);
}

int launch_adapters_backward(const AdapterParams& P, const void* grad,
                             const void* rows, const void* down, const void* up,
                             const float* hidden, void* g_rows, void* g_down,
                             void* g_up, void* workspace, hipStream_t stream) {
  return GS_BY_TYPE(adapters_backward_of)(P, grad, rows, down, up, hidden, g_rows, g_down, g_up,
                                 workspace, stream);
}
#undef GS_BY_TYPE

}  // namespace gs
