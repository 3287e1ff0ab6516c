// code_adapters.hip -- low-rank maps of splats' rows, each by its code's own.
//
//   h[j]   = down[c] x[n]                  (n: the splat at place j, c its code)
//   out[n] = base[n] + scale * up[c] h[j]
//   dh[j]  = scale * up[c]^T g[n]
//   gx[n]  = down[c]^T dh[j]
//   gdown[c] = sum over c's places of dh[j] x[n]^T,  gup[c] = scale * sum of g[n] h[j]^T
//
// A splat without a code has out = base and no gradient; one with a code out of
// range is NaN.
#include <algorithm>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;

// The code of place j: the last one that starts at or before it; K and more past
// the last code's end.
__device__ __forceinline__ int code_at(const AdapterParams& P, int64_t j) {
  int lo = 0, hi = P.K;  // starts[lo] <= j < starts[hi] (starts[K] too: none)
  if (j >= P.starts[P.K]) return P.K;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (P.starts[mid] <= j) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The row of place j (-1: out of range).
__device__ __forceinline__ int64_t row_at(const AdapterParams& P, int64_t j) {
  if (P.by_code) return j;
  const int64_t n = P.order[j];
  return n >= 0 && n < P.rows ? n : -1;
}

__device__ __forceinline__ float rest_value(const AdapterParams& P, int64_t j) {
  const int64_t i = P.order[j];
  return i >= 0 && i < P.rows && P.places[i] == kNoCode ? 0.0f : __builtin_nanf("");
}

// A wavefront per place: dots of x with the r rows of down (or of g with the
// columns of up).
template <typename T>
__global__ __launch_bounds__(kThreads) void adapters_hidden_kernel(
    AdapterParams P, const T* __restrict__ rows, int64_t stride, int D,
    const T* __restrict__ map, int64_t map_k, int64_t map_d, float factor,
    float* __restrict__ hidden) {
  const int lane = threadIdx.x & 63;
  const int64_t j = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (j >= P.rows) return;
  const int c = code_at(P, j);
  const int64_t n = row_at(P, j);
  for (int k = 0; k < P.r; ++k) {
    float a = 0.0f;
    if (c < P.K && n >= 0)
      for (int d = lane; d < D; d += 64)
        a = __builtin_fmaf(to_float(rows[n * stride + d]),
                           to_float(map[(int64_t)c * P.r * D + k * map_k + d * map_d]), a);
    a = wave_sum(a);
    if (lane == 0) hidden[j * P.r + k] = a * factor;
  }
}

// A wavefront per place: sums over the r values of its hidden row.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapters_out_kernel(
    AdapterParams P, const float* __restrict__ hidden, int E,
    const T* __restrict__ map, int64_t map_k, int64_t map_e, float factor,
    const T* __restrict__ base, T* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t j = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (j >= P.rows) return;
  const int c = code_at(P, j);
  const int64_t n = row_at(P, j);
  if (n < 0) return;
  for (int e = lane; e < E; e += 64) {
    float a = 0.0f;
    if (c < P.K)
      for (int k = 0; k < P.r; ++k)
        a = __builtin_fmaf(hidden[j * P.r + k],
                           to_float(map[(int64_t)c * P.r * E + k * map_k + e * map_e]), a);
    else
      a = rest_value(P, j);
    a *= factor;
    out[n * E + e] = static_cast<T>(base ? to_float(base[n * E + e]) + a : a);
  }
}

// Gradients of the maps: a thread per value, over its code's places.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapters_maps_kernel(
    AdapterParams P, const float* __restrict__ hidden, const T* __restrict__ rows,
    int64_t stride, int D, int64_t map_k, int64_t map_d, float factor,
    T* __restrict__ g_map) {
  const int64_t all = (int64_t)P.K * P.r * D;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= all) return;
  const int c = (int)(at / (P.r * D)), i = (int)(at - (int64_t)c * P.r * D);
  const int k = i / D, d = i - k * D;
  const int64_t from = max(P.starts[c], 0), to = min((int64_t)P.starts[c + 1], P.rows);
  float a = 0.0f;
  for (int64_t j = from; j < to; ++j) {
    const int64_t n = row_at(P, j);
    if (n >= 0) a = __builtin_fmaf(hidden[j * P.r + k], to_float(rows[n * stride + d]), a);
  }
  g_map[(int64_t)c * P.r * D + k * map_k + d * map_d] = static_cast<T>(a * factor);
}

template <typename T>
int forward_of(const AdapterParams& P, const void* rows, const void* down,
               const void* up, const void* base, void* out, float* hidden,
               hipStream_t stream) {
  const dim3 grid((unsigned)((P.rows + 3) / 4));
  launch_traced("adapters_hidden_kernel", (adapters_hidden_kernel<T>), grid, dim3(kThreads),
                0, stream, P, static_cast<const T*>(rows), P.stride, P.D,
                static_cast<const T*>(down), (int64_t)P.D, (int64_t)1, 1.0f, hidden);
  int rc = check_launch("adapters_hidden_kernel");
  if (rc) return rc;
  launch_traced("adapters_out_kernel", (adapters_out_kernel<T>), grid, dim3(kThreads), 0,
                stream, P, hidden, P.E, static_cast<const T*>(up), (int64_t)1,
                (int64_t)P.r, P.scale, static_cast<const T*>(base), static_cast<T*>(out));
  return check_launch("adapters_out_kernel");
}

template <typename T>
int backward_of(const AdapterParams& P, const void* grad, const void* rows,
                const void* down, const void* up, const float* hidden,
                void* g_rows, void* g_down, void* g_up, float* g_hidden,
                hipStream_t stream) {
  const dim3 grid((unsigned)((P.rows + 3) / 4));
  int rc = GSPLAT_OK;
  if ((g_rows || g_down) && P.rows > 0) {
    launch_traced("adapters_hidden_kernel", (adapters_hidden_kernel<T>), grid,
                  dim3(kThreads), 0, stream, P, static_cast<const T*>(grad), (int64_t)P.E,
                  P.E, static_cast<const T*>(up), (int64_t)1, (int64_t)P.r, P.scale, g_hidden);
    rc = check_launch("adapters_hidden_kernel");
    if (rc) return rc;
  }
  if (g_rows && P.rows > 0) {
    launch_traced("adapters_out_kernel", (adapters_out_kernel<T>), grid, dim3(kThreads), 0,
                  stream, P, g_hidden, P.D, static_cast<const T*>(down), (int64_t)P.D,
                  (int64_t)1, 1.0f, static_cast<const T*>(nullptr), static_cast<T*>(g_rows));
    rc = check_launch("adapters_out_kernel");
    if (rc) return rc;
  }
  if (g_down) {
    launch_traced("adapters_maps_kernel", (adapters_maps_kernel<T>),
                  dim3((unsigned)(((int64_t)P.K * P.r * P.D + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream,
                  P, g_hidden, static_cast<const T*>(rows), P.stride, P.D, (int64_t)P.D,
                  (int64_t)1, 1.0f, static_cast<T*>(g_down));
    rc = check_launch("adapters_maps_kernel");
    if (rc) return rc;
  }
  if (g_up) {
    launch_traced("adapters_maps_kernel", (adapters_maps_kernel<T>),
                  dim3((unsigned)(((int64_t)P.K * P.r * P.E + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream,
                  P, hidden, static_cast<const T*>(grad), (int64_t)P.E, P.E, (int64_t)1,
                  (int64_t)P.r, P.scale, static_cast<T*>(g_up));
    rc = check_launch("adapters_maps_kernel");
  }
  return rc;
}

}  // namespace

size_t adapters_forward_workspace_bytes(const AdapterParams& P) {
  return (size_t)P.rows * P.r * 4;
}
size_t adapters_backward_workspace_bytes(const AdapterParams& P) {
  return (size_t)P.rows * P.r * 4;
}

#define GS_BY_TYPE(F)                                         \
  (P.dtype == GSPLAT_F32 ? F<float> : P.dtype == GSPLAT_BF16 ? F<__bf16> : F<_Float16>)

int launch_adapters_forward(const AdapterParams& P, const void* rows,
                            const void* down, const void* up, const void* base,
                            void* out, float* hidden, void* workspace,
                            hipStream_t stream) {
  return GS_BY_TYPE(forward_of)(P, rows, down, up, base, out,
                                hidden ? hidden : static_cast<float*>(workspace), stream);
}

int launch_adapters_backward(const AdapterParams& P, const void* grad,
                             const void* rows, const void* down, const void* up,
                             const float* hidden, void* g_rows, void* g_down,
                             void* g_up, void* workspace, hipStream_t stream) {
  return GS_BY_TYPE(backward_of)(P, grad, rows, down, up, hidden, g_rows, g_down, g_up,
                                 static_cast<float*>(workspace), stream);
}
#undef GS_BY_TYPE

}  // namespace gs
