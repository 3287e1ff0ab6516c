// code_groups.hip -- splats' rows sorted by code and back.
//
//   order, places, starts: the choices sorted by code (stable), those without a
//                          code last; place of each choice; where codes begin
//   by code       y[j] = x[order[j] / S]              (S choices per splat)
//   from codes    x[n] = sum_s w[n,s] y[places[n,s]]
//
// Each is the other's gradient (with weights of 1, or w[order[j]]), and
// gw[n,s] = <gx[n], y[places[n,s]]>.  Sums are over s in its order: the same
// inputs give the same bits.
//
// Places are checked where they are read: a place outside the rows makes its
// splat NaN, as a code outside [0, K) does.
#include <algorithm>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;

// ---- sorting

__global__ __launch_bounds__(kThreads) void group_keys_kernel(
    GroupParams P, uint32_t* __restrict__ keys, uint32_t* __restrict__ ctl,
    int64_t ctl_words) {
  const int64_t step = (int64_t)gridDim.x * kThreads;
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t i = t; i < P.choices; i += step) {
    const int c = P.codes.at(i, P.K);
    keys[i] = c >= 0 ? (uint32_t)c : (uint32_t)P.K;
  }
  for (int64_t i = t; i < ctl_words; i += step) ctl[i] = 0;
}

// Places from the order, and where codes begin (a thread per code looks for it in
// the sorted keys).  A sort that gave up leaves no places: the choices count as
// codes out of range.
__global__ __launch_bounds__(kThreads) void group_finish_kernel(
    GroupParams P, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ err, int32_t* __restrict__ order,
    int32_t* __restrict__ places, int32_t* __restrict__ starts) {
  const int64_t step = (int64_t)gridDim.x * kThreads;
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const bool gave_up = err != nullptr && *err != 0;
  for (int64_t j = t; j < P.choices; j += step) {
    if (gave_up) {
      order[j] = (int32_t)j;
      places[j] = kBadCode;
    } else {
      const int32_t i = order[j];
      places[i] = keys[j] < (uint32_t)P.K ? (int32_t)j : P.codes.at(i, P.K);
    }
  }
  for (int64_t k = t; k <= P.K; k += step) {
    int64_t lo = 0, hi = gave_up ? 0 : P.choices;  // the first place of code k or above
    while (lo < hi) {
      const int64_t mid = (lo + hi) / 2;
      if (keys[mid] < (uint32_t)k) lo = mid + 1;
      else hi = mid;
    }
    starts[k] = (int32_t)lo;
  }
}

struct SortLayout {
  RadixPlan sort;
  size_t ctl, buffers, keys, sorted, total;
};

SortLayout sort_layout(const GroupParams& P) {
  SortLayout L{};
  if (P.choices == 0) return L;
  int bits = 1;
  while (bits < 32 && (int64_t(1) << bits) <= P.K) ++bits;
  L.sort = radix_plan(P.choices, 1, 0, bits);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += align_up(bytes, 256);
    return at;
  };
  L.ctl = take(radix_ctl_bytes(L.sort));
  L.buffers = take(L.sort.buffer_bytes);
  L.keys = take((size_t)P.choices * 4);
  L.sorted = take((size_t)P.choices * 4);
  L.total = off;
  return L;
}

// ---- rows

// What a place says of its choice: 0 a row, else kNoCode or kBadCode.
__device__ __forceinline__ int state_of(int place, int64_t rows) {
  if (place >= 0 && place < rows) return 0;
  return place == kNoCode ? kNoCode : kBadCode;
}

// The splat of the choice at place j, -1 or -2 where there is none; w its weight.
__device__ __forceinline__ int64_t splat_at(const RowsParams& P, int64_t j,
                                            const int32_t* order,
                                            const int32_t* places,
                                            const float* weights, float& w) {
  const int64_t all = P.splats * P.choices;
  const int64_t i = order[j];
  w = 1.0f;
  if (i < 0 || i >= all) return kBadCode;
  const int s = state_of(places[i], all);
  if (s != 0) return s;
  if (weights) w = weights[i];
  return i / P.choices;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void rows_by_code_kernel(
    RowsParams P, const T* __restrict__ rows, const int32_t* __restrict__ order,
    const int32_t* __restrict__ places, const float* __restrict__ weights,
    T* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t j = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (j >= P.splats * P.choices) return;
  float w;
  const int64_t n = splat_at(P, j, order, places, weights, w);
  for (int d = lane; d < P.D; d += 64)
    out[j * P.D + d] =
        static_cast<T>(n < 0 ? nan_for((int)n) : w * to_float(rows[n * P.stride + d]));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void rows_from_codes_kernel(
    RowsParams P, const T* __restrict__ rows, const int32_t* __restrict__ places,
    const float* __restrict__ weights, T* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (n >= P.splats) return;
  for (int d = lane; d < P.D; d += 64) {
    float a = 0.0f;
    for (int s = 0; s < P.choices; ++s) {
      const int64_t i = n * P.choices + s;
      const int at = places[i], state = state_of(at, P.splats * P.choices);
      if (state != 0) a += nan_for(state);
      else a = __builtin_fmaf(weights ? weights[i] : 1.0f, to_float(rows[at * P.stride + d]), a);
    }
    out[n * P.D + d] = static_cast<T>(a);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void rows_from_bwd_kernel(
    RowsParams P, const T* __restrict__ grad, const T* __restrict__ rows,
    const int32_t* __restrict__ order, const int32_t* __restrict__ places,
    const float* __restrict__ weights, T* __restrict__ g_rows,
    float* __restrict__ g_weights) {
  const int lane = threadIdx.x & 63;
  const int64_t j = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (j >= P.splats * P.choices) return;
  float w;
  const int64_t n = splat_at(P, j, order, places, weights, w);
  float dot = 0.0f;
  for (int d = lane; d < P.D; d += 64) {
    const float g = n < 0 ? nan_for((int)n) : to_float(grad[n * P.D + d]);
    if (g_rows) g_rows[j * P.D + d] = static_cast<T>(w * g);
    if (g_weights && n >= 0) dot = __builtin_fmaf(g, to_float(rows[j * P.stride + d]), dot);
  }
  if (!g_weights) return;
  dot = wave_sum(dot);
  const int64_t i = order[j];
  if (lane == 0 && i >= 0 && i < P.splats * P.choices)
    g_weights[i] = n < 0 ? nan_for((int)n) : dot;
}

template <typename T>
int by_code_of(const RowsParams& P, const void* rows, const int32_t* order,
               const int32_t* places, const float* weights, void* out,
               hipStream_t stream) {
  const int64_t all = P.splats * P.choices;
  launch_traced("rows_by_code_kernel", (rows_by_code_kernel<T>),
                dim3((unsigned)((all + 3) / 4)), dim3(kThreads), 0, stream, P,
                static_cast<const T*>(rows), order, places, weights, static_cast<T*>(out));
  return check_launch("rows_by_code_kernel");
}

template <typename T>
int from_codes_of(const RowsParams& P, const void* rows, const int32_t* places,
                  const float* weights, void* out, hipStream_t stream) {
  launch_traced("rows_from_codes_kernel", (rows_from_codes_kernel<T>),
                dim3((unsigned)((P.splats + 3) / 4)), dim3(kThreads), 0, stream, P,
                static_cast<const T*>(rows), places, weights, static_cast<T*>(out));
  return check_launch("rows_from_codes_kernel");
}

template <typename T>
int from_codes_bwd_of(const RowsParams& P, const void* grad, const void* rows,
                      const int32_t* order, const int32_t* places,
                      const float* weights, void* g_rows, float* g_weights,
                      hipStream_t stream) {
  const int64_t all = P.splats * P.choices;
  launch_traced("rows_from_bwd_kernel", (rows_from_bwd_kernel<T>),
                dim3((unsigned)((all + 3) / 4)), dim3(kThreads), 0, stream, P,
                static_cast<const T*>(grad), static_cast<const T*>(rows), order, places,
                weights, static_cast<T*>(g_rows), g_weights);
  return check_launch("rows_from_bwd_kernel");
}

}  // namespace

size_t group_workspace_bytes(const GroupParams& P) { return sort_layout(P).total; }

int launch_group_codes(const GroupParams& P, int32_t* order, int32_t* places,
                       int32_t* starts, void* workspace, hipStream_t stream) {
  uint32_t *sorted = nullptr, *err = nullptr;
  if (P.choices > 0) {
    const SortLayout L = sort_layout(P);
    char* w = static_cast<char*>(workspace);
    auto* keys = reinterpret_cast<uint32_t*>(w + L.keys);
    sorted = reinterpret_cast<uint32_t*>(w + L.sorted);
    const RadixCtl C = radix_ctl_at(L.sort, w + L.ctl);
    err = C.err;
    launch_traced("group_keys_kernel", group_keys_kernel,
                  dim3((unsigned)std::min<int64_t>((P.choices + kThreads - 1) / kThreads, 2048)),
                  dim3(kThreads), 0, stream, P, keys, C.ghist,
                  (int64_t)radix_ctl_bytes(L.sort) / 4);
    int rc = check_launch("group_keys_kernel");
    if (!rc) rc = radix_global_hist(L.sort, C, keys, nullptr, stream);
    if (!rc)
      rc = radix_passes(L.sort, C, w + L.buffers, keys, nullptr, nullptr, sorted,
                        reinterpret_cast<uint32_t*>(order), stream);
    if (rc) return rc;
  }
  launch_traced("group_finish_kernel", group_finish_kernel,
                dim3((unsigned)std::min<int64_t>(
                    std::max<int64_t>(P.choices, (int64_t)P.K + 1) / kThreads + 1, 65536)),
                dim3(kThreads), 0, stream, P, sorted, err, order, places, starts);
  return check_launch("group_finish_kernel");
}

#define GS_BY_TYPE(F)                                         \
  (P.dtype == GSPLAT_F32 ? F<float> : P.dtype == GSPLAT_BF16 ? F<__bf16> : F<_Float16>)

int launch_rows_by_code(const RowsParams& P, const void* rows,
                        const int32_t* order, const int32_t* places,
                        const float* weights, void* out, hipStream_t stream) {
  return GS_BY_TYPE(by_code_of)(P, rows, order, places, weights, out, stream);
}

int launch_rows_from_codes(const RowsParams& P, const void* rows,
                           const int32_t* places, const float* weights,
                           void* out, hipStream_t stream) {
  return GS_BY_TYPE(from_codes_of)(P, rows, places, weights, out, stream);
}

int launch_rows_from_codes_backward(const RowsParams& P, const void* grad,
                                    const void* rows, const int32_t* order,
                                    const int32_t* places, const float* weights,
                                    void* g_rows, float* g_weights,
                                    hipStream_t stream) {
  return GS_BY_TYPE(from_codes_bwd_of)(P, grad, rows, order, places, weights, g_rows,
                                       g_weights, stream);
}
#undef GS_BY_TYPE

}  // namespace gs
