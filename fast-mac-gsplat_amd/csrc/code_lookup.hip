// code_lookup.hip -- attributes of splats from a codebook, and the gradient.
//
//   out[n] = f s_n C[c_n]                     (c_n = -1: zeros)
//   gC[k]  = f * sum over n with c_n = k, in ascending n, of s_n g[n]
//   gs[n]  = f <g[n], C[c_n]>
//
// The gradient of the codebook is a sum by code.  The splats are sorted by
// code (stable), so a code's splats are one run of the sorted positions, and
// runs are cut at every kPiece-th position: a piece (a run's part between two
// cuts) is one wavefront's work however the splats are spread over the codes.
// Runs inside one cut are written at once; the others' pieces go to two
// partial rows per cut (one for the run that comes in from the left, one for
// the run that goes on to the right) and are added up by a second launch in
// the order of the positions.  No atomics: the same inputs give the same bits.
#include <algorithm>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 128;  // sorted positions between two cuts

template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_fwd_kernel(
    LookupParams P, const T* __restrict__ codebook,
    const float* __restrict__ scales, T* __restrict__ out) {
  const int64_t total = P.rows * P.D;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * kThreads) {
    const int64_t n = i / P.D;
    const int d = (int)(i - n * P.D);
    const int c = P.codes.at(n, P.K);
    float v = c == kBadCode ? __builtin_nanf("") : 0.0f;
    if (c >= 0) {
      v = to_float(codebook[c * P.stride + d]) * (scales ? P.factor * scales[n] : P.factor);
    }
    out[i] = static_cast<T>(v);
  }
}

__global__ __launch_bounds__(kThreads) void lookup_keys_kernel(
    LookupParams P, uint32_t* __restrict__ keys) {
  const int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (n >= P.rows) return;
  const int c = P.codes.at(n, P.K);
  keys[n] = c >= 0 ? (uint32_t)c : (uint32_t)P.K;  // (no code: after all codes)
}

// edges[k] = the first sorted position whose key is at least k, k = 0..K.
__global__ __launch_bounds__(kThreads) void lookup_edges_kernel(
    const uint32_t* __restrict__ keys, int64_t n, int K,
    int32_t* __restrict__ edges) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i > n) return;
  const int64_t before = i == 0 ? -1 : (int64_t)min(keys[i - 1], (uint32_t)K);
  const int64_t here = i == n ? (int64_t)K : (int64_t)min(keys[i], (uint32_t)K);
  for (int64_t k = before + 1; k <= here; ++k) edges[k] = (int32_t)i;
}

// The code whose pieces hold piece i: code k's pieces are numbered from
// k + edges[k] / kPiece (a number that grows with k by the cuts passed and one).
__device__ __forceinline__ int code_of_piece(const int32_t* edges, int K,
                                             int64_t i) {
  int lo = 0, hi = K - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (mid + edges[mid] / kPiece <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_pieces_kernel(
    LookupParams P, const int32_t* __restrict__ edges,
    const uint32_t* __restrict__ order, const T* __restrict__ grad,
    const float* __restrict__ scales, const uint32_t* __restrict__ err,
    float* __restrict__ partials, T* __restrict__ g_codebook) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int k = code_of_piece(edges, P.K, i);
  const int first = edges[k], end = edges[k + 1];
  const int64_t block = i - k;  // (of the sorted positions, kPiece each)
  const int64_t a = max((int64_t)first, block * kPiece);
  const int64_t b = min((int64_t)end, (block + 1) * kPiece);
  if (i >= P.K + (int64_t)edges[P.K] / kPiece) return;  // past the last piece
  const bool whole = end == first || first / kPiece == (end - 1) / kPiece;
  if (whole ? block != first / kPiece : a >= b) return;  // an empty last piece
  const bool bad = *err != 0;
  for (int d = lane; d < P.D; d += 64) {
    float acc = 0.0f;
    for (int64_t j = a; j < b; ++j) {
      const int64_t n = order[j];
      const float g = to_float(grad[n * P.D + d]);
      acc += scales ? g * scales[n] : g;
    }
    if (bad) acc = __builtin_nanf("");
    if (whole)
      g_codebook[(int64_t)k * P.D + d] = static_cast<T>(acc * P.factor);
    else
      partials[(2 * block + (a == first ? 1 : 0)) * P.D + d] = acc;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_join_kernel(
    LookupParams P, const int32_t* __restrict__ edges,
    const float* __restrict__ partials, T* __restrict__ g_codebook) {
  const int k = (int)blockIdx.x;
  const int first = edges[k], end = edges[k + 1];
  if (end == first || first / kPiece == (end - 1) / kPiece) return;
  for (int d = threadIdx.x; d < P.D; d += kThreads) {
    float acc = partials[(2 * (int64_t)(first / kPiece) + 1) * P.D + d];
    for (int64_t b = first / kPiece + 1; b <= (end - 1) / kPiece; ++b)
      acc += partials[2 * b * P.D + d];
    g_codebook[(int64_t)k * P.D + d] = static_cast<T>(acc * P.factor);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_scales_kernel(
    LookupParams P, const T* __restrict__ grad, const T* __restrict__ codebook,
    float* __restrict__ g_scales) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (n >= P.rows) return;
  const int c = P.codes.at(n, P.K);
  float acc = 0.0f;
  if (c >= 0)
    for (int d = lane; d < P.D; d += 64)
      acc += to_float(grad[n * P.D + d]) * to_float(codebook[c * P.stride + d]);
  acc = wave_sum(acc);
  if (lane == 0) g_scales[n] = c == kBadCode ? __builtin_nanf("") : acc * P.factor;
}

struct Layout {
  RadixPlan sort;
  size_t ctl, buffers, keys, sorted, order, edges, partials, total;
};

Layout layout(const LookupParams& P) {
  Layout L{};
  int bits = 1;
  while (bits < 32 && (int64_t(1) << bits) <= P.K) ++bits;
  L.sort = radix_plan(P.rows, 1, 0, bits);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += align_up(bytes, 256);
    return at;
  };
  L.ctl = take(radix_ctl_bytes(L.sort));
  L.buffers = take(L.sort.buffer_bytes);
  L.keys = take((size_t)P.rows * 4);
  L.sorted = take((size_t)P.rows * 4);
  L.order = take((size_t)P.rows * 4);
  L.edges = take((size_t)(P.K + 1) * 4);
  L.partials = take((size_t)(P.rows / kPiece + 1) * 2 * P.D * 4);
  L.total = off;
  return L;
}

template <typename T>
int forward_of(const LookupParams& P, const void* codebook, const float* scales,
               void* out, hipStream_t stream) {
  const int64_t total = P.rows * P.D;
  const int64_t grid = std::min<int64_t>((total + kThreads - 1) / kThreads, 1 << 20);
  launch_traced("lookup_fwd_kernel", (lookup_fwd_kernel<T>), dim3((unsigned)grid),
                dim3(kThreads), 0, stream, P, static_cast<const T*>(codebook),
                scales, static_cast<T*>(out));
  return check_launch("lookup_fwd_kernel");
}

template <typename T>
int backward_of(const LookupParams& P, const void* grad_out, const void* codebook,
                const float* scales, void* g_codebook, float* g_scales,
                void* workspace, hipStream_t stream) {
  const T* grad = static_cast<const T*>(grad_out);
  if (g_scales && P.rows > 0) {
    launch_traced("lookup_scales_kernel", (lookup_scales_kernel<T>),
                  dim3((unsigned)((P.rows + 3) / 4)), dim3(kThreads), 0, stream, P,
                  grad, static_cast<const T*>(codebook), g_scales);
    const int rc = check_launch("lookup_scales_kernel");
    if (rc) return rc;
  }
  if (!g_codebook) return GSPLAT_OK;
  const Layout L = layout(P);
  char* w = static_cast<char*>(workspace);
  auto* keys = reinterpret_cast<uint32_t*>(w + L.keys);
  auto* sorted = reinterpret_cast<uint32_t*>(w + L.sorted);
  auto* order = reinterpret_cast<uint32_t*>(w + L.order);
  auto* edges = reinterpret_cast<int32_t*>(w + L.edges);
  auto* partials = reinterpret_cast<float*>(w + L.partials);
  const RadixCtl C = radix_ctl_at(L.sort, w + L.ctl);
  int rc = GSPLAT_OK;
  if (P.rows > 0) {
    launch_traced("lookup_keys_kernel", lookup_keys_kernel,
                  dim3((unsigned)((P.rows + kThreads - 1) / kThreads)),
                  dim3(kThreads), 0, stream, P, keys);
    rc = check_launch("lookup_keys_kernel");
  }
  if (!rc) rc = launch_zero_u32(C.ghist, (int64_t)radix_ctl_bytes(L.sort) / 4, stream);
  if (!rc) rc = radix_global_hist(L.sort, C, keys, nullptr, stream);
  if (!rc)
    rc = radix_passes(L.sort, C, w + L.buffers, keys, nullptr, nullptr, sorted,
                      order, stream);
  if (rc) return rc;
  launch_traced("lookup_edges_kernel", lookup_edges_kernel,
                dim3((unsigned)((P.rows + kThreads) / kThreads)), dim3(kThreads), 0,
                stream, sorted, P.rows, P.K, edges);
  rc = check_launch("lookup_edges_kernel");
  if (rc) return rc;
  const int64_t pieces = P.K + P.rows / kPiece + 1;
  launch_traced("lookup_pieces_kernel", (lookup_pieces_kernel<T>),
                dim3((unsigned)((pieces + 3) / 4)), dim3(kThreads), 0, stream, P,
                edges, order, grad, scales, C.err, partials,
                static_cast<T*>(g_codebook));
  rc = check_launch("lookup_pieces_kernel");
  if (rc) return rc;
  launch_traced("lookup_join_kernel", (lookup_join_kernel<T>), dim3((unsigned)P.K),
                dim3(kThreads), 0, stream, P, edges, partials,
                static_cast<T*>(g_codebook));
  return check_launch("lookup_join_kernel");
}

}  // namespace

size_t lookup_backward_workspace_bytes(const LookupParams& P) {
  return layout(P).total;
}

int launch_lookup_forward(const LookupParams& P, const void* codebook,
                          const float* scales, void* out, hipStream_t stream) {
  if (P.rows == 0) return GSPLAT_OK;
  if (P.dtype == GSPLAT_F32)
    return forward_of<float>(P, codebook, scales, out, stream);
  if (P.dtype == GSPLAT_BF16)
    return forward_of<__bf16>(P, codebook, scales, out, stream);
  return forward_of<_Float16>(P, codebook, scales, out, stream);
}

int launch_lookup_backward(const LookupParams& P, const void* grad_out,
                           const void* codebook, const float* scales,
                           void* g_codebook, float* g_scales, void* workspace,
                           hipStream_t stream) {
  if (P.dtype == GSPLAT_F32)
    return backward_of<float>(P, grad_out, codebook, scales, g_codebook, g_scales,
                              workspace, stream);
  if (P.dtype == GSPLAT_BF16)
    return backward_of<__bf16>(P, grad_out, codebook, scales, g_codebook, g_scales,
                               workspace, stream);
  return backward_of<_Float16>(P, grad_out, codebook, scales, g_codebook, g_scales,
                               workspace, stream);
}

}  // namespace gs
