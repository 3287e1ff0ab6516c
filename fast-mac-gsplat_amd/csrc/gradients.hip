// gradients.hip -- the norm of many tensors together, and their clipping.
//
//   norm = sqrt(sum of all squares),  out = g * min(1, max_norm / norm)
//
// Two launches: sums of squares, a number per workgroup; then every workgroup
// adds those up itself (in their order: each has the same bits) and scales what
// it owns.  Tensors come as a table in the kernel's arguments, kTable of them a
// launch, cut into chunks of `chunk` elements; a workgroup finds its tensor in
// the table.  Nothing is copied to the device for it, so that a captured call
// needs no host memory later.
//
// Squares are added in 64 bits: they are exact there, a sum of 2^32 of them is
// within 2^-20 of a rounding to 32 bits, and no square overflows.
// What bounds it, on an MI355X: 68 million values in 305 tensors, 261 MB, 60 us of
// sums (one tensor of 201 MB at 5.2 TB/s, 176 small ones at latency) and 15 of the
// second launches, which write nothing where nothing is clipped; the host's checks
// of 305 tensors take 60.  Seven tensors, 0.2 MB: two launches of 4 us.
//
// A norm that is not finite, as the float that the caller gets, leaves the
// gradients as they are.
#include <algorithm>

#include "codes.h"
#include "gradients.h"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 128;

struct Table {
  const void* from[kTable];
  void* to[kTable];
  int64_t size[kTable];
  int first[kTable];  // the tensor's first workgroup
  uint8_t dtype[kTable];
  int count;
};

__device__ __forceinline__ int tensor_of(const Table& A, int block) {
  int lo = 0, hi = A.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (A.first[mid] <= block) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double squares(const T* x, int64_t n) {
  constexpr int V = kVec<T>;
  double a[V];
#pragma unroll
  for (int v = 0; v < V; ++v) a[v] = 0.0;
  int64_t i = (int64_t)threadIdx.x * V;
  auto add = [&](vec_t<T> y) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const double z = (double)to_float(y[v]);
      a[v] = __builtin_fma(z, z, a[v]);
    }
  };
  // (four loads on their way at a time)
  for (; i + 3 * kThreads * V + V <= n; i += 4 * kThreads * V) {
    vec_t<T> y[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) y[u] = load_vec(x + i + u * kThreads * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) add(y[u]);
  }
  for (; i + V <= n; i += kThreads * V) add(load_vec(x + i));
  for (; i < n; ++i) {
    const double z = (double)to_float(x[i]);
    a[0] = __builtin_fma(z, z, a[0]);
  }
#pragma unroll
  for (int v = V / 2; v > 0; v /= 2)
#pragma unroll
    for (int u = 0; u < v; ++u) a[u] += a[u + v];
  return a[0];
}

__device__ __forceinline__ double block_sum_f64(double v) {
  __shared__ double red[kThreads / 64];
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) r += red[w];
  return r;
}

__global__ __launch_bounds__(kThreads) void clip_sums_kernel(Table A, int64_t chunk,
                                                             double* __restrict__ sums) {
  const int t = tensor_of(A, blockIdx.x);
  const int64_t from = (int64_t)(blockIdx.x - A.first[t]) * chunk;
  const int64_t n = min(chunk, A.size[t] - from);
  double a = 0.0;
  if (A.dtype[t] == GSPLAT_F32) a = squares(static_cast<const float*>(A.from[t]) + from, n);
  else if (A.dtype[t] == GSPLAT_BF16) a = squares(static_cast<const __bf16*>(A.from[t]) + from, n);
  else a = squares(static_cast<const _Float16*>(A.from[t]) + from, n);
  a = block_sum_f64(a);
  if (threadIdx.x == 0) sums[blockIdx.x] = a;
}

// All sums to one, where there are too many for every workgroup to add up.
__global__ __launch_bounds__(kThreads) void clip_join_kernel(const double* __restrict__ sums,
                                                             int64_t n, double* __restrict__ out) {
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += kThreads) a += sums[i];
  a = block_sum_f64(a);
  if (threadIdx.x == 0) *out = a;
}

template <typename T>
__device__ __forceinline__ void scale(const T* x, T* y, int64_t n, float f) {
  constexpr int V = kVec<T>;
  int64_t i = (int64_t)threadIdx.x * V;
  auto put = [&](int64_t at, vec_t<T> z) {
    if (f != 1.0f)
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = static_cast<T>(to_float(z[v]) * f);
    store_vec(y + at, z);
  };
  for (; i + 3 * kThreads * V + V <= n; i += 4 * kThreads * V) {
    vec_t<T> z[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] = load_vec(x + i + u * kThreads * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) put(i + u * kThreads * V, z[u]);
  }
  for (; i + V <= n; i += kThreads * V) put(i, load_vec(x + i));
  for (; i < n; ++i) y[i] = f != 1.0f ? static_cast<T>(to_float(x[i]) * f) : x[i];
}

__global__ __launch_bounds__(kThreads) void clip_scale_kernel(
    Table A, int64_t chunk, const double* __restrict__ sums, int64_t n_sums,
    double max_norm, float* __restrict__ norm_out) {
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n_sums; i += kThreads) a += sums[i];
  const double norm = __builtin_sqrt(block_sum_f64(a));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const bool finite = (float)norm < __builtin_inff();
  const float f = finite && norm > max_norm ? (float)(max_norm / norm) : 1.0f;
  if (A.count == 0) return;
  const int t = tensor_of(A, blockIdx.x);
  if (f == 1.0f && A.from[t] == A.to[t]) return;
  const int64_t from = (int64_t)(blockIdx.x - A.first[t]) * chunk;
  const int64_t n = min(chunk, A.size[t] - from);
  const int d = A.dtype[t];
  if (d == GSPLAT_F32)
    scale(static_cast<const float*>(A.from[t]) + from, static_cast<float*>(A.to[t]) + from, n, f);
  else if (d == GSPLAT_BF16)
    scale(static_cast<const __bf16*>(A.from[t]) + from, static_cast<__bf16*>(A.to[t]) + from, n, f);
  else
    scale(static_cast<const _Float16*>(A.from[t]) + from, static_cast<_Float16*>(A.to[t]) + from, n, f);
}

// Elements of a chunk: as many as make about 4096 workgroups of all, 4096 to 2^24.
int64_t chunk_of(const ClipTensor* x, int64_t count) {
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) all += x[i].size;
  int64_t c = 4096;
  while (c < int64_t(1) << 24 && c * 4096 < all) c *= 2;
  return c;
}
int64_t blocks_of(const ClipTensor* x, int64_t count, int64_t chunk) {
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) n += (x[i].size + chunk - 1) / chunk;
  return n;
}
constexpr int64_t kMostSums = 8192;  // that every workgroup adds up itself

}  // namespace

size_t clip_workspace_bytes(const ClipTensor* x, int64_t count) {
  return (size_t)(blocks_of(x, count, chunk_of(x, count)) + 1) * sizeof(double);
}

int launch_clip(const ClipTensor* x, int64_t count, double max_norm, float* norm,
                void* workspace, hipStream_t stream) {
  const int64_t chunk = chunk_of(x, count), n_sums = blocks_of(x, count, chunk);
  auto* sums = static_cast<double*>(workspace);
  // launch(table, workgroups, first workgroup of all) for every table's worth
  auto in_tables = [&](auto launch) {
    int64_t before = 0;
    for (int64_t i = 0; i < count;) {
      Table A{};
      int64_t blocks = 0;
      for (; i < count && A.count < kTable; ++i) {
        if (x[i].size == 0) continue;
        const int k = A.count++;
        A.from[k] = x[i].from;
        A.to[k] = x[i].to;
        A.size[k] = x[i].size;
        A.dtype[k] = (uint8_t)x[i].dtype;
        A.first[k] = (int)blocks;
        blocks += (x[i].size + chunk - 1) / chunk;
      }
      if (blocks == 0) continue;
      const int rc = launch(A, blocks, before);
      if (rc) return rc;
      before += blocks;
    }
    return (int)GSPLAT_OK;
  };
  int rc = in_tables([&](const Table& A, int64_t blocks, int64_t before) {
    launch_traced("clip_sums_kernel", clip_sums_kernel, dim3((unsigned)blocks), dim3(kThreads), 0,
                  stream, A, chunk, sums + before);
    return check_launch("clip_sums_kernel");
  });
  if (rc) return rc;
  const double* from = sums;
  int64_t n = n_sums;
  if (n > kMostSums) {
    launch_traced("clip_join_kernel", clip_join_kernel, dim3(1), dim3(kThreads), 0, stream, sums, n,
                  sums + n);
    if ((rc = check_launch("clip_join_kernel"))) return rc;
    from = sums + n;
    n = 1;
  }
  if (n_sums == 0) {
    launch_traced("clip_scale_kernel", clip_scale_kernel, dim3(1), dim3(kThreads), 0, stream, Table{},
                  chunk, from, n, max_norm, norm);
    return check_launch("clip_scale_kernel");
  }
  return in_tables([&](const Table& A, int64_t blocks, int64_t before) {
    launch_traced("clip_scale_kernel", clip_scale_kernel, dim3((unsigned)blocks), dim3(kThreads), 0,
                  stream, A, chunk, from, n, max_norm, before == 0 ? norm : nullptr);
    return check_launch("clip_scale_kernel");
  });
}

}  // namespace gs
