// code_balance.hip -- how evenly the splats of an image use the codes.
//
//   f_k = (choices of code k) / (all choices),  P_k = mean over rows of p_nk
//   loss = K * sum_k f_k P_k          (1 when both are even; per image)
//   dL/dx_n = p_n (a - <a, p_n>) / rows,   a_k = K f_k g_loss + g_mean_k
//
// p_n is the softmax of row n's logits; a row without any code takes no part
// (nor does it count among the rows), a row with no logit above -inf has
// p = 0.  No gradient passes through the counts.  A code outside [-1, K) is
// not counted and makes its image's loss NaN.
//
// Sums over rows are taken in a fixed order (chunks of rows, then the chunks),
// counts are integers: the same inputs give the same bits.
#include <algorithm>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kChunk = 256;  // rows whose probabilities one workgroup adds up

// One wavefront per row: stats = {max, 1 / sum}, {., 0} for a row that takes
// no part; the row's choices are counted (counts and totals zero on entry).
// totals[b] = {rows that take part, choices, bad codes, 0}
template <typename T>
__global__ __launch_bounds__(kThreads) void balance_rows_kernel(
    BalanceParams P, const T* __restrict__ logits, int32_t* __restrict__ counts,
    float2* __restrict__ stats, int32_t* __restrict__ totals) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (r >= P.rows * P.batch) return;
  const int b = (int)(r / P.rows);
  const T* row = logits + r * P.stride;
  float m = -INFINITY;
  for (int i = lane; i < P.K; i += 64) m = fmaxf(m, to_float(row[i]));
  m = wave_max(m);
  if (m == -INFINITY) m = 0.0f;
  float s = 0.0f;
  for (int i = lane; i < P.K; i += 64) s += __expf(to_float(row[i]) - m);
  s = wave_sum(s);
  if (lane == 0) {
    int given = 0, bad = 0;
    for (int j = 0; j < P.choices; ++j) {
      const int c = P.codes.at(r * P.choices + j, P.K);
      if (c >= 0) {
        ++given;
        atomicAdd(&counts[(int64_t)b * P.K + c], 1);
      } else if (c == kBadCode) {
        ++bad;
      }
    }
    if (given) {
      atomicAdd(&totals[4 * b], 1);
      atomicAdd(&totals[4 * b + 1], given);
    }
    if (bad) atomicAdd(&totals[4 * b + 2], bad);
    stats[r] = make_float2(m, given && s != 0.0f ? 1.0f / s : 0.0f);
  }
}

__device__ __forceinline__ float prob(float x, float2 st) {
  return st.y == 0.0f ? 0.0f : __expf(x - st.x) * st.y;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void balance_columns_kernel(
    BalanceParams P, const T* __restrict__ logits,
    const float2* __restrict__ stats, int chunks, float* __restrict__ partials) {
  const int k = blockIdx.x * kThreads + threadIdx.x;
  const int chunk = blockIdx.y, b = blockIdx.z;
  if (k >= P.K) return;
  const int64_t end = min((int64_t)(chunk + 1) * kChunk, P.rows);
  float acc = 0.0f;
  for (int64_t n = (int64_t)chunk * kChunk; n < end; ++n) {
    const int64_t r = b * P.rows + n;
    acc += prob(to_float(logits[r * P.stride + k]), stats[r]);
  }
  partials[((int64_t)b * chunks + chunk) * P.K + k] = acc;
}

__global__ __launch_bounds__(kThreads) void balance_mean_kernel(
    BalanceParams P, const float* __restrict__ partials, int chunks,
    const int32_t* __restrict__ totals, float* __restrict__ mean) {
  const int k = blockIdx.x * kThreads + threadIdx.x, b = blockIdx.y;
  if (k >= P.K) return;
  float acc = 0.0f;
  for (int c = 0; c < chunks; ++c)
    acc += partials[((int64_t)b * chunks + c) * P.K + k];
  mean[(int64_t)b * P.K + k] = acc / (float)max(totals[4 * b], 1);
}

__global__ __launch_bounds__(kThreads) void balance_loss_kernel(
    BalanceParams P, const float* __restrict__ mean,
    const int32_t* __restrict__ counts, const int32_t* __restrict__ totals,
    float* __restrict__ loss) {
  __shared__ float red[kWaves];
  const int b = blockIdx.x;
  float acc = 0.0f;
  for (int k = threadIdx.x; k < P.K; k += kThreads)
    acc += (float)counts[(int64_t)b * P.K + k] * mean[(int64_t)b * P.K + k];
  acc = block_sum<kWaves>(acc, red);
  if (threadIdx.x == 0) {
    acc *= (float)P.K / (float)max(totals[4 * b + 1], 1);
    loss[b] = totals[4 * b + 2] ? __builtin_nanf("") : acc;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void balance_bwd_kernel(
    BalanceParams P, const T* __restrict__ logits,
    const int32_t* __restrict__ counts, const float2* __restrict__ stats,
    const int32_t* __restrict__ totals, const float* __restrict__ g_loss,
    const float* __restrict__ g_mean, T* __restrict__ g_logits) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (r >= P.rows * P.batch) return;
  const int b = (int)(r / P.rows);
  const T* row = logits + r * P.stride;
  T* out = g_logits + r * P.K;
  const float2 st = stats[r];
  const float per_row = 1.0f / (float)max(totals[4 * b], 1);
  const float per_count =
      g_loss ? g_loss[b] * ((float)P.K / (float)max(totals[4 * b + 1], 1)) : 0.0f;
  auto a_of = [&](int k) {
    const float f = per_count * (float)counts[(int64_t)b * P.K + k];
    return g_mean ? f + g_mean[(int64_t)b * P.K + k] : f;
  };
  float dot = 0.0f;
  for (int k = lane; k < P.K; k += 64) dot += prob(to_float(row[k]), st) * a_of(k);
  dot = wave_sum(dot);
  for (int k = lane; k < P.K; k += 64) {
    const float p = prob(to_float(row[k]), st);
    out[k] = static_cast<T>(p * (a_of(k) - dot) * per_row);
  }
}

int chunks_of(const BalanceParams& P) { return (int)((P.rows + kChunk - 1) / kChunk); }

template <typename T>
int forward_of(const BalanceParams& P, const void* logits, float* loss,
               int32_t* counts, float* mean, float2* stats, int32_t* totals,
               float* partials, hipStream_t stream) {
  const int64_t rows = P.rows * P.batch;
  const int chunks = chunks_of(P);
  const T* x = static_cast<const T*>(logits);
  int rc = launch_zero2(reinterpret_cast<uint32_t*>(counts), (int64_t)P.batch * P.K,
                        reinterpret_cast<uint32_t*>(totals), 4 * (int64_t)P.batch,
                        stream);
  if (rc) return rc;
  const unsigned cols = (unsigned)((P.K + kThreads - 1) / kThreads);
  if (rows > 0) {
    launch_traced("balance_rows_kernel", (balance_rows_kernel<T>),
                  dim3((unsigned)((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0,
                  stream, P, x, counts, stats, totals);
    rc = check_launch("balance_rows_kernel");
    if (rc) return rc;
    launch_traced("balance_columns_kernel", (balance_columns_kernel<T>),
                  dim3(cols, (unsigned)chunks, (unsigned)P.batch), dim3(kThreads), 0,
                  stream, P, x, stats, chunks, partials);
    rc = check_launch("balance_columns_kernel");
    if (rc) return rc;
  }
  launch_traced("balance_mean_kernel", balance_mean_kernel,
                dim3(cols, (unsigned)P.batch), dim3(kThreads), 0, stream, P,
                partials, chunks, totals, mean);
  rc = check_launch("balance_mean_kernel");
  if (rc) return rc;
  launch_traced("balance_loss_kernel", balance_loss_kernel, dim3((unsigned)P.batch),
                dim3(kThreads), 0, stream, P, mean, counts, totals, loss);
  return check_launch("balance_loss_kernel");
}

template <typename T>
int backward_of(const BalanceParams& P, const void* logits, const int32_t* counts,
                const float2* stats, const int32_t* totals, const float* g_loss,
                const float* g_mean, void* g_logits, hipStream_t stream) {
  const int64_t rows = P.rows * P.batch;
  launch_traced("balance_bwd_kernel", (balance_bwd_kernel<T>),
                dim3((unsigned)((rows + kWaves - 1) / kWaves)), dim3(kThreads), 0,
                stream, P, static_cast<const T*>(logits), counts, stats, totals,
                g_loss, g_mean, static_cast<T*>(g_logits));
  return check_launch("balance_bwd_kernel");
}

}  // namespace

size_t balance_workspace_bytes(const BalanceParams& P) {
  return align_up((size_t)P.batch * chunks_of(P) * P.K * 4, 256);
}

int launch_balance_forward(const BalanceParams& P, const void* logits,
                           float* loss, int32_t* counts, float* mean_probs,
                           float2* stats, int32_t* totals, void* workspace,
                           hipStream_t stream) {
  auto f = P.dtype == GSPLAT_F32    ? forward_of<float>
           : P.dtype == GSPLAT_BF16 ? forward_of<__bf16>
                                    : forward_of<_Float16>;
  return f(P, logits, loss, counts, mean_probs, stats, totals,
           static_cast<float*>(workspace), stream);
}

int launch_balance_backward(const BalanceParams& P, const void* logits,
                            const int32_t* counts, const float2* stats,
                            const int32_t* totals, const float* g_loss,
                            const float* g_mean, void* g_logits,
                            hipStream_t stream) {
  if (P.rows * P.batch == 0) return GSPLAT_OK;
  auto f = P.dtype == GSPLAT_F32    ? backward_of<float>
           : P.dtype == GSPLAT_BF16 ? backward_of<__bf16>
                                    : backward_of<_Float16>;
  return f(P, logits, counts, stats, totals, g_loss, g_mean, g_logits, stream);
}

}  // namespace gs
