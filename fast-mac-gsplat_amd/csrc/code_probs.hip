// code_probs.hip -- log probabilities of codes under logits x over K codes.
//
//   z = (x - max x) / T,  S = sum e^z,  log p = z - log S,  p = e^z / S
//   H = log S - (sum e^z z) / S                               (entropy)
//   dL/dx = (1/T) [ gl (delta_code - p) + sum_j gt_j (delta_tj - p)
//                   - gH p (log p + H) ]
//
// with gl, gH and gt the gradients of the code's log probability, of the
// entropy and of the alternatives' log probabilities.  A row with no logit
// above -inf has S = 0: log p = -inf, H = 0, and no gradient.  A NaN makes its
// row NaN.  The alternatives are ranked by the logits themselves (NaN first,
// -0 equal to +0, the lower index first among equal ones).
//
// A row's statistics (max x, log S) are kept for the backward, which is one
// pass over the logits: log S = -inf marks a row without probabilities.
#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Rank of a logit at column i: the larger logit, then the lower column.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t i) {
  return ((uint64_t)depth_key(x) << 32) | (uint32_t)~i;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void probs_fwd_kernel(
    ProbsParams P, const T* __restrict__ logits, float* __restrict__ log_probs,
    float* __restrict__ entropy, float* __restrict__ top_log_probs,
    int32_t* __restrict__ top_codes, float2* __restrict__ stats) {
  __shared__ float red[kWaves];
  __shared__ uint64_t best[kWaves];
  const int64_t n = blockIdx.x;
  const T* row = logits + n * P.stride;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < P.K; i += kThreads) m = fmaxf(m, to_float(row[i]));
  m = block_max<kWaves>(m, red);
  const float base = m == -INFINITY ? 0.0f : m;
  float s = 0.0f, sz = 0.0f;
  for (int i = threadIdx.x; i < P.K; i += kThreads) {
    const float z = (to_float(row[i]) - base) * P.inv_t;
    const float e = __expf(z);
    s += e;
    sz += e > 0.0f ? e * z : 0.0f;
  }
  s = block_sum<kWaves>(s, red);
  sz = block_sum<kWaves>(sz, red);
  const float log_s = __logf(s);
  auto log_prob = [&](float x) { return (x - base) * P.inv_t - (s == 0.0f ? 0.0f : log_s); };
  if (threadIdx.x == 0) {
    if (log_probs) {
      const int c = P.codes.at(n, P.K);
      log_probs[n] = c >= 0 ? log_prob(to_float(row[c]))
                            : (c == kNoCode ? 0.0f : __builtin_nanf(""));
    }
    entropy[n] = s == 0.0f ? 0.0f : log_s - sz / s;
    if (stats) stats[n] = make_float2(base, s == 0.0f ? -INFINITY : log_s);
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < P.top; ++j) {
    uint64_t k = 0;
    for (int i = threadIdx.x; i < P.K; i += kThreads) {
      const uint64_t r = rank_key(to_float(row[i]), i);
      if (r < last && r > k) k = r;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) k = max(k, (uint64_t)__shfl_xor(k, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = k;
    __syncthreads();
    k = best[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) k = max(k, best[w]);
    last = k;
    if (threadIdx.x == 0) {
      const int i = (int)~(uint32_t)k;
      top_codes[n * P.top + j] = i;
      top_log_probs[n * P.top + j] = log_prob(to_float(row[i]));
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void probs_bwd_kernel(
    ProbsParams P, const T* __restrict__ logits,
    const int32_t* __restrict__ top_codes, const float2* __restrict__ stats,
    const float* __restrict__ entropy, const float* __restrict__ g_log_probs,
    const float* __restrict__ g_entropy, const float* __restrict__ g_top,
    T* __restrict__ g_logits) {
  const int64_t n = blockIdx.x;
  const T* row = logits + n * P.stride;
  T* out = g_logits + n * P.K;
  const float2 st = stats[n];
  const bool some = st.y != -INFINITY;
  const float H = entropy[n];
  const float ge = g_entropy ? g_entropy[n] : 0.0f;
  int code = kNoCode;
  float gl = 0.0f;
  if (g_log_probs) {
    code = P.codes.at(n, P.K);
    if (code >= 0) gl = g_log_probs[n];
  }
  float total = gl;
  const float* gt = g_top ? g_top + n * P.top : nullptr;
  const int32_t* tc = top_codes + n * P.top;
  if (gt)
    for (int j = 0; j < P.top; ++j) total += gt[j];
  for (int i = threadIdx.x; i < P.K; i += kThreads) {
    float g = 0.0f;
    if (some) {
      const float lp = (to_float(row[i]) - st.x) * P.inv_t - st.y;
      const float p = exp_full(lp);
      g = -p * total - (p > 0.0f ? ge * p * (lp + H) : 0.0f);
      if (p != p) g = p;
      if (i == code) g += gl;
      if (gt)
        for (int j = 0; j < P.top; ++j)
          if (i == tc[j]) g += gt[j];
    }
    out[i] = static_cast<T>(g * P.inv_t);
  }
}

template <typename T>
int forward_of(const ProbsParams& P, const void* logits, float* log_probs,
               float* entropy, float* top_log_probs, int32_t* top_codes,
               float2* stats, hipStream_t stream) {
  launch_traced("probs_fwd_kernel", (probs_fwd_kernel<T>), dim3((unsigned)P.rows),
                dim3(kThreads), 0, stream, P, static_cast<const T*>(logits),
                log_probs, entropy, top_log_probs, top_codes, stats);
  return check_launch("probs_fwd_kernel");
}

template <typename T>
int backward_of(const ProbsParams& P, const void* logits, const int32_t* top_codes,
                const float2* stats, const float* entropy,
                const float* g_log_probs, const float* g_entropy,
                const float* g_top, void* g_logits, hipStream_t stream) {
  launch_traced("probs_bwd_kernel", (probs_bwd_kernel<T>), dim3((unsigned)P.rows),
                dim3(kThreads), 0, stream, P, static_cast<const T*>(logits),
                top_codes, stats, entropy, g_log_probs, g_entropy, g_top,
                static_cast<T*>(g_logits));
  return check_launch("probs_bwd_kernel");
}

}  // namespace

size_t probs_workspace_bytes(const ProbsParams&) { return 0; }

int launch_probs_forward(const ProbsParams& P, const void* logits,
                         float* log_probs, float* entropy, float* top_log_probs,
                         int32_t* top_codes, float2* stats, void*,
                         hipStream_t stream) {
  if (P.rows == 0) return GSPLAT_OK;
  auto f = P.dtype == GSPLAT_F32    ? forward_of<float>
           : P.dtype == GSPLAT_BF16 ? forward_of<__bf16>
                                    : forward_of<_Float16>;
  return f(P, logits, log_probs, entropy, top_log_probs, top_codes, stats, stream);
}

int launch_probs_backward(const ProbsParams& P, const void* logits,
                          const int32_t* top_codes, const float2* stats,
                          const float* entropy, const float* g_log_probs,
                          const float* g_entropy, const float* g_top,
                          void* g_logits, hipStream_t stream) {
  if (P.rows == 0) return GSPLAT_OK;
  auto f = P.dtype == GSPLAT_F32    ? backward_of<float>
           : P.dtype == GSPLAT_BF16 ? backward_of<__bf16>
                                    : backward_of<_Float16>;
  return f(P, logits, top_codes, stats, entropy, g_log_probs, g_entropy, g_top,
           g_logits, stream);
}

}  // namespace gs
