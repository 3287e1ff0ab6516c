// codes.h -- what the kernels of scenes in codes share (code_lookup.hip,
// code_probs.hip, code_balance.hip): element types, codes, wavefront sums.
#pragma once

#include "gs_internal.h"

namespace gs {

// Codebooks and logits are float, __bf16 or _Float16 (GSPLAT_F32 / _BF16 /
// _F16).  Sums and statistics are 32-bit floats; results are rounded to the
// element type once, on the way out.
template <typename T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }

// A splat's code: 0..K-1, kNoCode for -1 (the splat has none), kBadCode for
// any other value (nothing is read or counted for it; outputs become NaN).
constexpr int kNoCode = -1;
constexpr int kBadCode = -2;

struct Codes {
  const void* p;
  int wide;  // 64-bit codes, else 32-bit
  __device__ __forceinline__ int at(int64_t i, int K) const {
    const int64_t c = wide ? static_cast<const int64_t*>(p)[i]
                           : static_cast<const int32_t*>(p)[i];
    if (c >= 0 && c < K) return (int)c;
    return c == -1 ? kNoCode : kBadCode;
  }
};

// e^z with denormal results kept (the hardware's base-2 exponential flushes
// them): probabilities of gradients go down to the type's smallest values.
__device__ __forceinline__ float exp_full(float z) {
  return exp2f(z * 1.44269504088896340736f);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}

// The same over a workgroup of W wavefronts (red: W floats of LDS; every
// thread gets the result).
template <int W>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int w = 1; w < W; ++w) r += red[w];
  return r;
}

template <int W>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int w = 1; w < W; ++w) r = fmaxf(r, red[w]);
  return r;
}

// ---- code_lookup.hip
struct LookupParams {
  int64_t rows;    // splats
  int K, D;        // codes, values per code
  int64_t stride;  // elements between codebook rows
  int dtype;
  float factor;
  Codes codes;
};
size_t lookup_backward_workspace_bytes(const LookupParams& P);
int launch_lookup_forward(const LookupParams& P, const void* codebook,
                          const float* scales, void* out, hipStream_t stream);
int launch_lookup_backward(const LookupParams& P, const void* grad_out,
                           const void* codebook, const float* scales,
                           void* g_codebook, float* g_scales, void* workspace,
                           hipStream_t stream);

// ---- code_probs.hip
struct ProbsParams {
  int64_t rows;
  int K, top;
  int64_t stride;  // elements between rows of logits
  int dtype;
  float inv_t;     // 1 / temperature
  Codes codes;     // p null: none given
};
size_t probs_workspace_bytes(const ProbsParams& P);
int launch_probs_forward(const ProbsParams& P, const void* logits,
                         float* log_probs, float* entropy, float* top_log_probs,
                         int32_t* top_codes, float2* stats, void* workspace,
                         hipStream_t stream);
int launch_probs_backward(const ProbsParams& P, const void* logits,
                          const int32_t* top_codes, const float2* stats,
                          const float* entropy, const float* g_log_probs,
                          const float* g_entropy, const float* g_top,
                          void* g_logits, hipStream_t stream);

// ---- code_balance.hip
struct BalanceParams {
  int batch;
  int64_t rows;  // per image
  int K, choices;
  int64_t stride;
  int dtype;
  Codes codes;   // [batch][rows][choices]
};
size_t balance_workspace_bytes(const BalanceParams& P);
int launch_balance_forward(const BalanceParams& P, const void* logits,
                           float* loss, int32_t* counts, float* mean_probs,
                           float2* stats, int32_t* totals, void* workspace,
                           hipStream_t stream);
int launch_balance_backward(const BalanceParams& P, const void* logits,
                            const int32_t* counts, const float2* stats,
                            const int32_t* totals, const float* g_loss,
                            const float* g_mean, void* g_logits,
                            hipStream_t stream);

}  // namespace gs
