// codes.h -- what the kernels of scenes in codes share (code_lookup.hip,
// code_probs.hip, code_balance.hip): element types, codes, wavefront sums.
#pragma once

#include "gs_internal.h"

#define GS_HD __device__ __forceinline__
#include "exponent.h"

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
  // Those of rows n on.
  Codes from(int64_t n) const {
    return Codes{p ? static_cast<const char*>(p) + n * (wide ? 8 : 4) : nullptr, wide};
  }
};

// A launch has fewer than 2^32 threads: rows go in as many launches as that
// takes, `most` rows each.  launch(first, rows) returns a status.
template <typename Launch>
int in_launches(int64_t rows, int64_t most, Launch launch) {
  for (int64_t first = 0; first < rows; first += most) {
    const int rc = launch(first, rows - first < most ? rows - first : most);
    if (rc) return rc;
  }
  return GSPLAT_OK;
}
constexpr int64_t kMostBlocks = (1 << 24) - 1;  // of 256 threads

// 2^t with denormal results kept (the hardware's base-2 exponential flushes
// them): gradients go down to the type's smallest values.
__device__ __forceinline__ float exp2_full(float t) { return exp2f(t); }
// The hardware's exponential and logarithm: results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float t) { return __builtin_amdgcn_exp2f(t); }
__device__ __forceinline__ float log2_fast(float t) { return __builtin_amdgcn_logf(t); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// The largest of three in one instruction (fmaxf first quiets each operand that
// might be a signalling NaN, an instruction apiece).  Not for an operand of a
// cross-lane move: the compiler does not see that an instruction wrote it.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// 16 bytes of elements, loaded and stored at any multiple of the element size
// (rows of logits start anywhere; the memory pipeline takes dwordx4 accesses
// at any address).
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);
template <typename T>
using vec_t = T __attribute__((ext_vector_type(16 / sizeof(T))));

template <typename T>
__device__ __forceinline__ vec_t<T> load_vec(const T* p) {
  vec_t<T> v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, vec_t<T> v) {
  __builtin_memcpy(p, &v, 16);
}

// For what nothing reads soon: it leaves the caches to what is read again.
template <typename T>
__device__ __forceinline__ void store_vec_stream(T* p, vec_t<T> v) {
  typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
  __builtin_nontemporal_store(__builtin_bit_cast(words, v), reinterpret_cast<words*>(p));
}

template <typename T>
__device__ __forceinline__ vec_t<T> load_vec_stream(const T* p) {
  typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
  return __builtin_bit_cast(vec_t<T>, __builtin_nontemporal_load(reinterpret_cast<const words*>(p)));
}

// Whether a forward reads its logits past the caches: those of over 1 GiB are
// four times the last cache, and nothing of them is left there for a backward
// (64K x 16384 in bf16, forward and then both: 478 and 1205 us without, 430 and
// 1182 with; below, the backward loses more than the forward gains: 268 MB, 69
// and 160 without, 59 and 167 with).
inline bool past_caches(int64_t rows, int K, int dtype) {
  return rows * K * (dtype == GSPLAT_F32 ? 4 : 2) > (int64_t(1) << 30);
}

// The same 16 bytes, of which the compiler no longer knows that it has them as
// floats already: two passes over a row in registers convert its elements twice
// rather than keep twice the registers.
template <typename T>
__device__ __forceinline__ void forget(vec_t<T>& v) {
  if constexpr (sizeof(T) == 2) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    words w = __builtin_bit_cast(words, v);
    asm volatile("" : "+v"(w));
    v = __builtin_bit_cast(vec_t<T>, w);
  }
}

// A vector's bytes.
struct Words {
  uint64_t lo, hi;
};

// Elements i .. i + kVec - 1 of a row of n, `fill` past its end.  Even: n is a
// multiple of kVec, and a vector is in the row or past it (otherwise the
// addresses of a last vector's single elements cost a kernel that loops over
// rows half as many registers again).
template <typename T, bool Even = false, bool Stream = false>
__device__ __forceinline__ vec_t<T> load_part(const T* row, int i, int n, T fill) {
  if (Even ? i < n : i + kVec<T> <= n) return Stream ? load_vec_stream(row + i) : load_vec(row + i);
  vec_t<T> v;
#pragma unroll
  for (int j = 0; j < kVec<T>; ++j) v[j] = !Even && i + j < n ? row[i + j] : fill;
  return v;
}
template <typename T, bool Even = false, bool Stream = false>
__device__ __forceinline__ void store_part(T* row, int i, int n, vec_t<T> v) {
  if (Even ? i < n : i + kVec<T> <= n) {
    if (Stream) store_vec_stream(row + i, v);
    else store_vec(row + i, v);
    return;
  }
  if (Even || i >= n) return;
  // a last vector's elements by the binary digits of their number
  const int m = n - i;
  const Words w = __builtin_bit_cast(Words, v);
  T* to = row + i;
  uint64_t u = w.lo;
  if (m * sizeof(T) & 8) {
    __builtin_memcpy(to, &u, 8);
    to += 8 / sizeof(T);
    u = w.hi;
  }
  if (m * sizeof(T) & 4) {
    const uint32_t low = (uint32_t)u;
    __builtin_memcpy(to, &low, 4);
    to += 4 / sizeof(T);
    u >>= 32;
  }
  if (sizeof(T) == 2 && (m & 1)) {
    const uint16_t low = (uint16_t)u;
    __builtin_memcpy(to, &low, 2);
  }
}

// A thread's R vectors of a row of n: those at first, first + step, ...  Where
// rows are not whole vectors (and not shorter than one), a last vector is read as
// the row's last kVec elements, one load like the others, and fix_row brings
// them to their place once they are there.  (1M rows of 101 in bf16, the
// balance's backward: element by element 157 us, so 118.)
template <typename T, int R, bool Even, bool Stream>
__device__ __forceinline__ void load_row(vec_t<T> (&x)[R], const T* row, int first, int step, int n, T fill) {
  constexpr int V = kVec<T>;
  if (Even || n < V) {
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = load_part<T, Even, Stream>(row, first + r * step, n, fill);
    return;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = first + r * step;
    if (i < n) {
      const T* from = row + min(i, n - V);
      x[r] = Stream ? load_vec_stream(from) : load_vec(from);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) x[r][v] = fill;
    }
  }
}
template <typename T, int R, bool Even>
__device__ __forceinline__ void fix_row(vec_t<T> (&x)[R], int first, int step, int n, T fill) {
  constexpr int V = kVec<T>;
  if (Even || n < V) return;
  vec_t<T> fills;
#pragma unroll
  for (int v = 0; v < V; ++v) fills[v] = fill;
  const uint64_t more = __builtin_bit_cast(Words, fills).lo;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = first + r * step, past = i + V - n;  // elements to leave out
    if (past <= 0 || past >= V) continue;
    Words w = __builtin_bit_cast(Words, x[r]);
    int bits = past * (int)sizeof(T) * 8;
    if (bits >= 64) {
      w.lo = w.hi;
      w.hi = more;
      bits -= 64;
    }
    w.lo = (w.lo >> bits) | (w.hi << 1) << (63 - bits);
    w.hi = (w.hi >> bits) | (more << 1) << (63 - bits);
    x[r] = __builtin_bit_cast(vec_t<T>, w);
  }
}

// Reductions over teams of L consecutive lanes (a power of two up to the
// wavefront); every lane gets the result, the same bits in each.  Partners: in
// the quad by quad_perm, in eight and sixteen lanes by the mirrors (the lanes
// of a quad are equal by then), across 16 and 32 lanes by the row swaps.
template <int Ctrl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, Ctrl, 0xf, 0xf, true);
}
template <int L, typename Op>
__device__ __forceinline__ uint32_t team_reduce(uint32_t v, Op op) {
  if constexpr (L >= 2) v = op(v, dpp<0xB1>(v));   // quad_perm 1,0,3,2
  if constexpr (L >= 4) v = op(v, dpp<0x4E>(v));   // quad_perm 2,3,0,1
  if constexpr (L >= 8) v = op(v, dpp<0x141>(v));  // row_half_mirror
  if constexpr (L >= 16) v = op(v, dpp<0x140>(v)); // row_mirror
  if constexpr (L >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  if constexpr (L >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  return v;
}
// (As integers that keep the floats' order: one instruction a step.  A NaN is
// above everything or, negative, below.)
template <int L>
__device__ __forceinline__ float team_max(float v) {
  const uint32_t u = __float_as_uint(v);
  const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  const uint32_t r = team_reduce<L>(k, [](uint32_t a, uint32_t b) { return max(a, b); });
  return __uint_as_float(r ^ (~(uint32_t)((int32_t)r >> 31) | 0x80000000u));
}
template <int L>
__device__ __forceinline__ float team_sum(float v) {
  return __uint_as_float(team_reduce<L>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int L>
__device__ __forceinline__ uint32_t team_min(uint32_t v) {
  return team_reduce<L>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
template <int L>
__device__ __forceinline__ uint32_t team_umax(uint32_t v) {
  return team_reduce<L>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}

__device__ __forceinline__ int wave_isum(int v) {
  return (int)team_reduce<64>((uint32_t)v, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ float wave_sum(float v) { return team_sum<64>(v); }
__device__ __forceinline__ float wave_max(float v) { return team_max<64>(v); }

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
