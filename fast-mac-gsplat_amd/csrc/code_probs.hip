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
#include <algorithm>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Statistics of a part of a row, exponents in base 2: m = its largest logit
// (-inf: none), s = sum 2^t and st = sum 2^t t with t = (x - m) c, c = log2(e) / T.
struct Part {
  float m, s, st;
};

// An exponent for a product with its power: -inf (a power of 0) would make it NaN.
__device__ __forceinline__ float bounded(float t) { return fmaxf(t, -1000.0f); }

__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

// The statistics of a's and b's parts as one (a NaN in either s stays).
__device__ __forceinline__ Part joined(Part a, Part b, float c) {
  Part r;
  r.m = fmaxf(a.m, b.m);
  const float base = base_of(r.m);
  const float da = bounded((a.m - base) * c), db = bounded((b.m - base) * c);
  const float fa = exp2_fast(da), fb = exp2_fast(db);
  r.s = a.s * fa + b.s * fb;
  r.st = fa * (a.st + da * a.s) + fb * (b.st + db * b.s);
  return r;
}

// Rank of a logit at column i: the larger logit, then the lower column.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t i) {
  return ((uint64_t)depth_key(x) << 32) | (uint32_t)~i;
}

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// The largest key of a team of L lanes.
template <int L>
__device__ __forceinline__ uint64_t team_best(uint64_t k) {
  const uint32_t hi = team_umax<L>((uint32_t)(k >> 32));
  const uint32_t lo = team_umax<L>((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return ((uint64_t)hi << 32) | lo;
}

struct ProbsOut {
  float* log_probs;
  float* entropy;
  float* top_log_probs;
  int32_t* top_codes;
  float2* stats;
};

// What a row's statistics say about one of its logits.
struct RowEnd {
  float base, log2_s, inv_t;
  __device__ __forceinline__ RowEnd(Part p, float inv_t_)
      : base(base_of(p.m)), log2_s(p.s == 0.0f ? 0.0f : log2_fast(p.s)), inv_t(inv_t_) {}
  // (not in base 2: a masked logit of the type's lowest value would overflow)
  __device__ __forceinline__ float log_prob(float x) const {
    return __builtin_fmaf(-kLn2, log2_s, (x - base) * inv_t);
  }
};

// Written by one lane per row.  code_logit: the logit of the row's code.
__device__ __forceinline__ void write_row(const ProbsOut& out, int64_t n, Part p, RowEnd e,
                                          int code, float code_logit) {
  if (out.log_probs)
    out.log_probs[n] = code >= 0 ? e.log_prob(code_logit)
                                 : (code == kNoCode ? 0.0f : __builtin_nanf(""));
  const bool some = p.s != 0.0f;
  out.entropy[n] = some ? (e.log2_s - p.st / p.s) * kLn2 : 0.0f;
  if (out.stats) out.stats[n] = make_float2(e.base, some ? e.log2_s : INFINITY);
}

// The elements that a thread of a team of TL holds: vectors r = 0..R-1 of the
// team's rows of TL vectors.
template <typename T, int TL, int R>
struct Held {
  static constexpr int V = kVec<T>;
  vec_t<T> x[R];
  int lane;
  __device__ __forceinline__ void load(const T* row, int lane_, int n) {
    lane = lane_;
#pragma unroll
    for (int r = 0; r < R; ++r)
      x[r] = load_part<T>(row, (r * TL + lane) * V, n, static_cast<T>(-INFINITY));
  }
  __device__ __forceinline__ int column(int r, int v) const { return (r * TL + lane) * V + v; }
  __device__ __forceinline__ float max() const {
    float m = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) m = fmaxf(m, to_float(x[r][v]));
    return m;
  }
  // s and st of this thread's elements for the maximum m.
  __device__ __forceinline__ Part part(float m, float c) const {
    Part p{m, 0.0f, 0.0f};
    const float base = base_of(m);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float t = (to_float(x[r][v]) - base) * c;
        const float e = exp2_fast(t);
        p.s += e;
        p.st = __builtin_fmaf(e, bounded(t), p.st);
      }
    return p;
  }
  // The largest key below `last` among this thread's elements.
  __device__ __forceinline__ uint64_t best_below(uint64_t last) const {
    uint64_t k = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const uint64_t q = rank_key(to_float(x[r][v]), column(r, v));
        if (q < last) k = max64(k, q);
      }
    return k;
  }
  // The lowest column whose logit equals m.
  __device__ __forceinline__ uint32_t first_equal(float m) const {
    uint32_t i = ~0u;
#pragma unroll
    for (int r = R - 1; r >= 0; --r)
#pragma unroll
      for (int v = V - 1; v >= 0; --v)
        if (to_float(x[r][v]) == m) i = column(r, v);
    return i;
  }
};

// ---- rows of at most TL * kVec * R codes: a team of TL lanes per row

template <typename T, int TL, int R>
__global__ __launch_bounds__(kThreads) void probs_rows_kernel(
    ProbsParams P, const T* __restrict__ logits, ProbsOut out) {
  constexpr int kTeams = kThreads / TL;
  __shared__ uint64_t found[TL == 64 ? kWaves * 64 : 1];
  const int lane = threadIdx.x & (TL - 1);
  int64_t n = (int64_t)blockIdx.x * kTeams + threadIdx.x / TL;
  const bool active = n < P.rows;
  if (!active) n = P.rows - 1;  // (its lanes go along)
  const T* row = logits + n * P.stride;
  int code = kNoCode;
  float code_logit = 0.0f;
  if (P.codes.p) {
    code = P.codes.at(n, P.K);
    if (code >= 0) code_logit = to_float(row[code]);
  }
  Held<T, TL, R> x;
  x.load(row, lane, P.K);
  const float mine = x.max();
  const float c = P.inv_t * kLog2e;
  Part p = x.part(team_max<TL>(mine), c);
  p.s = team_sum<TL>(p.s);
  p.st = team_sum<TL>(p.st);
  const RowEnd e(p, P.inv_t);
  if (lane == 0 && active) write_row(out, n, p, e, code, code_logit);
  const int top = P.top;
  if (top == 0) return;
  auto put = [&](int j, uint32_t i, float v) {
    if (active) {
      out.top_codes[n * top + j] = (int)i;
      out.top_log_probs[n * top + j] = e.log_prob(v);
    }
  };
  int from = 0;
  const bool plain = p.s == p.s;  // (no NaN)
  if (plain) {
    // the best: the first column that has the maximum
    const uint32_t i = team_min<TL>(x.first_equal(p.m));
    if (lane == 0) put(0, i, p.m);
    from = 1;
  }
  if (from == top && __all(plain)) return;
  if constexpr (TL == 64) {
    // The top-th largest of the lanes' maxima is a lower bound of the top-th
    // largest logit: the logits from there up are few (ties aside), are
    // collected, and find their places by counting.
    if (plain && top > 1) {
      float rest = mine, bound = p.m;
      for (int j = 0; j < top; ++j) {
        bound = team_max<64>(rest);
        const uint64_t at = __ballot(rest == bound);
        if (lane == __builtin_ctzll(at)) rest = -INFINITY;
      }
      if (bound > -INFINITY) {
        uint64_t* list = found + (threadIdx.x & ~63);
        int total = 0;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int v = 0; v < kVec<T>; ++v) {
            const float f = to_float(x.x[r][v]);
            const uint64_t hit = __ballot(f >= bound);
            if (hit == 0) continue;
            const int at = total + __builtin_amdgcn_mbcnt_hi(
                                       (uint32_t)(hit >> 32),
                                       __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0));
            if (f >= bound && at < 64) list[at] = rank_key(f, x.column(r, v));
            total += __popcll(hit);
          }
        if (total <= 64) {
          __builtin_amdgcn_wave_barrier();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          const uint64_t k = lane < total ? list[lane] : 0;
          int place = 0;
          for (int j = 0; j < total; ++j) place += list[j] > k;
          if (lane < total && place < top) {
            const uint32_t i = ~(uint32_t)k;
            put(place, i, to_float(row[i]));
          }
          return;
        }
      }
    }
  }
  uint64_t last = ~0ull;
  if (plain) last = rank_key(p.m, team_min<TL>(x.first_equal(p.m)));
  for (int j = from; j < top; ++j) {
    last = team_best<TL>(x.best_below(last));
    const uint32_t i = ~(uint32_t)last;
    if (lane == 0) put(j, i, to_float(row[i]));
  }
}

// ---- longer rows: a workgroup per part of a row

// One part of a row per workgroup.  parts = 1: the row's outputs; else its
// statistics and best keys go to partials, for probs_join_kernel.
struct Split {
  int parts;    // per row
  int length;   // elements of a part (the last may be shorter)
  Part* stats;  // [rows][parts]
  uint64_t* best;  // [rows][parts][top]
};

constexpr int kFound = 256;  // logits collected for the best ones

template <typename T, int R>
__global__ __launch_bounds__(kThreads) void probs_parts_kernel(
    ProbsParams P, const T* __restrict__ logits, ProbsOut out, Split split) {
  __shared__ Part parts[kWaves];
  __shared__ float bounds[kWaves];
  __shared__ uint64_t found[kFound];
  __shared__ uint64_t best[kWaves];
  __shared__ int total;
  const int64_t n = blockIdx.x / (unsigned)split.parts;
  const int part = (int)(blockIdx.x - (uint32_t)n * (unsigned)split.parts);
  const int first = part * split.length;
  const int len = min(split.length, P.K - first);
  const T* row = logits + n * P.stride;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int code = kNoCode;
  float code_logit = 0.0f;
  if (P.codes.p && split.parts == 1) {
    code = P.codes.at(n, P.K);
    if (code >= 0) code_logit = to_float(row[code]);
  }
  Held<T, kThreads, R> x;
  x.load(row + first, threadIdx.x, len);
  const float mine = x.max();
  const float c = P.inv_t * kLog2e;
  Part p = x.part(wave_max(mine), c);
  p.s = wave_sum(p.s);
  p.st = wave_sum(p.st);
  const int top = min(P.top, len);
  float bound = p.m;
  if (top > 1) {
    float rest = mine;
    for (int j = 0; j < top; ++j) {
      bound = wave_max(rest);
      const uint64_t at = __ballot(rest == bound);
      if (lane == __builtin_ctzll(at)) rest = -INFINITY;
    }
  }
  if (lane == 0) {
    parts[w] = p;
    bounds[w] = bound;
  }
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  p = parts[0];
  bound = bounds[0];
#pragma unroll
  for (int j = 1; j < kWaves; ++j) {
    p = joined(p, parts[j], c);
    bound = fmaxf(bound, bounds[j]);
  }
  const RowEnd e(p, P.inv_t);
  if (threadIdx.x == 0) {
    if (split.parts == 1)
      write_row(out, n, p, e, code, code_logit);
    else
      split.stats[(int64_t)blockIdx.x] = p;
  }
  if (P.top == 0) return;
  auto put = [&](int j, uint64_t key) {
    if (split.parts == 1) {
      const uint32_t i = ~(uint32_t)key;
      out.top_codes[n * P.top + j] = (int)i;
      out.top_log_probs[n * P.top + j] = e.log_prob(to_float(row[i]));
    } else {
      // (columns of the whole row; 0 where the part has fewer than top)
      split.best[(int64_t)blockIdx.x * P.top + j] = key == 0 ? 0 : key - (uint32_t)first;
    }
  };
  for (int j = top + threadIdx.x; j < P.top; j += kThreads) put(j, 0);
  if (p.s == p.s && bound > -INFINITY) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < kVec<T>; ++v) {
        const float f = to_float(x.x[r][v]);
        if (f >= bound) {
          const int at = atomicAdd(&total, 1);
          if (at < kFound) found[at] = rank_key(f, x.column(r, v));
        }
      }
    __syncthreads();
    const int m = total;
    if (m <= kFound) {
      // (the list's order depends on the run, the places do not)
      if ((int)threadIdx.x < m) {
        const uint64_t k = found[threadIdx.x];
        int place = 0;
        for (int j = 0; j < m; ++j) place += found[j] > k;
        if (place < top) put(place, k);
      }
      return;
    }
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < top; ++j) {
    uint64_t k = team_best<64>(x.best_below(last));
    __syncthreads();
    if (lane == 0) best[w] = k;
    __syncthreads();
    k = best[0];
#pragma unroll
    for (int q = 1; q < kWaves; ++q) k = max64(k, best[q]);
    last = k;
    if (threadIdx.x == 0) put(j, k);
  }
}

// A wavefront per row joins the row's parts.
template <typename T>
__global__ __launch_bounds__(64) void probs_join_kernel(
    ProbsParams P, const T* __restrict__ logits, ProbsOut out, Split split) {
  const int64_t n = blockIdx.x;
  const int lane = threadIdx.x;
  const T* row = logits + n * P.stride;
  const float c = P.inv_t * kLog2e;
  Part p{-INFINITY, 0.0f, 0.0f};
  for (int j = lane; j < split.parts; j += 64) p = joined(p, split.stats[n * split.parts + j], c);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const Part q{__shfl_xor(p.m, d, 64), __shfl_xor(p.s, d, 64), __shfl_xor(p.st, d, 64)};
    p = joined(p, q, c);
  }
  const RowEnd e(p, P.inv_t);
  if (lane == 0) {
    int code = kNoCode;
    float code_logit = 0.0f;
    if (P.codes.p) {
      code = P.codes.at(n, P.K);
      if (code >= 0) code_logit = to_float(row[code]);
    }
    write_row(out, n, p, e, code, code_logit);
  }
  const uint64_t* keys = split.best + n * split.parts * P.top;
  uint64_t last = ~0ull;
  for (int j = 0; j < P.top; ++j) {
    uint64_t k = 0;
    for (int i = lane; i < split.parts * P.top; i += 64)
      if (keys[i] < last) k = max64(k, keys[i]);
    last = team_best<64>(k);
    if (lane == 0) {
      const uint32_t i = ~(uint32_t)last;
      out.top_codes[n * P.top + j] = (int)i;
      out.top_log_probs[n * P.top + j] = e.log_prob(to_float(row[i]));
    }
  }
}

// ---- backward

// dL/dx = -p (total + gH (log p + H)) + gl at the code + gt at the
// alternatives, over T: per element a fused multiply-add, a base-2 exponential
// and two products.  A team of TL lanes per part of a row of TL * kVec * R
// columns (`parts` of them per row).
template <typename T, int TL, int R>
__global__ __launch_bounds__(kThreads) void probs_bwd_kernel(
    ProbsParams P, const T* __restrict__ logits,
    const int32_t* __restrict__ top_codes, const float2* __restrict__ stats,
    const float* __restrict__ entropy, const float* __restrict__ g_log_probs,
    const float* __restrict__ g_entropy, const float* __restrict__ g_top,
    T* __restrict__ g_logits, int parts) {
  constexpr int kTeams = kThreads / TL, V = kVec<T>;
  const int lane = threadIdx.x & (TL - 1);
  const int64_t i = (int64_t)blockIdx.x * kTeams + threadIdx.x / TL;
  if (i >= P.rows * parts) return;
  const int64_t n = i / parts;
  const int first = (int)(i - n * parts) * (TL * V * R);
  const T* row = logits + n * P.stride;
  T* out = g_logits + n * P.K;
  vec_t<T> x[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    x[r] = load_part<T>(row, first + (r * TL + lane) * V, P.K, static_cast<T>(-INFINITY));
  const float2 st = stats[n];
  const bool some = st.y != INFINITY;  // (else p = 0 everywhere)
  const float ge = g_entropy && some ? g_entropy[n] : 0.0f;
  int code = kNoCode;
  float gl = 0.0f;
  if (g_log_probs && some) {
    code = P.codes.at(n, P.K);
    if (code >= 0) gl = g_log_probs[n];
  }
  float total = gl;
  const int top = g_top && some ? P.top : 0;
  const float* gt = g_top + n * P.top;
  const int32_t* tc = top_codes + n * P.top;
  for (int j = 0; j < top; ++j) total += gt[j];
  const float c = P.inv_t * kLog2e;
  const float per_t = ge * kLn2, fixed = total + ge * entropy[n];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int at = first + (r * TL + lane) * V;
    float g[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float t = (to_float(x[r][v]) - st.x) * c - st.y;
      g[v] = -exp2_full(t) * __builtin_fmaf(per_t, bounded(t), fixed);
    }
    auto add = [&](int col, float w) {
#pragma unroll
      for (int v = 0; v < V; ++v) g[v] += col == at + v ? w : 0.0f;
    };
    if ((unsigned)(code - at) < (unsigned)V) add(code, gl);
    for (int j = 0; j < top; ++j) {
      const int col = tc[j];
      if ((unsigned)(col - at) < (unsigned)V) add(col, gt[j]);
    }
    vec_t<T> o;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = static_cast<T>(g[v] * P.inv_t);
    store_part<T>(out, at, P.K, o);
  }
}

// Rows of at most this many codes are one team's; longer ones are cut.
template <typename T>
constexpr int kPartLong = kThreads * kVec<T> * (sizeof(T) == 4 ? 16 : 8);

Split split_of(const ProbsParams& P, int longest) {
  Split s{1, P.K, nullptr, nullptr};
  if (P.K <= longest) return s;
  // Few rows: shorter parts, until there is one for each of 512 workgroups.
  int64_t length = longest;
  while (length > 2048 && P.rows * ((P.K + length - 1) / length) < 512) length /= 2;
  s.length = (int)length;
  s.parts = (int)((P.K + length - 1) / length);
  return s;
}

int longest_of(const ProbsParams& P) {
  return P.dtype == GSPLAT_F32 ? kPartLong<float> : kPartLong<__bf16>;
}

template <typename T>
int forward_of(const ProbsParams& P, const void* logits, const ProbsOut& out,
               void* workspace, hipStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  constexpr int V = kVec<T>;
  const int vecs = (P.K + V - 1) / V;
#define GS_ROWS(TL, R)                                                           \
  if (vecs <= TL * R) {                                                          \
    launch_traced("probs_rows_kernel", (probs_rows_kernel<T, TL, R>),            \
                  dim3((unsigned)((P.rows + kThreads / TL - 1) / (kThreads / TL))), \
                  dim3(kThreads), 0, stream, P, x, out);                         \
    return check_launch("probs_rows_kernel");                                    \
  }
  GS_ROWS(2, 1) GS_ROWS(4, 1) GS_ROWS(8, 1) GS_ROWS(16, 1) GS_ROWS(32, 1)
  GS_ROWS(64, 1) GS_ROWS(64, 2) GS_ROWS(64, 4)
#undef GS_ROWS
  Split s = split_of(P, kPartLong<T>);
  if (s.parts > 1) {
    s.stats = static_cast<Part*>(workspace);
    s.best = reinterpret_cast<uint64_t*>(
        static_cast<char*>(workspace) +
        align_up((size_t)P.rows * s.parts * sizeof(Part), 256));
  }
  const dim3 grid((unsigned)(P.rows * s.parts));
  const int len = (s.length + V - 1) / V;
#define GS_PARTS(R)                                                            \
  launch_traced("probs_parts_kernel", (probs_parts_kernel<T, R>), grid,        \
                dim3(kThreads), 0, stream, P, x, out, s)
  if (len <= 2 * kThreads) GS_PARTS(2);
  else if (len <= 4 * kThreads) GS_PARTS(4);
  else if (len <= 8 * kThreads) GS_PARTS(8);
  else if constexpr (sizeof(T) == 4) GS_PARTS(16);
#undef GS_PARTS
  const int rc = check_launch("probs_parts_kernel");
  if (rc || s.parts == 1) return rc;
  launch_traced("probs_join_kernel", (probs_join_kernel<T>), dim3((unsigned)P.rows),
                dim3(64), 0, stream, P, x, out, s);
  return check_launch("probs_join_kernel");
}

template <typename T>
int backward_of(const ProbsParams& P, const void* logits, const int32_t* top_codes,
                const float2* stats, const float* entropy,
                const float* g_log_probs, const float* g_entropy,
                const float* g_top, void* g_logits, hipStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  T* g = static_cast<T*>(g_logits);
  const int vecs = (P.K + kVec<T> - 1) / kVec<T>;
#define GS_BWD(TL, R)                                                          \
  {                                                                            \
    const int parts = (vecs + TL * R - 1) / (TL * R);                          \
    const int64_t teams = P.rows * parts, per = kThreads / TL;                 \
    launch_traced("probs_bwd_kernel", (probs_bwd_kernel<T, TL, R>),            \
                  dim3((unsigned)((teams + per - 1) / per)), dim3(kThreads), 0, \
                  stream, P, x, top_codes, stats, entropy, g_log_probs,        \
                  g_entropy, g_top, g, parts);                                 \
    return check_launch("probs_bwd_kernel");                                   \
  }
  if (vecs <= 2) GS_BWD(2, 1)
  if (vecs <= 4) GS_BWD(4, 1)
  if (vecs <= 8) GS_BWD(8, 1)
  if (vecs <= 16) GS_BWD(16, 1)
  if (vecs <= 32) GS_BWD(32, 1)
  if (vecs <= 64) GS_BWD(64, 1)
  if (vecs <= 128) GS_BWD(64, 2)
  GS_BWD(64, 4)
#undef GS_BWD
}

}  // namespace

size_t probs_workspace_bytes(const ProbsParams& P) {
  const Split s = split_of(P, longest_of(P));
  if (s.parts == 1) return 0;
  return align_up((size_t)P.rows * s.parts * sizeof(Part), 256) +
         (size_t)P.rows * s.parts * P.top * sizeof(uint64_t);
}

int launch_probs_forward(const ProbsParams& P, const void* logits,
                         float* log_probs, float* entropy, float* top_log_probs,
                         int32_t* top_codes, float2* stats, void* workspace,
                         hipStream_t stream) {
  if (P.rows == 0) return GSPLAT_OK;
  auto f = P.dtype == GSPLAT_F32    ? forward_of<float>
           : P.dtype == GSPLAT_BF16 ? forward_of<__bf16>
                                    : forward_of<_Float16>;
  return f(P, logits, ProbsOut{log_probs, entropy, top_log_probs, top_codes, stats},
           workspace, stream);
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
