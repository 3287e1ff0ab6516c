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
// Sums over rows are taken in a fixed order (rows of a team, teams of a
// workgroup, workgroups), counts are integers: the same inputs give the same
// bits.
//
// One launch reads the logits once and leaves each workgroup's column sums and
// counts, a second joins them; the backward is one pass.  On an MI355X: four
// images of 64K rows x 256 floats 50 + 9 us forward (4.6 TB/s: start and end of
// the persistent workgroups and the join are a fifth of it) and 81 us backward
// (6.7 TB/s); 200K rows x 4096 in bf16 348 + 16 us (4.6 TB/s, VALU issue beside
// HBM) and 605 us (5.4 TB/s).  Above 16384 codes both directions read the logits
// twice: 4096 rows x 32768 floats 141 + 103 + 19 us and 349 us.
#include <algorithm>
#include <type_traits>

#include "codes.h"

namespace gs {
namespace {

// A team reads a row once and holds it in registers: TL lanes of one wavefront
// (W = 1), or W wavefronts.  A thread holds R vectors (12 or 16 floats, 16 or 24
// elements of 16 bits, 32 of long rows) of the row at hand, its probabilities and
// (forward) its columns' sums or (backward) its columns' a; the next row is
// loaded once its probabilities are there.  What a row costs besides its elements
// (reductions, its choices) is the same for a lane with 4 elements and one
// with 32, so teams are as narrow as that allows.  The workgroups take rows in
// turn, so that all of them together move through the logits from front to back
// (each in a range of its own: 512K rows of 256 floats 122 us forward and 208
// backward; in turn 113 and 186).
//
// (Four wavefronts per SIMD: the compiler would otherwise take more registers
// than it needs with 32 elements a lane.)
#define GS_WAVES __attribute__((amdgpu_waves_per_eu(4)))
template <typename T, int TL, int W, int R, bool Even>
struct Team {
  static constexpr int V = kVec<T>;
  static constexpr int kThreads = W > 4 ? 64 * W : 256;
  static constexpr int kTeams = kThreads / (TL * W);  // per workgroup
  static constexpr int kColumns = TL * W * V * R;
  static __device__ __forceinline__ int team() { return threadIdx.x / (TL * W); }
  static __device__ __forceinline__ int member() { return threadIdx.x & (TL * W - 1); }
  static __device__ __forceinline__ int wave() { return W > 1 ? (threadIdx.x >> 6) & (W - 1) : 0; }
  static __device__ __forceinline__ int column(int r) { return (r * TL * W + member()) * V; }
  // (Late: fix is called once the vectors are there.  The backward of 32 bits is
  // better without: 522K rows of 257 floats 245 us, 263 with.)
  template <bool Stream, bool Late = true>
  static __device__ __forceinline__ void load(vec_t<T> (&x)[R], const T* row, int K) {
    const T fill = static_cast<T>(-INFINITY);
    if constexpr (Late) {
      load_row<T, R, Even, Stream>(x, row, column(0), TL * W * V, K, fill);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = load_part<T, Even, Stream>(row, column(r), K, fill);
    }
  }
  static __device__ __forceinline__ void fix(vec_t<T> (&x)[R], int K) {
    fix_row<T, R, Even>(x, column(0), TL * W * V, K, static_cast<T>(-INFINITY));
  }
};

// What the workgroups of the row pass leave: for image b and workgroup i
// (blocks of them per image) sums[(b * blocks + i) * K + k], and counts and
// totals likewise for i < count_blocks.
struct Partials {
  int blocks, count_blocks;
  float* sums;
  int32_t* counts;
  int4* totals;  // rows that take part, choices, bad codes
  float* loss;   // [batch][column groups]
  uint32_t* tickets;  // [batch], zeroed by the row pass
  bool stream;  // past_caches
};

// The choices of a row (kept by the lanes of a wavefront): counts them.
struct Choices {
  int given = 0, bad = 0;
  __device__ __forceinline__ void count(int c, int32_t* hist) {
    if (c >= 0) {
      ++given;
      if (hist) atomicAdd(&hist[c], 1);
    } else if (c == kBadCode) {
      ++bad;
    }
  }
};

template <typename T, int TL, int W, int R, bool Even>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) GS_WAVES void balance_rows_kernel(
    BalanceParams P, const T* __restrict__ logits, float2* __restrict__ stats,
    Partials out) {
  using G = Team<T, TL, W, R, Even>;
  constexpr int V = G::V;
  extern __shared__ int32_t lds[];  // K counts, then (teams > 1) K sums
  __shared__ float2 slots[2][G::kTeams][W];
  __shared__ int sum3[3];
  int32_t* hist = lds;
  float* sums = reinterpret_cast<float*>(lds + P.K);
  const int b = blockIdx.y;
  for (int k = threadIdx.x; k < P.K; k += G::kThreads) hist[k] = 0;
  if (threadIdx.x < 3) sum3[threadIdx.x] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) out.tickets[b] = 0;
  __syncthreads();

  const float c = kLog2e;
  const int lane = threadIdx.x & (TL - 1), w = G::wave();
  const int S = P.choices;
  float acc[R * V];
#pragma unroll
  for (int j = 0; j < R * V; ++j) acc[j] = 0.0f;
  int took = 0, given = 0, bad = 0;
  vec_t<T> x[R];
  auto load = [&](const T* row) {
    if (out.stream)
      G::template load<true>(x, row, P.K);
    else
      G::template load<false>(x, row, P.K);
  };
  const int64_t base_row = b * P.rows, step = (int64_t)gridDim.x * G::kTeams;
  auto row_of = [&](int64_t i) { return base_row + min(i, P.rows - 1); };
  int64_t from = (int64_t)blockIdx.x * G::kTeams;  // the workgroup's first row of a turn
  int64_t i = from + G::team();
  int code = kNoCode;
  if (from < P.rows) {
    load(logits + row_of(i) * P.stride);
    if (lane < S) code = P.codes.at(row_of(i) * S + lane, P.K);
  }
  // (every team makes the same number of turns; those past the rows count nothing)
  for (int turn = 0; from < P.rows; turn ^= 1, from += step, i += step) {
    G::fix(x, P.K);
    const int64_t r0 = row_of(i);
    const bool here = i < P.rows;
    Choices mine;
    if (here) {
      int32_t* h = w == 0 ? hist : nullptr;
      if (lane < S) mine.count(code, h);
      for (int j = lane + TL; j < S; j += TL) mine.count(P.codes.at(r0 * S + j, P.K), h);
    }
    const bool part = team_umax<TL>(mine.given) != 0;
    given += mine.given;
    bad += mine.bad;
    took += part && lane == 0;

    float m = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float most = to_float(x[r][0]);
#pragma unroll
      for (int v = 1; v + 1 < V; v += 2) most = max3(most, to_float(x[r][v]), to_float(x[r][v + 1]));
      m = max3(m, most, to_float(x[r][V - 1]));
    }
    m = team_max<TL>(m);
    const Exponent ex(m == -INFINITY ? 0.0f : m, 0.0f, c);
    float e[R * V], s = 0.0f;
    auto powers = [&](auto exponent) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        forget<T>(x[r]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          e[r * V + v] = exp2_fast(exponent(to_float(x[r][v])));
          s += e[r * V + v];
        }
      }
    };
    if (ex.plain)
      powers([&](float y) { return ex.fast(y); });
    else
      powers([&](float y) { return ex.slow(y); });
    if (from + step < P.rows) {  // (x is free: the next row)
      const int64_t rn = row_of(i + step);
      load(logits + rn * P.stride);
      code = lane < S ? P.codes.at(rn * S + lane, P.K) : kNoCode;
    }
    s = team_sum<TL>(s);
    // (the powers lack ex.shift: it cancels from e / s, not from log2 s)
    float base = ex.m, shift = ex.shift, f = 1.0f;
    if constexpr (W > 1) {  // (two sets of slots: one barrier a row)
      float2* slot = slots[turn][W > 1 ? G::team() : 0];
      if (lane == 0) slot[w] = make_float2(m, s * exp2_fast(shift));
      __syncthreads();
      const float2 q = slot[lane & (W - 1)];
      const float all = team_max<W>(q.x);
      base = all == -INFINITY ? 0.0f : all;
      s = team_sum<W>(q.y * exp2_fast(fmaxf((q.x - base) * c, -1000.0f)));
      f = exp2_fast(fmaxf((m - base) * c, -1000.0f) + shift);
      shift = 0.0f;
    }
    const bool counts_in = here && part && s != 0.0f;
    if (here && G::member() == 0)
      stats[r0] = make_float2(base, counts_in ? log2_fast(s) + shift : INFINITY);
    if (counts_in) {
      f *= __builtin_amdgcn_rcpf(s);
#pragma unroll
      for (int j = 0; j < R * V; ++j) acc[j] = __builtin_fmaf(e[j], f, acc[j]);
    }
  }

  // rows, choices and bad codes of the workgroup (wavefront 0 of a wide team)
  if (W == 1 || w == 0) {
    given = wave_isum(given);
    bad = wave_isum(bad);
    took = wave_isum(took);
    if ((threadIdx.x & 63) == 0) {
      atomicAdd(&sum3[0], took);
      atomicAdd(&sum3[1], given);
      atomicAdd(&sum3[2], bad);
    }
  }
  const int64_t at = (int64_t)b * out.blocks + blockIdx.x;
  if constexpr (G::kTeams > 1) {
    // teams of a wavefront, then wavefronts or wider teams one after another
    if constexpr (TL < 64)
#pragma unroll
      for (int j = 0; j < R * V; ++j)
#pragma unroll
        for (int d = TL; d < 64; d <<= 1) acc[j] += __shfl_xor(acc[j], d, 64);
    const int group = threadIdx.x / (64 * W);
    for (int q = 0; q < G::kThreads / (64 * W); ++q) {
      if (group == q && (threadIdx.x & 63) < TL)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int k = G::column(r);
          if (k >= P.K) continue;
          float had[V];  // (reads, then writes: both in whole vectors)
#pragma unroll
          for (int v = 0; v < V; ++v) had[v] = q == 0 || (!Even && k + v >= P.K) ? 0.0f : sums[k + v];
#pragma unroll
          for (int v = 0; v < V; ++v)
            if (Even || k + v < P.K) sums[k + v] = had[v] + acc[r * V + v];
        }
      __syncthreads();
    }
    for (int k = threadIdx.x; k < P.K; k += G::kThreads) out.sums[at * P.K + k] = sums[k];
  } else {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = G::column(r);
      float* to = out.sums + at * P.K + k;
      if (k >= P.K) continue;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (Even || k + v < P.K) to[v] = acc[r * V + v];
    }
  }
  for (int k = threadIdx.x; k < P.K; k += G::kThreads) out.counts[at * P.K + k] = hist[k];
  if (threadIdx.x == 0) out.totals[at] = make_int4(sum3[0], sum3[1], sum3[2], 0);
}

// ---- the workgroups' sums joined: Columns (32 or 64) columns of an image per
// workgroup, whole cache lines, in slices that each take every so many-th of the
// sums.  The image's last workgroup adds up the loss.

constexpr int kJoinThreads = 1024;

template <int Columns>
__global__ __launch_bounds__(kJoinThreads) void balance_join_kernel(
    BalanceParams P, Partials in, float* __restrict__ loss,
    int32_t* __restrict__ counts, float* __restrict__ mean,
    int4* __restrict__ totals) {
  constexpr int kSlices = kJoinThreads / Columns;
  __shared__ float sums[kJoinThreads];
  __shared__ int nums[kJoinThreads];
  __shared__ int all[3];
  const int slice = threadIdx.x / Columns, b = blockIdx.y;
  const int k = blockIdx.x * Columns + threadIdx.x % Columns;
  if (threadIdx.x < 3) all[threadIdx.x] = 0;
  __syncthreads();
  int4 t = make_int4(0, 0, 0, 0);
  for (int i = threadIdx.x; i < in.count_blocks; i += kJoinThreads) {
    const int4 q = in.totals[(int64_t)b * in.count_blocks + i];
    t.x += q.x;
    t.y += q.y;
    t.z += q.z;
  }
  if (t.x) atomicAdd(&all[0], t.x);
  if (t.y) atomicAdd(&all[1], t.y);
  if (t.z) atomicAdd(&all[2], t.z);
  float s = 0.0f;
  int n = 0;
  if (k < P.K) {
    // (eight of each on their way: with loads waited for one after another the
    // launch is latency)
    const float* ps = in.sums + (int64_t)b * in.blocks * P.K + k;
    const int32_t* pn = in.counts + (int64_t)b * in.count_blocks * P.K + k;
    const int last = max(in.blocks, in.count_blocks);
    for (int i0 = slice; i0 < last; i0 += 8 * kSlices) {
      float x[8];
      int y[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * kSlices;
        x[u] = i < in.blocks ? ps[(int64_t)i * P.K] : 0.0f;
        y[u] = i < in.count_blocks ? pn[(int64_t)i * P.K] : 0;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        s += x[u];
        n += y[u];
      }
    }
  }
  sums[threadIdx.x] = s;
  nums[threadIdx.x] = n;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  // one wavefront: its lanes take every slice, or each half of them every second
  const int lane = threadIdx.x;
  for (int j = lane + 64; j < kJoinThreads; j += 64) {
    s += sums[j];
    n += nums[j];
  }
#pragma unroll
  for (int d = Columns; d < 64; d <<= 1) {
    s += __shfl_xor(s, d, 64);
    n += __shfl_xor(n, d, 64);
  }
  const float mu = s / (float)max(all[0], 1);
  const bool mine = lane < Columns && k < P.K;
  if (mine) {
    counts[(int64_t)b * P.K + k] = n;
    mean[(int64_t)b * P.K + k] = mu;
  }
  if (blockIdx.x == 0 && lane == 0) totals[b] = make_int4(all[0], all[1], all[2], 0);
  // (an image with nothing counted: 0, whatever the means are)
  float l = wave_sum(mine && n ? (float)n * mu : 0.0f);
  const float factor = (float)P.K / (float)max(all[1], 1);
  if (gridDim.x > 1) {
    float* parts = in.loss + (int64_t)b * gridDim.x;
    uint32_t ticket = 0;
    if (lane == 0) {
      __hip_atomic_store(&parts[blockIdx.x], l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      ticket = __hip_atomic_fetch_add(&in.tickets[b], 1u, __ATOMIC_ACQ_REL,
                                      __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((uint32_t)__builtin_amdgcn_readfirstlane((int)ticket) != gridDim.x - 1) return;
    l = 0.0f;
    for (unsigned i = lane; i < gridDim.x; i += 64)
      l += __hip_atomic_load(&parts[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    l = wave_sum(l);
  }
  if (lane == 0) loss[b] = all[2] ? __builtin_nanf("") : l * factor;
}

// ---- backward

template <typename T, int TL, int W, int R, bool Even, bool Past>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) GS_WAVES void balance_bwd_kernel(
    BalanceParams P, const T* __restrict__ logits,
    const int32_t* __restrict__ counts, const float2* __restrict__ stats,
    const int4* __restrict__ totals, const float* __restrict__ g_loss,
    const float* __restrict__ g_mean, T* __restrict__ g_logits) {
  using G = Team<T, TL, W, R, Even>;
  constexpr int V = G::V;
  constexpr float kUp = sizeof(T) == 2 ? 32.0f : 0.0f;
  __shared__ float slots[2][G::kTeams][W];
  const int b = blockIdx.y;
  const int lane = threadIdx.x & (TL - 1), w = G::wave();
  const int4 tot = totals[b];
  const float per_row = 1.0f / (float)max(tot.x, 1);
  const float per_count = g_loss ? g_loss[b] * ((float)P.K / (float)max(tot.y, 1)) : 0.0f;
  float a[R * V];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    // (without a branch, and in whole vectors where the rows are)
    const int k = G::column(r), last = k < P.K ? k : 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      a[r * V + v] = per_count * (float)(counts + (int64_t)b * P.K)[Even ? last + v : min(k + v, P.K - 1)];
    if (g_mean)
#pragma unroll
      for (int v = 0; v < V; ++v)
        a[r * V + v] += (g_mean + (int64_t)b * P.K)[Even ? last + v : min(k + v, P.K - 1)];
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (k + v >= P.K) a[r * V + v] = 0.0f;
  }
  const int64_t base_row = b * P.rows, step = (int64_t)gridDim.x * G::kTeams;
  auto row_of = [&](int64_t i) { return base_row + min(i, P.rows - 1); };
  int64_t from = (int64_t)blockIdx.x * G::kTeams;  // the workgroup's first row of a turn
  int64_t i = from + G::team();
  vec_t<T> x[R];
  G::template load<true, sizeof(T) == 2>(x, logits + row_of(i) * P.stride, P.K);
  float2 st = stats[row_of(i)];
  for (int turn = 0; from < P.rows; turn ^= 1, from += step, i += step) {
    if (sizeof(T) == 2) G::fix(x, P.K);
    const int64_t r0 = row_of(i);
    // p = 2^(t + down) with t from Exponent (16 bits: exponents 32 up, as in
    // code_probs.hip); a row that takes no part has log2 s = inf and p = 0.
    const Exponent ex(st.x, st.y - kUp, kLog2e);
    const float down = exp2_fast(ex.shift - kUp);
    float p[R * V], dot = 0.0f;
    auto products = [&](auto exponent) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        forget<T>(x[r]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int j = r * V + v;
          // (a NaN in a row that takes no part is no part of it; one that does
          // has a NaN in its constants)
          const float t = fmaxf(exponent(to_float(x[r][v])), -1000.0f);
          p[j] = sizeof(T) == 2 ? exp2_fast(t) : exp2_full(t);
          dot = __builtin_fmaf(p[j], a[j], dot);
        }
      }
    };
    if (ex.plain)
      products([&](float y) { return ex.fast(y); });
    else
      products([&](float y) { return ex.slow(y); });
    if (from + step < P.rows) {  // (x is free: the next row)
      const int64_t rn = row_of(i + step);
      G::template load<true, sizeof(T) == 2>(x, logits + rn * P.stride, P.K);
      st = stats[rn];
    }
    dot = team_sum<TL>(dot) * down;
    if constexpr (W > 1) {
      float* slot = slots[turn][W > 1 ? G::team() : 0];
      if (lane == 0) slot[w] = dot;
      __syncthreads();
      dot = team_sum<W>(slot[lane & (W - 1)]);
    }
    if (i < P.rows) {
      T* out = g_logits + r0 * P.K;
      const float f = down * per_row, less = -dot * f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        vec_t<T> o;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int j = r * V + v;
          o[v] = static_cast<T>(p[j] * __builtin_fmaf(a[j], f, less));
        }
        store_part<T, Even, Past>(out, G::column(r), P.K, o);
      }
    }
  }
}

// ---- codebooks above 16384: a row does not fit a workgroup's registers, and
// is read twice in each direction

constexpr int kThreads = 256;
constexpr int kWaves = 4;

__device__ __forceinline__ float prob(float x, float2 st) {
  return st.y == INFINITY ? 0.0f : exp2_full((x - st.x) * kLog2e - st.y);
}

// A workgroup per row.  The only counts and totals of an image: zero on entry.
template <typename T>
__global__ __launch_bounds__(kThreads) void balance_long_rows_kernel(
    BalanceParams P, const T* __restrict__ logits, float2* __restrict__ stats,
    Partials out) {
  __shared__ float2 slots[kWaves];
  const int64_t r = blockIdx.x;
  const int b = (int)(r / P.rows);
  const T* row = logits + r * P.stride;
  // online: (m, s) of this thread's elements
  float m = -INFINITY, s = 0.0f;
  for (int i = threadIdx.x * kVec<T>; i < P.K; i += kThreads * kVec<T>) {
    const vec_t<T> x = load_part<T>(row, i, P.K, static_cast<T>(-INFINITY));
    float top = m;
#pragma unroll
    for (int v = 0; v < kVec<T>; ++v) top = fmaxf(top, to_float(x[v]));
    const float base = top == -INFINITY ? 0.0f : top;
    s *= exp2_fast(fmaxf((m - base) * kLog2e, -1000.0f));
#pragma unroll
    for (int v = 0; v < kVec<T>; ++v) s += exp2_fast((to_float(x[v]) - base) * kLog2e);
    m = top;
  }
  const float wm = wave_max(m), wb = wm == -INFINITY ? 0.0f : wm;
  s = wave_sum(s * exp2_fast(fmaxf((m - wb) * kLog2e, -1000.0f)));
  if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = make_float2(wm, s);
  Choices mine;
  for (int j = threadIdx.x; j < P.choices; j += kThreads)
    mine.count(P.codes.at(r * P.choices + j, P.K), out.counts + (int64_t)b * P.K);
  if (mine.given) atomicAdd(&out.totals[b].y, mine.given);
  if (mine.bad) atomicAdd(&out.totals[b].z, mine.bad);
  const bool part = __syncthreads_or(mine.given);
  if (threadIdx.x != 0) return;
  m = slots[0].x;
  for (int j = 1; j < kWaves; ++j) m = fmaxf(m, slots[j].x);
  const float base = m == -INFINITY ? 0.0f : m;
  s = 0.0f;
  for (int j = 0; j < kWaves; ++j)
    s += slots[j].y * exp2_fast(fmaxf((slots[j].x - base) * kLog2e, -1000.0f));
  stats[r] = make_float2(base, part && s != 0.0f ? log2_fast(s) : INFINITY);
  if (part) atomicAdd(&out.totals[b].x, 1);
}

// Sums of columns over a chunk of an image's rows.
template <typename T>
__global__ __launch_bounds__(kThreads) void balance_columns_kernel(
    BalanceParams P, const T* __restrict__ logits,
    const float2* __restrict__ stats, Partials out) {
  const int k = (blockIdx.x * kThreads + threadIdx.x) * kVec<T>;
  const int b = blockIdx.z;
  if (k >= P.K) return;
  const int64_t per = (P.rows + out.blocks - 1) / out.blocks;
  const int64_t first = blockIdx.y * per, end = min(first + per, P.rows);
  float acc[kVec<T>];
#pragma unroll
  for (int v = 0; v < kVec<T>; ++v) acc[v] = 0.0f;
  for (int64_t n = first; n < end; ++n) {
    const int64_t r = b * P.rows + n;
    const float2 st = stats[r];
    const vec_t<T> x = load_part<T>(logits + r * P.stride, k, P.K, static_cast<T>(-INFINITY));
#pragma unroll
    for (int v = 0; v < kVec<T>; ++v) acc[v] += prob(to_float(x[v]), st);
  }
  float* to = out.sums + ((int64_t)b * out.blocks + blockIdx.y) * P.K;
#pragma unroll
  for (int v = 0; v < kVec<T>; ++v)
    if (k + v < P.K) to[k + v] = acc[v];
}

// kLongRows rows of an image per workgroup, so that the columns' weights are
// read once for as many elements.
template <typename T, int kLongRows>
__global__ __launch_bounds__(kThreads) void balance_long_bwd_kernel(
    BalanceParams P, const T* __restrict__ logits,
    const int32_t* __restrict__ counts, const float2* __restrict__ stats,
    const int4* __restrict__ totals, const float* __restrict__ g_loss,
    const float* __restrict__ g_mean, T* __restrict__ g_logits) {
  constexpr int V = kVec<T>;
  __shared__ float red[kWaves];
  const int b = blockIdx.y;
  const int64_t first = (int64_t)blockIdx.x * kLongRows;
  const int rows = (int)min((int64_t)kLongRows, P.rows - first);
  const int4 tot = totals[b];
  const float per_row = 1.0f / (float)max(tot.x, 1);
  const float per_count = g_loss ? g_loss[b] * ((float)P.K / (float)max(tot.y, 1)) : 0.0f;
  const int32_t* count = counts + (int64_t)b * P.K;
  const float* mean = g_mean ? g_mean + (int64_t)b * P.K : nullptr;
  auto weights = [&](int k, float (&a)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[v] = k + v < P.K ? per_count * (float)count[k + v] : 0.0f;
      if (mean && k + v < P.K) a[v] += mean[k + v];
    }
  };
  const T* x[kLongRows];
  float2 st[kLongRows];
  float dot[kLongRows];
#pragma unroll
  for (int q = 0; q < kLongRows; ++q) {
    const int64_t r = b * P.rows + first + min(q, rows - 1);
    x[q] = logits + r * P.stride;
    st[q] = stats[r];
    dot[q] = 0.0f;
  }
  for (int k = threadIdx.x * V; k < P.K; k += kThreads * V) {
    float a[V];
    weights(k, a);
#pragma unroll
    for (int q = 0; q < kLongRows; ++q) {
      const vec_t<T> y = load_part<T>(x[q], k, P.K, static_cast<T>(-INFINITY));
#pragma unroll
      for (int v = 0; v < V; ++v) dot[q] = __builtin_fmaf(prob(to_float(y[v]), st[q]), a[v], dot[q]);
    }
  }
#pragma unroll
  for (int q = 0; q < kLongRows; ++q) dot[q] = block_sum<kWaves>(dot[q], red);
  for (int k = threadIdx.x * V; k < P.K; k += kThreads * V) {
    float a[V];
    weights(k, a);
#pragma unroll
    for (int q = 0; q < kLongRows; ++q) {
      if (q >= rows) break;
      const vec_t<T> y = load_part<T>(x[q], k, P.K, static_cast<T>(-INFINITY));
      vec_t<T> o;
#pragma unroll
      for (int v = 0; v < V; ++v)
        o[v] = static_cast<T>(prob(to_float(y[v]), st[q]) * (a[v] - dot[q]) * per_row);
      store_part<T, false, true>(g_logits + (b * P.rows + first + q) * P.K, k, P.K, o);
    }
  }
}

// ---- host

constexpr int kLongest = 16384;  // codes of a row that a workgroup holds

// Teams of a workgroup of the kernel that GS_TEAMS takes.
int teams_of(const BalanceParams& P) {
  const bool narrow = P.dtype != GSPLAT_F32;
  int threads = 2;
  while (threads < 64 && threads * (narrow ? 24 : 16) < P.K) threads *= 2;
  if (threads * (narrow ? 24 : 16) < P.K)
    while (threads * (narrow && P.K % 8 == 0 ? 32 : 16) < P.K) threads *= 2;
  return std::max(1, 256 / threads);
}

// Workgroups per image of the row pass, each of which leaves its columns' sums
// and counts, 8 bytes per code: 1024 in all keep the GPU busy (200K rows x 4096
// 368 us, with 512 476, with 2048 371; four images x 256 54, 60, 59).
// Above 16384 codes, chunks of an image's rows, whose columns are shared out over
// further workgroups: eight rows at least, so that the sums are an eighth of the
// logits in 32 bits, a quarter in 16 (forwards of 64 images of 256 rows x 32768 in
// bf16 1457 us with 143 MB of sums, a chunk a row 3474 with 2156 MB; one of 100 x
// 100000 79 and 110, of 4096 x 32768 191 and 190).
int blocks_of(const BalanceParams& P) {
  if (P.rows == 0) return 1;
  if (P.K > kLongest) {
    const int64_t most = std::max(1, std::min(256, 1024 / P.batch));
    return (int)std::clamp<int64_t>(P.rows / 8, 1, most);
  }
  // two rows for each team, at least: what a workgroup costs at its start and
  // end, and the join its sums, is then worth it (16384 rows of 64 floats: 14 us,
  // 17 with eight rows a workgroup; 1024 of 4096 in bf16 20 and 27)
  const int64_t least = 2 * teams_of(P);
  const int64_t most = std::max<int64_t>(1, (P.K > 8192 ? 256 : P.K > 4096 ? 512 : 1024) / P.batch);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, P.rows / least));
}

// (The tickets of an image's workgroups are taken one after another, 33 ns each:
// above 4096 columns in all, half as many workgroups.  Four images of 8192 codes
// 18 us and 37, of 2048 11 and 13; one of 4096 17.5 and 15.)
int join_columns(const BalanceParams& P) {
  return (int64_t)P.K * P.batch > 4096 ? 64 : 32;
}

int column_groups(const BalanceParams& P) {
  return (P.K + join_columns(P) - 1) / join_columns(P);
}

struct Layout {
  size_t sums, counts, totals, loss, tickets, total;
};
Layout layout(const BalanceParams& P) {
  const size_t blocks = (size_t)blocks_of(P) * P.batch;
  const size_t count_blocks = P.K > kLongest ? (size_t)P.batch : blocks;
  Layout L{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += align_up(bytes, 256);
    return at;
  };
  L.sums = take(blocks * P.K * 4);
  L.counts = take(count_blocks * P.K * 4);
  L.totals = take(count_blocks * sizeof(int4));
  L.loss = take((size_t)P.batch * column_groups(P) * 4);
  L.tickets = take((size_t)P.batch * 4);
  L.total = off;
  return L;
}

// The kernel for rows of K codes: CALL(TL, W, R).  Three vectors a lane between
// the powers of two (672K rows of 192 in bf16: 73 us forward, with lanes half idle
// 99; 512K of 257 floats 151 and 161), in 16 bits from LEAST lanes on: a backward's
// stores of a narrower team are parts of lines (1M rows of 48: 56 us, and 43
// with two vectors).
#define GS_TEAMS(CALL, LEAST)                                               \
  constexpr int kR = 16 / kVec<T>;                                          \
  constexpr int kA = sizeof(T) == 2 ? kR : 3, kB = sizeof(T) == 2 ? 3 : kR; \
  if (vecs <= 2) CALL(2, 1, 1);                                             \
  if (vecs <= 2 * kA) CALL(2, 1, kA);                                       \
  if (vecs <= 2 * kB && (kB > 3 || 2 >= LEAST)) CALL(2, 1, kB);             \
  if (vecs <= 4 * kA) CALL(4, 1, kA);                                       \
  if (vecs <= 4 * kB && (kB > 3 || 4 >= LEAST)) CALL(4, 1, kB);             \
  if (vecs <= 8 * kA) CALL(8, 1, kA);                                       \
  if (vecs <= 8 * kB) CALL(8, 1, kB);                                       \
  if (vecs <= 16 * kA) CALL(16, 1, kA);                                     \
  if (vecs <= 16 * kB) CALL(16, 1, kB);                                     \
  if (vecs <= 32 * kA) CALL(32, 1, kA);                                     \
  if (vecs <= 32 * kB) CALL(32, 1, kB);                                     \
  if (vecs <= 64 * kA) CALL(64, 1, kA);                                     \
  if (vecs <= 64 * kB) CALL(64, 1, kB);                                     \
  if constexpr (sizeof(T) == 2 && Even) {                                   \
    if (vecs <= 128 * kR) CALL(64, 1, 2 * kR);                              \
    if (vecs <= 256 * kR) CALL(64, 2, 2 * kR);                              \
    if (vecs <= 512 * kR) CALL(64, 4, 2 * kR);                              \
    CALL(64, 8, 2 * kR);                                                    \
  } else {                                                                  \
    if (vecs <= 128 * kR) CALL(64, 2, kR);                                  \
    if (vecs <= 256 * kR) CALL(64, 4, kR);                                  \
    if (vecs <= 512 * kR) CALL(64, 8, kR);                                  \
    CALL(64, 16, kR);                                                       \
  }

template <typename T, bool Even>
int rows_of(const BalanceParams& P, const T* x, float2* stats, const Partials& w,
            hipStream_t stream) {
  const int vecs = (P.K + kVec<T> - 1) / kVec<T>;
#define GS_ROWS(TL, W, R)                                                     \
  {                                                                           \
    using G = Team<T, TL, W, R, Even>;                                              \
    launch_traced("balance_rows_kernel", (balance_rows_kernel<T, TL, W, R, Even>),  \
                  dim3((unsigned)w.blocks, (unsigned)P.batch), dim3(G::kThreads), \
                  (size_t)P.K * (G::kTeams > 1 ? 8 : 4), stream, P, x, stats, w); \
    return check_launch("balance_rows_kernel");                               \
  }
  GS_TEAMS(GS_ROWS, 2)
#undef GS_ROWS
}

template <typename T>
int forward_of(const BalanceParams& P, const void* logits, float* loss,
               int32_t* counts, float* mean, float2* stats, int32_t* totals,
               char* ws, hipStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  const Layout L = layout(P);
  const bool is_long = P.K > kLongest;
  Partials w{blocks_of(P), is_long ? 1 : blocks_of(P),
             reinterpret_cast<float*>(ws + L.sums),
             reinterpret_cast<int32_t*>(ws + L.counts),
             reinterpret_cast<int4*>(ws + L.totals),
             reinterpret_cast<float*>(ws + L.loss),
             reinterpret_cast<uint32_t*>(ws + L.tickets),
             past_caches(P.rows * P.batch, P.K, P.dtype)};
  int rc;
  if (!is_long) {
    rc = P.K % kVec<T> == 0 ? rows_of<T, true>(P, x, stats, w, stream)
                            : rows_of<T, false>(P, x, stats, w, stream);
  } else {
    // (one launch zeroes counts, totals, the loss' parts and the tickets; the
    // sums of no rows are zeroed too)
    rc = launch_zero_u32(reinterpret_cast<uint32_t*>(ws + (P.rows ? L.counts : L.sums)),
                         (int64_t)(L.total - (P.rows ? L.counts : L.sums)) / 4, stream);
    if (rc) return rc;
    if (P.rows > 0) {
      launch_traced("balance_long_rows_kernel", (balance_long_rows_kernel<T>),
                    dim3((unsigned)(P.rows * P.batch)), dim3(kThreads), 0, stream, P, x,
                    stats, w);
      rc = check_launch("balance_long_rows_kernel");
      if (rc) return rc;
      const int per = kThreads * kVec<T>;
      launch_traced("balance_columns_kernel", (balance_columns_kernel<T>),
                    dim3((unsigned)((P.K + per - 1) / per), (unsigned)w.blocks,
                         (unsigned)P.batch),
                    dim3(kThreads), 0, stream, P, x, stats, w);
      rc = check_launch("balance_columns_kernel");
    }
  }
  if (rc) return rc;
  launch_traced("balance_join_kernel",
                join_columns(P) == 64 ? balance_join_kernel<64> : balance_join_kernel<32>,
                dim3((unsigned)column_groups(P), (unsigned)P.batch),
                dim3(kJoinThreads), 0, stream, P, w, loss, counts, mean,
                reinterpret_cast<int4*>(totals));
  return check_launch("balance_join_kernel");
}

template <typename T, bool Even>
int gradients_of(const BalanceParams& P, const T* x, const int32_t* counts,
                 const float2* stats, const int4* totals, const float* g_loss,
                 const float* g_mean, T* g, hipStream_t stream) {
  const int vecs = (P.K + kVec<T> - 1) / kVec<T>;
  // Gradients go past the caches, which are left to the logits (forward and
  // backward of 256 MiB of rows of 1024 floats 146 us so and 184 through the
  // caches, of 128 MiB 84 and 86; the backward alone, of logits that nothing read
  // before, 96 and 87), where a store writes whole lines of a row, or many: 1M
  // rows of 100 floats (128 bytes of a row per store, anywhere in its lines) 276
  // us so and 188 through the caches, of 32 (half a line) 140 and 81.
  const bool whole = P.K * sizeof(T) % 128 == 0;
#define GS_BWD(TL, W, R)                                                      \
  {                                                                           \
    using G = Team<T, TL, W, R, Even>;                                              \
    const int64_t most = std::max(1, (W > 4 ? 4096 / W : 1024) / P.batch);         \
    const int64_t turns = (P.rows + G::kTeams - 1) / G::kTeams;               \
    auto launch = [&](auto past) {                                            \
      launch_traced("balance_bwd_kernel",                                     \
                    (balance_bwd_kernel<T, TL, W, R, Even, past.value>),      \
                    dim3((unsigned)std::min(most, turns), (unsigned)P.batch), \
                    dim3(G::kThreads), 0, stream, P, x, counts, stats,        \
                    totals, g_loss, g_mean, g);                               \
    };                                                                        \
    if (TL >= 32 || (TL >= 8 && whole))                                       \
      launch(std::integral_constant<bool, (TL >= 8)>{});                      \
    else                                                                      \
      launch(std::false_type{});                                              \
    return check_launch("balance_bwd_kernel");                                \
  }
  GS_TEAMS(GS_BWD, 8)
#undef GS_BWD
}
#undef GS_TEAMS

template <typename T>
int backward_of(const BalanceParams& P, const void* logits, const int32_t* counts,
                const float2* stats, const int4* totals, const float* g_loss,
                const float* g_mean, void* g_logits, hipStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  T* g = static_cast<T*>(g_logits);
  if (P.K <= kLongest)
    return P.K % kVec<T> == 0
               ? gradients_of<T, true>(P, x, counts, stats, totals, g_loss, g_mean, g, stream)
               : gradients_of<T, false>(P, x, counts, stats, totals, g_loss, g_mean, g, stream);
#define GS_LONG(Q)                                                              \
  launch_traced("balance_long_bwd_kernel", (balance_long_bwd_kernel<T, Q>),     \
                dim3((unsigned)((P.rows + Q - 1) / Q), (unsigned)P.batch),      \
                dim3(kThreads), 0, stream, P, x, counts, stats, totals, g_loss, \
                g_mean, g)
  // (4096 rows of 32768: 430 us in 32 bits with four rows, 602 with one, 281 and
  // 915 in 16; 1342 rows of 100000: 909, 859 and 706 us in 32 bits with four, two
  // and one, 577, 619 and 1061 in 16)
  if (sizeof(T) == 2 || P.rows * P.batch >= 4096) GS_LONG(4);
  else GS_LONG(1);
#undef GS_LONG
  return check_launch("balance_long_bwd_kernel");
}

}  // namespace

size_t balance_workspace_bytes(const BalanceParams& P) { return layout(P).total; }

int launch_balance_forward(const BalanceParams& P, const void* logits,
                           float* loss, int32_t* counts, float* mean_probs,
                           float2* stats, int32_t* totals, void* workspace,
                           hipStream_t stream) {
  auto f = P.dtype == GSPLAT_F32    ? forward_of<float>
           : P.dtype == GSPLAT_BF16 ? forward_of<__bf16>
                                    : forward_of<_Float16>;
  return f(P, logits, loss, counts, mean_probs, stats, totals,
           static_cast<char*>(workspace), stream);
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
  return f(P, logits, counts, stats, reinterpret_cast<const int4*>(totals), g_loss,
           g_mean, g_logits, stream);
}

}  // namespace gs
