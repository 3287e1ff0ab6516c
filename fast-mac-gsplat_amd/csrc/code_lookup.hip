// code_lookup.hip -- attributes of splats from a codebook, and the gradient.
//
//   out[n] = f s_n C[c_n]                     (c_n = -1: zeros)
//   gC[k]  = f * sum over n with c_n = k of s_n g[n]
//   gs[n]  = f <g[n], C[c_n]>
//
// The gradient of the codebook is a sum by code, in an order that does not
// depend on the run (no atomics: the same inputs give the same bits).
//
// Few splats: a workgroup takes one to four codes, reads every splat's code,
// lists those that name one of its own and adds up their rows (one launch, or two
// where the splats are taken in chunks: chunks_of below).
//
// More splats: they are sorted by code (stable), so that a code's splats are
// one run of the sorted positions.  A team of lanes adds up `piece` positions,
// whatever runs they belong to: runs that begin and end there are written at
// once, the others meet in a segmented scan over the workgroup's teams, and
// what runs over the workgroup's ends goes to two partial rows, which a second
// launch adds up.  Every workgroup has the same work however the splats are
// spread over the codes.  The splats' rows are read once, for both gradients.
//
// What bounds it, on an MI355X: the forward of a million splats x 128 floats
// over 16384 codes (8 MB of codebook, twice an XCD's L2) takes 120 us, 4.6 TB/s
// of codes read and rows written, 7.1 TB/s with the codebook's misses; the
// output's stores stream past the caches (165 us without).  Its backward: 49 us
// of sorting (two passes of 17 us, keys and histogram of 6 and 9, latency), 134 us
// of runs (rows in sorted order are gathers of 512 bytes: 5.4 TB/s), 11 us of
// joining.  262144 splats x 48 bf16 with scales, most on a few codes: 9 us
// forward, and in the backward six launches of 3 to 19 us, each a chain of
// dependent loads.  The gradient of the scales alone is bound by the launch of a
// wavefront a splat, most of whose lanes idle in narrow rows: a million splats x 3
// floats 180 us for 21 MB, x 128 floats 228 us for 550 MB.
#include <algorithm>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;

// ---- forward

// Each thread writes kUnroll vectors of 16 bytes of the output, taken as one
// array; block b starts at element b * kThreads * V * kUnroll.  div: the
// quotient of a 32-bit offset by D.
template <typename T, bool Rows, int kUnroll>
__global__ __launch_bounds__(kThreads) void lookup_fwd_kernel(
    LookupParams P, Divide div, const T* __restrict__ codebook,
    const float* __restrict__ scales, T* __restrict__ out) {
  constexpr int V = kVec<T>;
  const int64_t total = P.rows * P.D;
  const int64_t start = (int64_t)blockIdx.x * (kThreads * V * kUnroll);
  const int64_t row0 = start / P.D;
  const uint32_t skip = (uint32_t)(start - row0 * P.D);
  int64_t at[kUnroll], n[kUnroll];
  uint32_t d[kUnroll];
  int c[kUnroll];
  float s[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t i = (u * kThreads + threadIdx.x) * V;
    at[u] = start + i;
    const uint32_t q = div(skip + i);
    d[u] = skip + i - q * P.D;
    n[u] = row0 + q;
    const bool in = at[u] < total;
    c[u] = in ? P.codes.at(n[u], P.K) : kNoCode;
    s[u] = P.factor;
    if (scales && in) s[u] *= scales[n[u]];
  }
  vec_t<T> y[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const T* row = codebook + (int64_t)max(c[u], 0) * P.stride;
    if (Rows || d[u] + V <= (uint32_t)P.D) {
      y[u] = load_vec(row + d[u]);
    } else {
      // the vector goes on in the next rows
      uint32_t e = d[u];
      int64_t r = n[u];
      int k = c[u];
      float f = s[u];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float z = nan_for(k);
        if (k >= 0) z = to_float(codebook[(int64_t)k * P.stride + e]) * f;
        y[u][v] = static_cast<T>(z);
        if (++e == (uint32_t)P.D) {
          e = 0;
          ++r;
          if (v + 1 < V && r < P.rows) {
            k = P.codes.at(r, P.K);
            f = scales ? P.factor * scales[r] : P.factor;
          }
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (at[u] >= total) continue;
    if (Rows || d[u] + V <= (uint32_t)P.D)
#pragma unroll
      for (int v = 0; v < V; ++v)
        y[u][v] = static_cast<T>(c[u] >= 0 ? to_float(y[u][v]) * s[u] : nan_for(c[u]));
    if (at[u] + V <= total) {
      store_vec_stream(out + at[u], y[u]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (at[u] + v < total) out[at[u] + v] = y[u][v];
    }
  }
}

// ---- backward

// A team of TL lanes holds R vectors per lane of a row's columns from c0 on.
template <typename T, int TL, int R, bool Even>
struct Columns {
  static constexpr int V = kVec<T>;
  static constexpr int kWidth = TL * V * R;
  static constexpr int kTeams = kThreads / TL;
  static __device__ __forceinline__ int lane() { return threadIdx.x & (TL - 1); }
  static __device__ __forceinline__ int column(int c0, int r) { return c0 + (r * TL + lane()) * V; }
  template <bool Stream = false>
  static __device__ __forceinline__ void load(vec_t<T> (&x)[R], const T* row, int c0, int D) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      x[r] = load_part<T, Even, Stream>(row, column(c0, r), D, static_cast<T>(0.0f));
  }
  static __device__ __forceinline__ void store(T* row, int c0, int D, const float (&a)[R * V],
                                               float f) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      vec_t<T> o;
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = static_cast<T>(a[r * V + v] * f);
      if (column(c0, r) < D) store_part<T, Even>(row, column(c0, r), D, o);
    }
  }
  static __device__ __forceinline__ void load_sums(float (&a)[R * V], const float* row, int c0,
                                                   int D) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int k = column(c0, r) + v;
        a[r * V + v] = k < D ? row[k] : 0.0f;
      }
  }
  static __device__ __forceinline__ void store_sums(float* row, int c0, int D,
                                                    const float (&a)[R * V]) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int k = column(c0, r) + v;
        if (k < D) row[k] = a[r * V + v];
      }
  }
};

// Few splats.  A workgroup takes Q codes.  Its wavefronts each read a quarter of
// kRowsAtOnce splats' codes and list the splats of the workgroup's codes, in
// order; the rows listed for a code are shared out over the workgroup's teams,
// four on their way at a time, and the teams' sums are added in their order.
//
// Where one code's splats could be too many for a workgroup, blockIdx.z takes
// `span` splats, leaves its sums in partial[z][K][D], and lookup_scan_join_kernel
// adds those up in order.
constexpr int kRowsAtOnce = 2048;
constexpr int kQuarter = kRowsAtOnce / 4;

template <typename T, int TL, int R, int Q, bool Even>
__global__ __launch_bounds__(kThreads) void lookup_scan_kernel(
    LookupParams P, const T* __restrict__ grad, const T* __restrict__ codebook,
    const float* __restrict__ scales, T* __restrict__ g_codebook,
    float* __restrict__ g_scales, float* __restrict__ partial, int64_t span) {
  using C = Columns<T, TL, R, Even>;
  constexpr int V = C::V, kTeams = C::kTeams, kAhead = 4;
  __shared__ uint16_t lists[Q][4][kQuarter];
  __shared__ int counts[Q][4];
  __shared__ float sums[4][C::kWidth];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int team = threadIdx.x / TL;
  const int first = (int)blockIdx.x * Q;
  const int c0 = blockIdx.y * C::kWidth;
  const bool dots = g_scales != nullptr;
  float acc[Q][R * V];
#pragma unroll
  for (int q = 0; q < Q; ++q)
#pragma unroll
    for (int j = 0; j < R * V; ++j) acc[q][j] = 0.0f;
  const int64_t from_row = blockIdx.z * span, to_row = min(from_row + span, P.rows);
  for (int64_t base = from_row; base < to_row; base += kRowsAtOnce) {
    int mine[kQuarter / 64];
#pragma unroll
    for (int u = 0; u < kQuarter / 64; ++u) {
      const int64_t n = base + w * kQuarter + u * 64 + lane;
      mine[u] = n < to_row ? P.codes.at(n, P.K) : kNoCode;
      if (dots && first == 0 && n < to_row && mine[u] < 0) g_scales[n] = nan_for(mine[u]);
    }
    int found[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) found[q] = 0;
#pragma unroll
    for (int u = 0; u < kQuarter / 64; ++u) {
      const unsigned rel = (unsigned)(mine[u] - first);
      if (__ballot(rel < (unsigned)Q) == 0) continue;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const uint64_t hit = __ballot(rel == (unsigned)q);
        if (rel == (unsigned)q)
          lists[q][w][found[q] + __builtin_amdgcn_mbcnt_hi(
                                     (uint32_t)(hit >> 32),
                                     __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0))] =
              (uint16_t)(w * kQuarter + u * 64 + lane);
        found[q] += __popcll(hit);
      }
    }
    if (lane == 0)
#pragma unroll
      for (int q = 0; q < Q; ++q) counts[q][w] = found[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      // (the lists of the four wavefronts, one after another)
      const int e0 = counts[q][0], e1 = e0 + counts[q][1], e2 = e1 + counts[q][2],
                total = e2 + counts[q][3];
      if (total == 0) continue;
      vec_t<T> row[R];
      if (dots) C::load(row, codebook + (int64_t)(first + q) * P.stride, c0, P.D);
      // (every team makes the same number of turns: the sums of a row's
      // products run over whole teams)
      for (int i0 = 0; i0 < total; i0 += kAhead * kTeams) {
        int64_t n[kAhead];
        float s[kAhead];
        vec_t<T> g[kAhead][R];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int i = min(i0 + u * kTeams + team, total - 1);
          const int from = (i >= e0) + (i >= e1) + (i >= e2);
          n[u] = base + lists[q][from][i - (from == 0 ? 0 : from == 1 ? e0 : from == 2 ? e1 : e2)];
          s[u] = scales ? scales[n[u]] : 1.0f;
          C::load(g[u], grad + n[u] * P.D, c0, P.D);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          if (i0 + u * kTeams >= total) break;
          const bool here = i0 + u * kTeams + team < total;
          float dot = 0.0f;
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < V; ++v) {
              const float x = to_float(g[u][r][v]);
              if (here) acc[q][r * V + v] = __builtin_fmaf(x, s[u], acc[q][r * V + v]);
              if (dots) dot = __builtin_fmaf(x, to_float(row[r][v]), dot);
            }
          if (dots) {
            dot = team_sum<TL>(dot);
            if (here && C::lane() == 0) g_scales[n[u]] = dot * P.factor;
          }
        }
      }
    }
    __syncthreads();
  }
  if (g_codebook == nullptr) return;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    if (first + q >= P.K) return;
#pragma unroll
    for (int j = 0; j < R * V; ++j)
#pragma unroll
      for (int d = TL; d < 64; d <<= 1) acc[q][j] += __shfl_xor(acc[q][j], d, 64);
    if (lane < TL)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) sums[w][(r * TL + lane) * V + v] = acc[q][r * V + v];
    __syncthreads();
    if (threadIdx.x < TL) {
#pragma unroll
      for (int t = 1; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int v = 0; v < V; ++v)
            acc[q][r * V + v] += sums[t][(r * TL + lane) * V + v];
      if (partial)
        C::store_sums(partial + ((int64_t)blockIdx.z * P.K + first + q) * P.D, c0, P.D, acc[q]);
      else
        C::store(g_codebook + (int64_t)(first + q) * P.D, c0, P.D, acc[q], P.factor);
    }
    __syncthreads();
  }
}

// A value of the codebook's gradient per thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_scan_join_kernel(
    LookupParams P, const float* __restrict__ partial, int chunks, T* __restrict__ g_codebook) {
  const int64_t values = (int64_t)P.K * P.D, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= values) return;
  float a = 0.0f;
#pragma unroll 16
  for (int z = 0; z < chunks; ++z) a += partial[z * values + i];
  g_codebook[i] = static_cast<T>(a * P.factor);
}

// Keys of the sort (K for splats without a code: after all others), and zeros
// for the sort's control words and the codebook's gradient (zero_bytes of it,
// 16 at a time and the rest by bytes).
__global__ __launch_bounds__(kThreads) void lookup_keys_kernel(
    LookupParams P, uint32_t* __restrict__ keys, uint32_t* __restrict__ ctl,
    int64_t ctl_words, char* __restrict__ g_codebook, int64_t zero_bytes) {
  const int64_t step = (int64_t)gridDim.x * kThreads;
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t n = t; n < P.rows; n += step) {
    const int c = P.codes.at(n, P.K);
    keys[n] = c >= 0 ? (uint32_t)c : (uint32_t)P.K;
  }
  for (int64_t i = t; i < ctl_words; i += step) ctl[i] = 0;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int64_t i = t; i < zero_bytes / 16; i += step)
    __builtin_memcpy(g_codebook + 16 * i, &zero, 16);
  for (int64_t i = zero_bytes / 16 * 16 + t; i < zero_bytes; i += step) g_codebook[i] = 0;
}

// The sorted splats and the two partial rows of each workgroup's positions
// [b * span, (b + 1) * span): in[b] the end of a run that began before them, out[b]
// the part of a run that goes on after them.
constexpr uint32_t kNone = ~0u;
struct Sorted {
  const uint32_t* keys;
  const uint32_t* order;
  const uint32_t* err;  // the sort gave up: neither holds anything
  int piece, span, blocks;
  uint32_t* out_key;  // [blocks] the run that goes on after them, or kNone
  float* in;          // [blocks][D]
  float* out;
};

template <typename T, int TL, int R, bool Even>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 4 && R == 1 ? (Even ? 6 : 5) : 4))) void
lookup_runs_kernel(
    LookupParams P, Sorted S, const T* __restrict__ grad,
    const T* __restrict__ codebook, const float* __restrict__ scales,
    T* __restrict__ g_codebook, float* __restrict__ g_scales) {
  using C = Columns<T, TL, R, Even>;
  constexpr int V = C::V, kTeams = C::kTeams, kRows = R > 1 ? 2 : 4;
  __shared__ float open[kTeams][C::kWidth + 1];  // (+ 1: teams of one lane)
  __shared__ uint8_t ended[kTeams];
  const int team = threadIdx.x / TL, c0 = blockIdx.y * C::kWidth;
  const int64_t first = (int64_t)blockIdx.x * S.span;
  const int64_t last = min(first + S.span, P.rows);
  if (*S.err != 0) {
    if (g_scales)
      for (int64_t n = first + threadIdx.x; n < last; n += kThreads)
        g_scales[n] = __builtin_nanf("");
    return;
  }
  const int64_t a = min(first + (int64_t)team * S.piece, last);
  const int64_t b = min(a + S.piece, last);
  const bool dots = g_scales != nullptr;
  auto write = [&](uint32_t k, const float (&x)[R * V]) {
    if (k < (uint32_t)P.K) C::store(g_codebook + (int64_t)k * P.D, c0, P.D, x, P.factor);
  };
  float acc[R * V], head[R * V];
#pragma unroll
  for (int j = 0; j < R * V; ++j) acc[j] = head[j] = 0.0f;
  // The run that came in from the left, until it ends.
  const uint32_t before = a > 0 && a < b ? S.keys[a - 1] : kNone;
  bool coming = a < b && before == S.keys[a];
  const uint32_t head_key = before;
  bool head_ended = false, any_end = false;
  vec_t<T> now[R];
  uint32_t held = kNone;
  // (the next rows' codes and places are loaded while these rows are on their way)
  uint32_t key[kRows + 1], key_next[kRows];
  int n[kRows], n_next[kRows];
  auto look = [&](int64_t j0) {
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      key_next[u] = S.keys[min(j0 + u, P.rows - 1)];
      n_next[u] = (int)S.order[min(j0 + u, P.rows - 1)];
    }
  };
  if (a < b) look(a);
  for (int64_t j0 = a; j0 < b; j0 += kRows) {
    float s[kRows];
    vec_t<T> g[kRows][R], row[kRows][R];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      key[u] = key_next[u];
      n[u] = n_next[u];
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      s[u] = scales ? scales[n[u]] : 1.0f;
      C::template load<true>(g[u], grad + (int64_t)n[u] * P.D, c0, P.D);
    }
    look(j0 + kRows);
    key[kRows] = key_next[0];
    if (dots) {
      // (the codebook's row of each new run)
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (key[u] != held) {
          C::load(now, codebook + (int64_t)min(key[u], (uint32_t)P.K - 1) * P.stride, c0, P.D);
          held = key[u];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) row[u][r] = now[r];
      }
    }
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      if (j0 + u >= b) break;
      float dot = 0.0f;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float x = to_float(g[u][r][v]);
          acc[r * V + v] = __builtin_fmaf(x, s[u], acc[r * V + v]);
          if (dots) dot = __builtin_fmaf(x, to_float(row[u][r][v]), dot);
        }
      if (dots) {
        dot = team_sum<TL>(dot) * P.factor;
        if (C::lane() == 0)
          g_scales[n[u]] = key[u] < (uint32_t)P.K ? dot : nan_for(P.codes.at(n[u], P.K));
      }
      if (key[u] != key[u + 1] || j0 + u + 1 == P.rows) {  // the run ends
        any_end = true;
        if (coming) {
          coming = false;
          head_ended = true;
#pragma unroll
          for (int q = 0; q < R * V; ++q) head[q] = acc[q];
        } else {
          write(key[u], acc);
        }
#pragma unroll
        for (int q = 0; q < R * V; ++q) acc[q] = 0.0f;
      }
    }
  }
  if (g_codebook == nullptr) return;
  // Inclusive segmented scan of the teams' open sums: open[t] becomes the sum of
  // the run that goes on after team t, from the workgroup's first position on.
  auto column_of = [&](int r, int v) { return (r * TL + C::lane()) * V + v; };
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v) open[team][column_of(r, v)] = acc[r * V + v];
  if (C::lane() == 0) ended[team] = any_end;
  __syncthreads();
  bool seen = any_end;
  for (int d = 1; d < kTeams; d <<= 1) {
    const bool take = team >= d && !seen;
    const bool more = team >= d && ended[team - d];
    if (take)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v)
          acc[r * V + v] += open[team - d][column_of(r, v)];
    __syncthreads();
    if (take) {
      seen = more;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v) open[team][column_of(r, v)] = acc[r * V + v];
      if (C::lane() == 0) ended[team] = seen;
    }
    __syncthreads();
  }
  const uint32_t left = first > 0 ? S.keys[first - 1] : kNone;
  if (head_ended) {
    if (team > 0)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; ++v)
          head[r * V + v] += open[team - 1][column_of(r, v)];
    if (left == head_key) {
      C::store_sums(S.in + (int64_t)blockIdx.x * P.D, c0, P.D, head);
    } else {
      write(head_key, head);
    }
  }
  const uint32_t right = last < P.rows ? S.keys[last] : kNone;
  const uint32_t last_key = S.keys[last - 1];
  if (threadIdx.x == 0 && blockIdx.y == 0)
    S.out_key[blockIdx.x] = last_key == right ? last_key : kNone;
  if (team == kTeams - 1 && last_key == right)
    C::store_sums(S.out + (int64_t)blockIdx.x * P.D, c0, P.D, acc);
}

// One workgroup per workgroup of the launch above: where a run begins that goes
// on after its positions, that run's partial rows are added up (teams take
// every kTeams-th row, then the teams in order).  A sort that gave up makes
// the gradient NaN.
template <typename T, int TL, int R, bool Even>
__global__ __launch_bounds__(kThreads) void lookup_join_kernel(
    LookupParams P, Sorted S, T* __restrict__ g_codebook) {
  using C = Columns<T, TL, R, Even>;
  constexpr int V = C::V, kTeams = C::kTeams;
  __shared__ float sums[kTeams][C::kWidth + 1];
  __shared__ int ends[kThreads / 64];
  if (*S.err != 0) {
    const int64_t total = (int64_t)P.K * P.D;
    if (blockIdx.y == 0)
      for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total;
           i += (int64_t)gridDim.x * kThreads)
        g_codebook[i] = static_cast<T>(__builtin_nanf(""));
    return;
  }
  const int b = blockIdx.x, c0 = blockIdx.y * C::kWidth;
  const uint32_t k = S.out_key[b];
  if (k >= (uint32_t)P.K) return;  // (kNone, or the splats without a code)
  const int64_t first = (int64_t)b * S.span;
  if (first > 0 && S.keys[first] == k && S.keys[first - 1] == k) return;  // began before
  // the workgroup where the run ends: the first after b whose out_key is not k
  int end = b + 1;
  for (;; end += kThreads) {
    const int i = end + threadIdx.x;
    const uint64_t other = __ballot(i >= S.blocks || S.out_key[i] != k);
    if ((threadIdx.x & 63) == 0)
      ends[threadIdx.x >> 6] = other ? __builtin_ctzll(other) + (int)(threadIdx.x & ~63) : kThreads;
    __syncthreads();
    int e = kThreads;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) e = min(e, ends[w]);
    __syncthreads();
    if (e < kThreads) {
      end += e;
      break;
    }
  }
  const int team = threadIdx.x / TL;
  float acc[R * V], x[R * V];
#pragma unroll
  for (int j = 0; j < R * V; ++j) acc[j] = 0.0f;
  for (int i = b + team; i <= end; i += kTeams) {
    C::load_sums(x, (i < end ? S.out : S.in) + (int64_t)i * P.D, c0, P.D);
#pragma unroll
    for (int j = 0; j < R * V; ++j) acc[j] += x[j];
  }
  auto column_of = [&](int r, int v) { return (r * TL + C::lane()) * V + v; };
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v) sums[team][column_of(r, v)] = acc[r * V + v];
  __syncthreads();
  if (team != 0) return;
  for (int t = 1; t < kTeams; ++t)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[r * V + v] += sums[t][column_of(r, v)];
  C::store(g_codebook + (int64_t)k * P.D, c0, P.D, acc, P.factor);
}

// A wavefront per splat: the gradient of the scales where a row takes several
// workgroups, or where it is the only gradient.
template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_scales_kernel(
    LookupParams P, const T* __restrict__ grad, const T* __restrict__ codebook,
    float* __restrict__ g_scales) {
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (n >= P.rows) return;
  const int c = P.codes.at(n, P.K);
  float acc = 0.0f;
  if (c >= 0)
    for (int d = lane * V; d < P.D; d += 64 * V) {
      const vec_t<T> g = load_part<T>(grad + n * P.D, d, P.D, static_cast<T>(0.0f));
      const vec_t<T> x =
          load_part<T>(codebook + (int64_t)c * P.stride, d, P.D, static_cast<T>(0.0f));
#pragma unroll
      for (int v = 0; v < V; ++v) acc = __builtin_fmaf(to_float(g[v]), to_float(x[v]), acc);
    }
  acc = wave_sum(acc);
  if (lane == 0) g_scales[n] = c < 0 ? nan_for(c) : acc * P.factor;
}

// ---- host

// Lanes of a team and vectors of a lane for rows of D values: CALL(TL, R).
#define GS_WIDTHS(CALL)          \
  if (vecs <= 1) CALL(1, 1)      \
  if (vecs <= 2) CALL(2, 1)      \
  if (vecs <= 4) CALL(4, 1)      \
  if (vecs <= 8) CALL(8, 1)      \
  if (vecs <= 16) CALL(16, 1)    \
  if (vecs <= 32) CALL(32, 1)    \
  if (vecs <= 64) CALL(64, 1)    \
  CALL(64, 2)

int vec_of(const LookupParams& P) { return P.dtype == GSPLAT_F32 ? 4 : 8; }
int vecs_of(const LookupParams& P) { return (P.D + vec_of(P) - 1) / vec_of(P); }
int lanes_of(const LookupParams& P) {
  int tl = 1;
  while (tl < 64 && tl < vecs_of(P)) tl *= 2;
  return tl;
}

// Chunks of the splats that the scan takes, or 0: sorted.  The scan reads all codes
// once for each code (or four) of the codebook.  Kernels of both ways, rows of 64
// floats: 8192 splats and 256 codes 13 us against 28 sorted, 8192 x 4096 25 against
// 29, 4096 x 16384 27 against 28, 8192 x 16384 44 against 29, 16384 x 16 43 against
// 24; the sort's five to six launches cost the host 20 us more.
// Chunks bound what one code that many splats share takes: where a chunk's splats
// are all of one code, kMostTurns turns of a workgroup's loads (8192 splats x 700 in
// bf16, 64 codes, 80% of the splats on eight of them: 144 us of kernels forward and
// backward as one chunk, 36 in eight).  Their sums cost a uniform choice of codes
// time: 16 MB of them 20 us.
// Narrow rows, of which a workgroup takes 256 and more at once, go this way up to 64K
// splats (kernels forward and backward, 65536 x 3 floats of 64 codes 17 us and 32
// sorted, 16384 of 512 codes 22 and 36, 32768 x 16 of 512 codes 26 and 32; at 2^25
// splats x codes 39 to 56 and 30 to 41).
// Codebooks of 2^26 codes are sorted whatever the splats: four codes a workgroup are
// as many threads as a launch does not have.
constexpr int kMostTurns = 64;
int chunks_of(const LookupParams& P) {
  const int64_t work = P.rows * P.K;
  if (P.K >= 1 << 26) return 0;
  if (P.rows <= 8192 ? work > int64_t(1) << 26
                     : vecs_of(P) > 4 || P.rows > 65536 || work > int64_t(1) << 24)
    return 0;
  // (sums of 8 MB at most)
  const int64_t limit = std::clamp<int64_t>((int64_t(1) << 21) / ((int64_t)P.K * P.D), 1, 64);
  const int64_t most = kMostTurns * 4 * (kThreads / lanes_of(P));  // splats of a chunk
  const int64_t chunks = std::max<int64_t>(1, (P.rows + most - 1) / most);
  if (P.rows > 8192) {
    const int64_t wide = std::max(chunks, (P.rows + kRowsAtOnce - 1) / kRowsAtOnce);
    return wide <= limit ? (int)wide : 0;
  }
  // (more than the limit: larger chunks, up to four times, where a workgroup has one
  // code; else sorted: 4096 splats x 700 in bf16, 80% of them on eight of 8192
  // codes, 337 us a pass as one chunk and 63 sorted)
  return chunks <= (P.K >= 4096 ? 1 : 4) * limit ? (int)std::min(chunks, limit) : 0;
}

struct Layout {
  int chunks;  // of the one-launch way, or 0: sorted
  RadixPlan sort;
  int piece, span, blocks;
  size_t ctl, buffers, keys, sorted, order, out_key, in, out, total;
};

Layout layout(const LookupParams& P) {
  Layout L{};
  if (P.rows == 0) return L;  // (zeros)
  L.chunks = chunks_of(P);
  if (L.chunks > 1) L.total = (size_t)L.chunks * P.K * P.D * 4;
  if (L.chunks > 0) return L;
  int bits = 1;
  while (bits < 32 && (int64_t(1) << bits) <= P.K) ++bits;
  L.sort = radix_plan(P.rows, 1, 0, bits);
  // Positions per team: 4 to 64.  Eight at a time keep more loads on their way
  // than four once there are 512 workgroups, and 8192 workgroups of short
  // pieces end more evenly than fewer of long ones (a million splats x 128
  // values: 209 us with 2048 workgroups, 179 with 8192).
  const int tl = lanes_of(P);
  L.piece = 4;
  while (L.piece < 64 &&
         P.rows * tl > (int64_t)L.piece * kThreads * (L.piece < 8 ? 512 : 8192))
    L.piece *= 2;
  L.span = L.piece * (kThreads / tl);
  L.blocks = (int)((P.rows + L.span - 1) / L.span);
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
  L.out_key = take((size_t)L.blocks * 4);
  L.in = take((size_t)L.blocks * P.D * 4);
  L.out = take((size_t)L.blocks * P.D * 4);
  L.total = off;
  return L;
}

template <typename T>
int forward_of(const LookupParams& P, const void* codebook, const float* scales,
               void* out, hipStream_t stream) {
  const int64_t vecs = (P.rows * P.D + kVec<T> - 1) / kVec<T>;
  const T* book = static_cast<const T*>(codebook);
  T* o = static_cast<T*>(out);
  const Divide div((uint32_t)P.D);
  // Four vectors a thread, with as many chains of loads on their way, where the
  // codebook does not fit an XCD's 4 MB of L2 (a million splats x 128 floats over
  // 16384 codes: 120 us against 133); one where it does (over 4096 codes 82
  // against 88, 64K x 11 4.2 against 7.8).  A launch
  // has fewer than 2^32 threads: outputs of 32 GiB and more take four too (and those
  // of 256 GiB, which no device holds, are refused by launch_traced).
  const bool missing = (int64_t)P.K * P.D * sizeof(T) > (int64_t(4) << 20) &&
                       vecs >= (int64_t)kThreads * 4 * 1024;
  const bool four = missing || vecs >= int64_t(1) << 31;
#define GS_LOOKUP(ROWS, U)                                                      \
  launch_traced("lookup_fwd_kernel", (lookup_fwd_kernel<T, ROWS, U>),           \
                dim3((unsigned)std::min<int64_t>((vecs + kThreads * U - 1) / (kThreads * U), ~0u)), \
                dim3(kThreads), 0, stream, P, div, book, scales, o)
  const bool rows = P.D % kVec<T> == 0;
  if (rows && four) GS_LOOKUP(true, 4);
  else if (rows) GS_LOOKUP(true, 1);
  else if (four) GS_LOOKUP(false, 4);
  else GS_LOOKUP(false, 1);
#undef GS_LOOKUP
  return check_launch("lookup_fwd_kernel");
}

template <typename T, bool Even>
int backward_of(const LookupParams& P, const void* grad_out, const void* codebook,
                const float* scales, void* g_codebook, float* g_scales,
                void* workspace, hipStream_t stream) {
  const T* grad = static_cast<const T*>(grad_out);
  const T* book = static_cast<const T*>(codebook);
  T* g_book = static_cast<T*>(g_codebook);
  const int vecs = vecs_of(P);
  // (a row of up to 128 vectors is one team's)
  const unsigned tiles = (unsigned)((vecs + 127) / 128);
  if (g_scales && P.rows > 0 && (tiles > 1 || !g_book)) {
    // (a loop over the rows in the kernel instead: 1M x 3 floats 188 us, 180 so)
    const int rc = in_launches(P.rows, kMostBlocks * 4, [&](int64_t n, int64_t rows) {
      LookupParams Q = P;
      Q.rows = rows;
      Q.codes = P.codes.from(n);
      launch_traced("lookup_scales_kernel", (lookup_scales_kernel<T>),
                    dim3((unsigned)((rows + 3) / 4)), dim3(kThreads), 0, stream, Q,
                    grad + n * P.D, book, g_scales + n);
      return check_launch("lookup_scales_kernel");
    });
    if (rc) return rc;
    g_scales = nullptr;
  }
  if (!g_book) return GSPLAT_OK;
  const int64_t zero_bytes = (int64_t)P.K * P.D * sizeof(T);
  auto prepare = [&](uint32_t* keys, uint32_t* ctl, int64_t ctl_words) {
    const int64_t most = std::max(P.rows, zero_bytes / 16) / kThreads + 1;
    launch_traced("lookup_keys_kernel", lookup_keys_kernel,
                  dim3((unsigned)std::min<int64_t>(most, 2048)), dim3(kThreads), 0,
                  stream, P, keys, ctl, ctl_words, reinterpret_cast<char*>(g_book),
                  zero_bytes);
    return check_launch("lookup_keys_kernel");
  };
  if (P.rows == 0) return prepare(nullptr, nullptr, 0);
  const Layout L = layout(P);
  if (L.chunks > 0) {
    float* partial = L.chunks > 1 ? static_cast<float*>(workspace) : nullptr;
    const int64_t span = (P.rows + L.chunks - 1) / L.chunks;
    // (four codes a workgroup where that leaves 1024 of them: 1024 splats x 64,
    // 16384 codes 16 us against 25 with one, 4096 codes 8 against 9.  Not for the
    // chunks of wide rows: 80% of 8192 splats x 700 in bf16 on eight of 1024 codes
    // 175 us a pass with four, 72 with one)
    const bool four = P.K >= 4096 || (vecs <= 4 && P.K * L.chunks >= 4096);
#define GS_SCAN_OF(TL, R, Q)                                                      \
    launch_traced("lookup_scan_kernel", (lookup_scan_kernel<T, TL, R, Q, Even>),  \
                  dim3((unsigned)((P.K + Q - 1) / Q), tiles, (unsigned)L.chunks), \
                  dim3(kThreads), 0, stream, P, grad, book, scales, g_book,       \
                  g_scales, partial, span)
#define GS_SCAN(TL, R)                                                          \
  {                                                                             \
    if (four) GS_SCAN_OF(TL, R, 4);                                             \
    else GS_SCAN_OF(TL, R, 1);                                                  \
    const int rc = check_launch("lookup_scan_kernel");                          \
    if (rc || !partial) return rc;                                              \
    launch_traced("lookup_scan_join_kernel", (lookup_scan_join_kernel<T>),      \
                  dim3((unsigned)(((int64_t)P.K * P.D + kThreads - 1) / kThreads)), \
                  dim3(kThreads), 0, stream, P, partial, L.chunks, g_book);     \
    return check_launch("lookup_scan_join_kernel");                             \
  }
    GS_WIDTHS(GS_SCAN)
#undef GS_SCAN
#undef GS_SCAN_OF
  }
  char* w = static_cast<char*>(workspace);
  auto* keys = reinterpret_cast<uint32_t*>(w + L.keys);
  auto* sorted = reinterpret_cast<uint32_t*>(w + L.sorted);
  auto* order = reinterpret_cast<uint32_t*>(w + L.order);
  const RadixCtl C = radix_ctl_at(L.sort, w + L.ctl);
  int rc = prepare(keys, C.ghist, (int64_t)radix_ctl_bytes(L.sort) / 4);
  if (!rc) rc = radix_global_hist(L.sort, C, keys, nullptr, stream);
  if (!rc)
    rc = radix_passes(L.sort, C, w + L.buffers, keys, nullptr, nullptr, sorted,
                      order, stream);
  if (rc) return rc;
  const Sorted S{sorted, order, C.err, L.piece, L.span, L.blocks,
                 reinterpret_cast<uint32_t*>(w + L.out_key),
                 reinterpret_cast<float*>(w + L.in), reinterpret_cast<float*>(w + L.out)};
  const dim3 grid((unsigned)L.blocks, tiles);
#define GS_RUNS(TL, R)                                                          \
  {                                                                             \
    launch_traced("lookup_runs_kernel", (lookup_runs_kernel<T, TL, R, Even>), grid,   \
                  dim3(kThreads), 0, stream, P, S, grad, book, scales, g_book,  \
                  g_scales);                                                    \
    rc = check_launch("lookup_runs_kernel");                                    \
    if (rc) return rc;                                                          \
    launch_traced("lookup_join_kernel", (lookup_join_kernel<T, TL, R, Even>), grid,   \
                  dim3(kThreads), 0, stream, P, S, g_book);                     \
    return check_launch("lookup_join_kernel");                                  \
  }
  GS_WIDTHS(GS_RUNS)
#undef GS_RUNS
}
#undef GS_WIDTHS

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
  const bool even = P.D % vec_of(P) == 0;
  auto f = P.dtype == GSPLAT_F32    ? (even ? backward_of<float, true> : backward_of<float, false>)
           : P.dtype == GSPLAT_BF16 ? (even ? backward_of<__bf16, true> : backward_of<__bf16, false>)
                                    : (even ? backward_of<_Float16, true> : backward_of<_Float16, false>);
  return f(P, grad_out, codebook, scales, g_codebook, g_scales, workspace, stream);
}

}  // namespace gs
