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
//
// Sorting: few choices are ranked against all others in one launch; more of up to
// kMostBins codes are counted by code in chunks, the counts scanned over the
// chunks, and each chunk's choices ranked and placed; the rest goes through the
// radix sort.
//
// Rows: a thread has 16 bytes of a row, taken as one array of whole vectors per
// row (the last one of a row that is not whole vectors overlaps the one before:
// both hold the same values there); the rows' and weights' gradients together, a
// team of lanes a row.  All loads of a thread are issued before the first is
// looked at; places past the last code are looked up by those few threads alone.
//
// What bounds it, on an MI355X: rows are HBM's, gathers of whole rows; stores go
// past the caches.  A million rows of 128 floats by code 195 us (5.5 TB/s; 208
// through the caches), 262144 splats x 4 rows of 128 bfloat16 back 62 us and 139 for
// both gradients (5.4 and 4.3 TB/s, 6.8 with a splat's row read for each of its
// codes).  Sorting is latency: 512 choices 5 us, 524288 of 256 codes 20 (three
// launches; by radix 45), a million of 16384 codes 62 (five launches, 16 us of them
// the places' scattered stores).
#include <algorithm>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;

// ---- sorting

// What a choice is sorted by: its code, or K.
__device__ __forceinline__ uint32_t key_of(const GroupParams& P, int64_t i) {
  const int c = P.codes.at(i, P.K);
  return c >= 0 ? (uint32_t)c : (uint32_t)P.K;
}

// Few choices: an item is a choice, whose place is the number of choices before it
// in the order, or a code, whose start is the number of choices of lower codes.
// Four lanes an item compare it with a quarter of the choices each, held in LDS
// as (key, index) in one word.
constexpr int kFew = 2048, kFewBits = 11;

__global__ __launch_bounds__(kThreads) void group_few_kernel(GroupParams P,
                                                             int32_t* __restrict__ order,
                                                             int32_t* __restrict__ places,
                                                             int32_t* __restrict__ starts) {
  __shared__ __attribute__((aligned(16))) uint32_t words[kFew];
  const int N = (int)P.choices, padded = (N + 15) / 16 * 16;
  for (int i = threadIdx.x; i < padded; i += kThreads)
    words[i] = i < N ? key_of(P, i) << kFewBits | (uint32_t)i : ~0u;
  __syncthreads();
  const int item = blockIdx.x * (kThreads / 4) + (threadIdx.x >> 2), part = threadIdx.x & 3;
  const bool choice = item < N;
  const uint32_t mine = choice ? words[item] : (uint32_t)min(item - N, P.K) << kFewBits;
  int before = 0;
  for (int i = 4 * part; i < padded; i += 16) {
    const uint4 w = *reinterpret_cast<const uint4*>(words + i);
    before += (w.x < mine) + (w.y < mine) + (w.z < mine) + (w.w < mine);
  }
  before = (int)team_reduce<4>((uint32_t)before, [](uint32_t x, uint32_t y) { return x + y; });
  if (part != 0) return;
  if (choice) {
    order[before] = item;
    places[item] = mine >> kFewBits < (uint32_t)P.K ? before : P.codes.at(item, P.K);
  } else if (item - N <= P.K) {
    starts[item - N] = before;
  }
}

// More choices, up to kMostBins codes: bins are the codes and K.
constexpr int kMostBins = 2048;

// counts[chunk][bin] of `rounds` * kThreads choices.
__global__ __launch_bounds__(kThreads) void group_count_kernel(GroupParams P, int rounds,
                                                               uint32_t* __restrict__ counts) {
  __shared__ uint32_t bins[kMostBins];
  for (int k = threadIdx.x; k <= P.K; k += kThreads) bins[k] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * rounds * kThreads;
#pragma unroll 4
  for (int r = 0; r < rounds; ++r) {
    const int64_t i = first + r * kThreads + threadIdx.x;
    if (i < P.choices) atomicAdd(&bins[key_of(P, i)], 1u);
  }
  __syncthreads();
  for (int k = threadIdx.x; k <= P.K; k += kThreads)
    counts[(int64_t)blockIdx.x * (P.K + 1) + k] = bins[k];
}

// Each bin's counts to the sums of the chunks before, and its total.  A workgroup
// has 16 bins; 64 threads a bin take a part of the chunks each.
constexpr int kScanParts = 64;
__global__ __launch_bounds__(16 * kScanParts) void group_scan_kernel(GroupParams P, int chunks,
                                                                     uint32_t* __restrict__ counts,
                                                                     uint32_t* __restrict__ totals) {
  __shared__ uint32_t sums[kScanParts][17];
  const int lane = threadIdx.x & 15, part = threadIdx.x >> 4;
  const int bin = blockIdx.x * 16 + lane, bins = P.K + 1, safe = min(bin, bins - 1);
  const int span = (chunks + kScanParts - 1) / kScanParts;
  const int from = min(part * span, chunks), to = min(from + span, chunks);
  uint32_t a = 0;
#pragma unroll 4
  for (int c = from; c < to; ++c) a += counts[(int64_t)c * bins + safe];
  sums[part][lane] = a;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll 16
  for (int q = 0; q < kScanParts; ++q) {
    const uint32_t n = sums[q][lane];
    if (q < part) before += n;
    total += n;
  }
  if (bin >= bins) return;
  if (part == 0) totals[bin] = total;
#pragma unroll 4
  for (int c = from; c < to; ++c) {
    const uint32_t n = counts[(int64_t)c * bins + bin];
    counts[(int64_t)c * bins + bin] = before;
    before += n;
  }
}

// A chunk's choices ranked: a wavefront has consecutive ones, 64 at a time; lanes
// of the same key are found bit by bit, the first of them counts them all.
template <int kRounds>
__global__ __launch_bounds__(kThreads) void group_place_kernel(
    GroupParams P, int bits, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, int32_t* __restrict__ order,
    int32_t* __restrict__ places, int32_t* __restrict__ starts) {
  __shared__ uint32_t bins[4][kMostBins];
  __shared__ uint32_t sums[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n_bins = P.K + 1;
  for (int k = lane; k < n_bins; k += 64) bins[w][k] = 0;
  __syncthreads();
  const int64_t first = ((int64_t)blockIdx.x * 4 + w) * kRounds * 64;
  uint32_t key[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * 64 + lane;
    key[r] = i < P.choices ? key_of(P, i) : ~0u;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool in = key[r] != ~0u;
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const bool set = key[r] >> b & 1;
      const uint64_t ones = __ballot(set);
      same &= set ? ones : ~ones;
    }
    const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32),
                                                __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
    uint32_t before = 0;
    if (in && below == 0) before = atomicAdd(&bins[w][key[r]], (uint32_t)__popcll(same));
    before = __shfl(before, in ? __builtin_ctzll(same) : 0, 64);
    rank[r] = before + below;
  }
  __syncthreads();
  // Where each bin begins: the bins before it (a thread has 8 of them), the chunks
  // before this one, the wavefronts before.
  uint32_t mine[kMostBins / kThreads], all = 0;
#pragma unroll
  for (int q = 0; q < kMostBins / kThreads; ++q) {
    const int k = threadIdx.x * (kMostBins / kThreads) + q;
    mine[q] = k < n_bins ? totals[k] : 0;
    all += mine[q];
  }
  uint32_t before = all;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = __shfl_up(before, d, 64);
    if (lane >= d) before += up;
  }
  if (lane == 63) sums[w] = before;
  __syncthreads();
  before -= all;
  for (int u = 0; u < w; ++u) before += sums[u];
#pragma unroll
  for (int q = 0; q < kMostBins / kThreads; ++q) {
    const int k = threadIdx.x * (kMostBins / kThreads) + q;
    if (k < n_bins) {
      if (blockIdx.x == 0) starts[k] = (int32_t)before;
      uint32_t at = before + counts[(int64_t)blockIdx.x * n_bins + k];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t n = bins[u][k];
        bins[u][k] = at;
        at += n;
      }
    }
    before += mine[q];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = first + r * 64 + lane;
    if (i >= P.choices) continue;
    const uint32_t place = bins[w][key[r]] + rank[r];
    if (place >= P.choices) continue;  // (codes that changed between the launches)
    order[place] = (int32_t)i;
    places[i] = key[r] < (uint32_t)P.K ? (int32_t)place : P.codes.at(i, P.K);
  }
}

__global__ __launch_bounds__(kThreads) void group_keys_kernel(
    GroupParams P, uint32_t* __restrict__ keys, uint32_t* __restrict__ ctl,
    int64_t ctl_words) {
  const int64_t step = (int64_t)gridDim.x * kThreads;
  const int64_t t = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t i = t; i < P.choices; i += step) {
    keys[i] = key_of(P, i);
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

// How choices are sorted, us of a call.  Few: one launch, 512 choices 5, 2048 12; 4096
// would take 23, counted 13.  Counted, as long as a workgroup's LDS holds a bin a
// wavefront and code, and by radix: 2049 choices of 2047 codes 16 and 18, 16384 of 1024
// codes 15 and 22, 262144 of 64 codes 14 and 42, of 2047 codes 20 and 42 (there are twice
// as many counts as choices then), 524288 of 256 codes 20 and 48, 2 million of 2047 codes
// 60 and 81, 4 million of 256 codes 54 and 127.
enum class Way { kFew, kCounted, kRadix };
Way way_of(const GroupParams& P) {
  if (P.choices <= kFew && P.K <= 16384) return Way::kFew;
  if (P.choices <= 1 << 25 && P.K < kMostBins) return Way::kCounted;
  return Way::kRadix;
}
// Choices of a chunk over kThreads: small ones while there are less of them than
// compute units (524288 choices: 31 us in chunks of 4096, 25 of 2048).
int rounds_of(const GroupParams& P) { return P.choices <= 1 << 18 ? 4 : P.choices <= 1 << 20 ? 8 : 16; }

struct SortLayout {
  RadixPlan sort;
  int chunks;
  size_t ctl, buffers, keys, sorted, totals, counts, total;
};

SortLayout sort_layout(const GroupParams& P) {
  SortLayout L{};
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off += align_up(bytes, 256);
    return at;
  };
  const Way way = way_of(P);
  if (way == Way::kCounted) {
    const int64_t chunk = (int64_t)rounds_of(P) * kThreads;
    L.chunks = (int)((P.choices + chunk - 1) / chunk);
    L.totals = take((size_t)(P.K + 1) * 4);
    L.counts = take((size_t)L.chunks * (P.K + 1) * 4);
  } else if (way == Way::kRadix && P.choices > 0) {
    int bits = 1;
    while (bits < 32 && (int64_t(1) << bits) <= P.K) ++bits;
    L.sort = radix_plan(P.choices, 1, 0, bits);
    L.ctl = take(radix_ctl_bytes(L.sort));
    L.buffers = take(L.sort.buffer_bytes);
    L.keys = take((size_t)P.choices * 4);
    L.sorted = take((size_t)P.choices * 4);
  }
  L.total = off;
  return L;
}

// ---- rows

// What a place says of its choice: 0 a row, else kNoCode or kBadCode.
__device__ __forceinline__ int state_of(int place, int64_t rows) {
  if (place >= 0 && place < rows) return 0;
  return place == kNoCode ? kNoCode : kBadCode;
}

// The choice at place j as order[j] has it: 0 a row, else kNoCode or kBadCode.  The
// first `named` places have codes, the others are few.
__device__ __forceinline__ int state_at(int choice, int64_t j, int64_t all, int64_t named,
                                        const int32_t* places) {
  if ((uint32_t)choice >= (uint32_t)all) return kBadCode;
  if (j < named) return 0;
  return places[choice] == kNoCode ? kNoCode : kBadCode;
}
// (a row, whatever the choice is)
__device__ __forceinline__ uint32_t safe_choice(int choice, int64_t all) {
  return (uint32_t)choice < (uint32_t)all ? choice : 0;
}

// Rows as vectors: thread t of a launch's block b has vectors b * kThreads * U +
// u * kThreads + t of all, counted row by row.
struct Vectors {
  Divide per_row;   // vectors of a row
  int64_t all, begin;  // of the rows; the launch's first block
};
template <typename T>
Vectors vectors_of(int64_t rows, int D) {
  const uint32_t n = (uint32_t)((D + kVec<T> - 1) / kVec<T>);
  return Vectors{Divide(n), rows * n, 0};
}
struct At {
  int64_t row;
  int d;    // the first of its values
  bool in;
};
template <int U>
__device__ __forceinline__ void at_of(const Vectors& X, int D, int V, At (&at)[U]) {
  const int64_t start = (X.begin + blockIdx.x) * (kThreads * U);
  const int64_t row0 = start / X.per_row.d;
  const uint32_t skip = (uint32_t)(start - row0 * X.per_row.d);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = skip + u * kThreads + threadIdx.x, q = X.per_row(i);
    const int d = (int)(i - q * X.per_row.d) * V;
    at[u] = At{row0 + q, D >= V ? min(d, D - V) : d, start + u * kThreads + threadIdx.x < X.all};
  }
}
// (a row of less than a vector is read and written by elements)
template <typename T>
__device__ __forceinline__ vec_t<T> load_at(const T* row, int d, int D) {
  return D >= kVec<T> ? load_vec(row + d) : load_part(row, d, D, static_cast<T>(0.0f));
}
template <typename T>
__device__ __forceinline__ void store_at(T* row, int d, int D, vec_t<T> v) {
  if (D >= kVec<T>) store_vec_stream(row + d, v);
  else store_part(row, d, D, v);
}

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void rows_by_code_kernel(
    RowsParams P, Vectors X, Divide choices, const T* __restrict__ rows,
    const int32_t* __restrict__ order, const int32_t* __restrict__ places,
    const int32_t* __restrict__ named, const float* __restrict__ weights,
    T* __restrict__ out) {
  constexpr int V = kVec<T>;
  const int64_t all = P.splats * P.choices, codes = *named;
  At at[U];
  at_of<U>(X, P.D, V, at);
  int i[U];
#pragma unroll
  for (int u = 0; u < U; ++u) i[u] = order[min(at[u].row, all - 1)];
  vec_t<T> y[U];
  float w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t choice = safe_choice(i[u], all);
    y[u] = load_at(rows + choices(choice) * P.stride, at[u].d, P.D);
    w[u] = 1.0f;
    if (weights) w[u] = weights[choice];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!at[u].in) continue;
    const int state = state_at(i[u], at[u].row, all, codes, places);
    if (weights)
#pragma unroll
      for (int v = 0; v < V; ++v) y[u][v] = static_cast<T>(w[u] * to_float(y[u][v]));
    if (state != 0)
#pragma unroll
      for (int v = 0; v < V; ++v) y[u][v] = static_cast<T>(nan_for(state));
    store_at(out + at[u].row * P.D, at[u].d, P.D, y[u]);
  }
}

// C choices at a time, U vectors a thread.
template <typename T, int C, int U>
__global__ __launch_bounds__(kThreads) void rows_from_codes_kernel(
    RowsParams P, Vectors X, const T* __restrict__ rows, const int32_t* __restrict__ places,
    const float* __restrict__ weights, T* __restrict__ out) {
  constexpr int V = kVec<T>;
  const int64_t all = P.splats * P.choices;
  At at[U];
  at_of<U>(X, P.D, V, at);
  float a[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int v = 0; v < V; ++v) a[u][v] = 0.0f;
  for (int s0 = 0; s0 < P.choices; s0 += C) {
    int place[U][C];
    float w[U][C];
    vec_t<T> y[U][C];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < C; ++s) {
        const bool in = at[u].in && (C == 1 || s0 + s < P.choices);
        const int64_t i = in ? at[u].row * P.choices + s0 + s : 0;
        place[u][s] = places[i];
        w[u][s] = 1.0f;
        if (weights) w[u][s] = weights[i];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < C; ++s) {
        const bool in = at[u].in && (C == 1 || s0 + s < P.choices);
        const int state = in ? state_of(place[u][s], all) : kNoCode;
        y[u][s] = load_at(rows + (state == 0 ? place[u][s] : 0) * P.stride, at[u].d, P.D);
        place[u][s] = state;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int s = 0; s < C; ++s)
#pragma unroll
        for (int v = 0; v < V; ++v)
          a[u][v] = place[u][s] == 0 ? __builtin_fmaf(w[u][s], to_float(y[u][s][v]), a[u][v])
                                     : a[u][v] + nan_for(place[u][s]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!at[u].in) continue;
    vec_t<T> y;
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = static_cast<T>(a[u][v]);
    store_at(out + at[u].row * P.D, at[u].d, P.D, y);
  }
}

// Both gradients: a team of TL lanes has a place's row, kAhead of them at a time.
template <typename T, int TL, bool Whole>
__global__ __launch_bounds__(kThreads) void rows_from_bwd_kernel(
    RowsParams P, Divide choices, int64_t begin, const T* __restrict__ grad,
    const T* __restrict__ rows, const int32_t* __restrict__ order,
    const int32_t* __restrict__ places, const int32_t* __restrict__ named,
    const float* __restrict__ weights, T* __restrict__ g_rows, float* __restrict__ g_weights) {
  constexpr int V = kVec<T>, kTeams = kThreads / TL, kAhead = 4;
  const int team = threadIdx.x / TL, lane = threadIdx.x % TL;
  const int64_t all = P.splats * P.choices, codes = *named;
  const int64_t j0 = (begin + blockIdx.x) * (kTeams * kAhead) + team;
  int i[kAhead], state[kAhead];
  int64_t n[kAhead];
  float w[kAhead], dot[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) i[u] = order[min(j0 + u * kTeams, all - 1)];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const uint32_t choice = safe_choice(i[u], all);
    n[u] = choices(choice);
    w[u] = weights[choice];
    dot[u] = 0.0f;
  }
#pragma unroll
  for (int u = 0; u < kAhead; ++u) state[u] = state_at(i[u], j0 + u * kTeams, all, codes, places);
  for (int d = lane * V; d < P.D; d += TL * V) {
    vec_t<T> g[kAhead], y[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t j = min(j0 + u * kTeams, all - 1);
      g[u] = load_part<T, Whole>(grad + n[u] * P.D, d, P.D, static_cast<T>(0.0f));
      y[u] = load_part<T, Whole, true>(rows + j * P.stride, d, P.D, static_cast<T>(0.0f));
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float x = to_float(g[u][v]);
        dot[u] = __builtin_fmaf(x, to_float(y[u][v]), dot[u]);
        g[u][v] = static_cast<T>(state[u] != 0 ? nan_for(state[u]) : w[u] * x);
      }
      if (g_rows && j0 + u * kTeams < all)
        store_part<T, Whole, true>(g_rows + (j0 + u * kTeams) * P.D, d, P.D, g[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const float sum = team_sum<TL>(dot[u]);
    const int64_t j = j0 + u * kTeams;
    if (lane != 0 || j >= all) continue;
    if ((uint32_t)i[u] < (uint32_t)all) g_weights[i[u]] = state[u] != 0 ? nan_for(state[u]) : sum;
  }
}

// ---- host

template <typename T>
int by_code_of(const RowsParams& P, const void* rows, const int32_t* order,
               const int32_t* places, const int32_t* named, const float* weights, void* out,
               hipStream_t stream) {
  Vectors X = vectors_of<T>(P.splats * P.choices, P.D);
  constexpr int U = 4;
  return in_launches((X.all + kThreads * U - 1) / (kThreads * U), kMostBlocks,
                     [&](int64_t first, int64_t blocks) {
    X.begin = first;
    launch_traced("rows_by_code_kernel", (rows_by_code_kernel<T, U>), dim3((unsigned)blocks),
                  dim3(kThreads), 0, stream, P, X, Divide((uint32_t)P.choices),
                  static_cast<const T*>(rows), order, places, named, weights,
                  static_cast<T*>(out));
    return check_launch("rows_by_code_kernel");
  });
}

template <typename T>
int from_codes_of(const RowsParams& P, const void* rows, const int32_t* places,
                  const float* weights, void* out, hipStream_t stream) {
  Vectors X = vectors_of<T>(P.splats, P.D);
  auto run = [&](auto kernel, int U) {
    return in_launches((X.all + kThreads * U - 1) / (kThreads * U), kMostBlocks,
                       [&](int64_t first, int64_t blocks) {
      X.begin = first;
      launch_traced("rows_from_codes_kernel", kernel, dim3((unsigned)blocks), dim3(kThreads), 0,
                    stream, P, X, static_cast<const T*>(rows), places, weights,
                    static_cast<T*>(out));
      return check_launch("rows_from_codes_kernel");
    });
  };
  if (P.choices == 1) return run(rows_from_codes_kernel<T, 1, 4>, 4);
  if (P.choices == 2) return run(rows_from_codes_kernel<T, 2, 2>, 2);
  return run(rows_from_codes_kernel<T, 4, 1>, 1);
}

template <typename T>
int from_codes_bwd_of(const RowsParams& P, const void* grad, const void* rows,
                      const int32_t* order, const int32_t* places, const int32_t* named,
                      const float* weights, void* g_rows, float* g_weights,
                      hipStream_t stream) {
  if (!g_weights) {
    RowsParams Q = P;
    Q.stride = P.D;
    return by_code_of<T>(Q, grad, order, places, named, weights, g_rows, stream);
  }
  const int vecs = (P.D + kVec<T> - 1) / kVec<T>;
  const int64_t all = P.splats * P.choices;
  auto run = [&](auto kernel, int lanes) {
    const int64_t rows_of_block = kThreads / lanes * 4;
    return in_launches((all + rows_of_block - 1) / rows_of_block, kMostBlocks,
                       [&](int64_t first, int64_t blocks) {
      launch_traced("rows_from_bwd_kernel", kernel, dim3((unsigned)blocks), dim3(kThreads), 0,
                    stream, P, Divide((uint32_t)P.choices), first, static_cast<const T*>(grad),
                    static_cast<const T*>(rows), order, places, named, weights,
                    static_cast<T*>(g_rows), g_weights);
      return check_launch("rows_from_bwd_kernel");
    });
  };
  const bool whole = P.D % kVec<T> == 0;
#define GS_LANES(TL) \
  if (vecs <= TL || TL == 64) \
    return whole ? run(rows_from_bwd_kernel<T, TL, true>, TL) : run(rows_from_bwd_kernel<T, TL, false>, TL);
  GS_LANES(1) GS_LANES(2) GS_LANES(4) GS_LANES(8) GS_LANES(16) GS_LANES(32) GS_LANES(64)
#undef GS_LANES
}

}  // namespace

size_t group_workspace_bytes(const GroupParams& P) { return sort_layout(P).total; }

int launch_group_codes(const GroupParams& P, int32_t* order, int32_t* places,
                       int32_t* starts, void* workspace, hipStream_t stream) {
  const Way way = way_of(P);
  if (way == Way::kFew) {
    launch_traced("group_few_kernel", group_few_kernel,
                  dim3((unsigned)((P.choices + P.K + 1 + kThreads / 4 - 1) / (kThreads / 4))),
                  dim3(kThreads), 0, stream, P, order, places, starts);
    return check_launch("group_few_kernel");
  }
  const SortLayout L = sort_layout(P);
  char* w = static_cast<char*>(workspace);
  if (way == Way::kCounted) {
    auto* totals = reinterpret_cast<uint32_t*>(w + L.totals);
    auto* counts = reinterpret_cast<uint32_t*>(w + L.counts);
    const int rounds = rounds_of(P);
    launch_traced("group_count_kernel", group_count_kernel, dim3(L.chunks), dim3(kThreads), 0,
                  stream, P, rounds, counts);
    int rc = check_launch("group_count_kernel");
    if (rc) return rc;
    launch_traced("group_scan_kernel", group_scan_kernel, dim3((P.K + 16) / 16), dim3(16 * kScanParts), 0,
                  stream, P, L.chunks, counts, totals);
    if ((rc = check_launch("group_scan_kernel"))) return rc;
    int bits = 1;
    while ((1 << bits) <= P.K) ++bits;
    auto place = rounds == 4 ? group_place_kernel<4> : rounds == 8 ? group_place_kernel<8> : group_place_kernel<16>;
    launch_traced("group_place_kernel", place, dim3(L.chunks), dim3(kThreads), 0, stream, P, bits,
                  counts, totals, order, places, starts);
    return check_launch("group_place_kernel");
  }
  uint32_t *sorted = nullptr, *err = nullptr;
  if (P.choices > 0) {
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
                        const int32_t* named, const float* weights, void* out,
                        hipStream_t stream) {
  return GS_BY_TYPE(by_code_of)(P, rows, order, places, named, weights, out, stream);
}

int launch_rows_from_codes(const RowsParams& P, const void* rows,
                           const int32_t* places, const float* weights,
                           void* out, hipStream_t stream) {
  return GS_BY_TYPE(from_codes_of)(P, rows, places, weights, out, stream);
}

int launch_rows_from_codes_backward(const RowsParams& P, const void* grad,
                                    const void* rows, const int32_t* order,
                                    const int32_t* places, const int32_t* named,
                                    const float* weights, void* g_rows, float* g_weights,
                                    hipStream_t stream) {
  return GS_BY_TYPE(from_codes_bwd_of)(P, grad, rows, order, places, named, weights, g_rows,
                                       g_weights, stream);
}
#undef GS_BY_TYPE

}  // namespace gs
