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
// A row's statistics (max x, log2 S) are kept for the backward, which is one
// pass over the logits: log2 S = inf marks a row without probabilities.
//
// The forward reads a row once and holds it in registers: teams of 2 to 64
// lanes up to 2048 codes (1024 in 32 bits), a workgroup up to 16384, and parts
// of 2048 to 16384 codes, joined by a second launch, above (or for few long
// rows).  What bounds it, on an MI355X: HBM where rows are short (a million
// rows of 512 floats, best code: 393 us, 5.5 TB/s), VALU issue where 16-bit
// rows are long (64K rows of 16384, 8 best: 473 us, 4.6 TB/s, with 12 VALU
// instructions an element) or several best codes are wanted of short ones (a
// million rows of 64 in bf16, 8 best: 96 us, 2.4 TB/s).  The backward is bound by
// HBM at all lengths (64K x 16384: 664 us, 6.6 TB/s; 64K x 1024: 47 us, 6.0 TB/s).
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

// A part whose exponents lacked a shift, as small as a rounding's error.
__device__ __forceinline__ Part shifted(Part p, float shift) {
  const float f = exp2_fast(shift);
  return Part{p.m, p.s * f, (p.st + shift * p.s) * f};
}

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

// A lower bound of the top-th largest of 64 lanes' values, of its 16 leading bits:
// found bit by bit with a count of the lanes that reach it.
__device__ __forceinline__ float top_bound(float v, int top) {
  const uint32_t key = depth_key(v) >> 16;
  uint32_t t = 0;
#pragma unroll
  for (int bit = 15; bit >= 0; --bit) {
    const uint32_t q = t | (1u << bit);
    if (__popcll(__ballot(key >= q)) >= top) t = q;
  }
  const uint32_t u = t << 16;
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// A logit that may be among the best, and its column.
struct Found {
  float x;
  uint32_t i;
};

// How many of the first n lanes' keys are above this lane's.
__device__ __forceinline__ int place_among(uint64_t k, int n) {
  int place = 0;
  for (int j = 0; j < n; ++j) {
    const uint64_t q =
        ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), j) << 32) |
        (uint32_t)__builtin_amdgcn_readlane((int)k, j);
    place += q > k;
  }
  return place;
}

// Keys of ranks, the larger the better: for 16-bit logits and columns below 2^16
// one word, the logit's bits in their order above the column's complement; for
// floats rank_key.
template <typename T>
struct Rank {
  using Key = uint64_t;
  static __device__ __forceinline__ Key of(T x, uint32_t i) { return rank_key(x, i); }
  static __device__ __forceinline__ uint32_t column(Key k) { return ~(uint32_t)k; }
  static __device__ __forceinline__ float logit(Key k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
  }
  template <int L>
  static __device__ __forceinline__ Key best(Key k) { return team_best<L>(k); }
};
template <typename T>
struct Rank16 {
  using Key = uint32_t;
  static __device__ __forceinline__ Key of(T x, uint32_t i) {
    uint32_t u = __builtin_bit_cast(uint16_t, x);
    if (x == static_cast<T>(0.0f)) u = 0;
    if (!(x == x)) u = 0x7fff;
    return (u & 0x8000u ? ~u << 16 : (u | 0x8000u) << 16) | (0xffffu - i);
  }
  static __device__ __forceinline__ uint32_t column(Key k) { return 0xffffu - (k & 0xffffu); }
  static __device__ __forceinline__ float logit(Key k) {
    const uint32_t u = k >> 16;
    return to_float(__builtin_bit_cast(T, (uint16_t)(u & 0x8000u ? u ^ 0x8000u : ~u)));
  }
  template <int L>
  static __device__ __forceinline__ Key best(Key k) { return team_umax<L>(k); }
};
template <>
struct Rank<__bf16> : Rank16<__bf16> {};
template <>
struct Rank<_Float16> : Rank16<_Float16> {};

// A lane's E keys (4 or 8), the best first: an odd-even merge network.
template <int E, typename Key>
__device__ __forceinline__ void sort_keys(Key (&k)[E]) {
  auto order = [&](int a, int b) {
    const Key hi = k[a] > k[b] ? k[a] : k[b], lo = k[a] > k[b] ? k[b] : k[a];
    k[a] = hi;
    k[b] = lo;
  };
#pragma unroll
  for (int h = 0; h < E; h += 4) {
    order(h, h + 1);
    order(h + 2, h + 3);
    order(h, h + 2);
    order(h + 1, h + 3);
    order(h + 1, h + 2);
  }
  if constexpr (E == 8) {
    order(0, 4);
    order(1, 5);
    order(2, 6);
    order(3, 7);
    order(2, 4);
    order(3, 5);
    order(1, 2);
    order(3, 4);
    order(5, 6);
  }
}

struct ProbsOut {
  float* log_probs;
  float* entropy;
  float* top_log_probs;
  int32_t* top_codes;
  float2* stats;
  // Those of rows n on.
  ProbsOut from(int64_t n, int top) const {
    return ProbsOut{log_probs ? log_probs + n : nullptr, entropy + n,
                    top_log_probs ? top_log_probs + n * top : nullptr,
                    top_codes ? top_codes + n * top : nullptr, stats ? stats + n : nullptr};
  }
};

// The call's rows first .. first + rows - 1.
ProbsParams rows_of(ProbsParams P, int64_t first, int64_t rows) {
  P.rows = rows;
  P.codes = P.codes.from(first);
  return P;
}

// What a row's statistics say about one of its logits.
struct RowEnd {
  float base, log2_s, inv_t;
  __device__ __forceinline__ RowEnd(Part p, float inv_t_)
      : base(base_of(p.m)), log2_s(p.s == 0.0f ? 0.0f : log2_fast(p.s)), inv_t(inv_t_) {}
  // (not in base 2: a masked logit of the type's lowest value would overflow; the
  // difference by halves: it may be past the range where it is not over T)
  __device__ __forceinline__ float log_prob(float x) const {
    const float half = __builtin_fmaf(0.5f, x, -0.5f * base) * inv_t;
    return __builtin_fmaf(-kLn2, log2_s, half + half);
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
template <typename T, int TL, int R, bool Even>
struct Held {
  static constexpr int V = kVec<T>;
  vec_t<T> x[R];
  int lane;
  template <bool Stream = false>
  __device__ __forceinline__ void load(const T* row, int lane_, int n) {
    lane = lane_;
    constexpr bool kFix = R <= 8;  // (more vectors: fix_row's registers are not there)
    const T fill = static_cast<T>(-INFINITY);
    if constexpr (kFix || Even) {
      load_row<T, R, Even, Stream>(x, row, lane * V, TL * V, n, fill);
      fix_row<T, R, Even>(x, lane * V, TL * V, n, fill);
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) x[r] = load_part<T, Even, Stream>(row, (r * TL + lane) * V, n, fill);
    }
  }
  __device__ __forceinline__ int column(int r, int v) const { return (r * TL + lane) * V + v; }
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int r = 0; r < R; ++r) gs::forget<T>(x[r]);
  }
  // The largest element of vector r (of the thread: the largest of them).
  __device__ __forceinline__ float max_of(int r) const {
    float m = max3(to_float(x[r][0]), to_float(x[r][1]), to_float(x[r][2]));
#pragma unroll
    for (int v = 3; v + 1 < V; v += 2) m = max3(m, to_float(x[r][v]), to_float(x[r][v + 1]));
    return fmaxf(m, to_float(x[r][V - 1]));
  }
  // s and st of this thread's elements, exponents from e (without its shift).
  __device__ __forceinline__ Part part(const Exponent& e) {
    Part p{e.m, 0.0f, 0.0f};
    auto sum = [&](auto exponent) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        gs::forget<T>(x[r]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float t = exponent(to_float(x[r][v]));
          const float y = exp2_fast(t);
          p.s += y;
          p.st = __builtin_fmaf(y, bounded(t), p.st);
        }
      }
    };
    if (e.plain)
      sum([&](float x) { return e.fast(x); });
    else
      sum([&](float x) { return e.slow(x); });
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
  // The team's lowest column whose logit equals m; most[r]: max_of(r).  Vectors
  // are in the order of the columns: those after the first that holds m are
  // not looked at (by a wavefront as a whole).
  __device__ __forceinline__ uint32_t first_equal(float m, const float (&most)[R]) const {
    uint32_t i = ~0u;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool hit = most[r] == m && i == ~0u;
      if (__ballot(hit) == 0) continue;
      uint32_t j = ~0u;
#pragma unroll
      for (int v = V - 1; v >= 0; --v)
        if (to_float(x[r][v]) == m) j = column(r, v);
      if (hit) i = j;
      if (TL == 64) break;
    }
    return team_min<TL>(i);
  }
};

// ---- rows of at most TL * kVec * R codes: a team of TL lanes per row
//
// 12 to 32 elements a lane, in steps of a third or a half between the powers of
// two, where no more than the best code is wanted: what a row costs beside its
// elements is shared by more of them, and fewer lanes idle.  (64K rows of 1024 in
// bf16: 33 us with 32 elements a lane, 38 with 16; 1M rows of 104 floats 92 us
// with 16, 182 with 4; 1M of 130 in bf16 82 with 24, 123 with 16 and half the
// lanes idle.)

template <typename T, int TL, int R, bool Even>
__global__ __launch_bounds__(kThreads) void probs_rows_kernel(
    ProbsParams P, const T* __restrict__ logits, ProbsOut out) {
  constexpr int kTeams = kThreads / TL;
  __shared__ Found found[TL == 64 ? kWaves * 64 : 1];
  const int lane = threadIdx.x & (TL - 1);
  const int team = TL == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TL) : threadIdx.x / TL;
  int64_t n = (int64_t)blockIdx.x * kTeams + team;
  const bool active = n < P.rows;
  if (!active) n = P.rows - 1;  // (its lanes go along)
  const T* row = logits + n * P.stride;
  Held<T, TL, R, Even> x;
  x.load(row, lane, P.K);
  const int code = P.codes.p ? P.codes.at(n, P.K) : kNoCode;
  float most[R];  // of each vector
#pragma unroll
  for (int r = 0; r < R; ++r) most[r] = x.max_of(r);
  float mine = most[0];
#pragma unroll
  for (int r = 1; r < R; ++r) mine = fmaxf(mine, most[r]);
  const float m = team_max<TL>(mine);
  T code_logit = static_cast<T>(0.0f);
  if (code >= 0) code_logit = row[code];
  const Exponent ex(base_of(m), 0.0f, P.inv_t * kLog2e);
  Part p = x.part(ex);
  p.m = m;
  p.s = team_sum<TL>(p.s);
  p.st = team_sum<TL>(p.st);
  p = shifted(p, ex.shift);
  const RowEnd e(p, P.inv_t);
  if (lane == 0 && active) write_row(out, n, p, e, code, to_float(code_logit));
  x.forget();
  const int top = P.top;
  if (top == 0) return;
  auto put = [&](int j, uint32_t i, float v) {
    if (active) {
      out.top_codes[n * top + j] = (int)i;
      out.top_log_probs[n * top + j] = e.log_prob(v);
    }
  };
  if constexpr (TL < 64 && R * kVec<T> <= 8) {
    // Several codes of a narrow team: every lane sorts its keys, and in each
    // turn the team's best head is taken and its lane goes on to its next.
    if (top > 1) {
      using K = Rank<T>;
      constexpr int V = kVec<T>, E = R * V;
      typename K::Key k[E], mine_key = 0;
#pragma unroll
      for (int v = 0; v < E; ++v) k[v] = K::of(x.x[v / V][v % V], x.column(v / V, v % V));
      sort_keys<E>(k);
      for (int j = 0; j < top; ++j) {
        const typename K::Key best = K::template best<TL>(k[0]);
        if (k[0] == best) {
#pragma unroll
          for (int v = 0; v + 1 < E; ++v) k[v] = k[v + 1];
          k[E - 1] = 0;
        }
        if (lane == (j & (TL - 1))) mine_key = best;
        // (as many as the team has lanes are written at once)
        if ((j & (TL - 1)) == TL - 1 || j == top - 1) {
          const int at = (j & ~(TL - 1)) + lane;
          if (at <= j) put(at, K::column(mine_key), K::logit(mine_key));
        }
      }
      return;
    }
  }
  int from = 0;
  const bool plain = p.s == p.s;  // (no NaN)
  if (plain) {
    // the best: the first column that has the maximum
    const uint32_t i = x.first_equal(p.m, most);
    if (lane == 0) put(0, i, p.m);
    from = 1;
  }
  if (from == top && __all(plain)) return;
  if constexpr (TL == 64) {
    // The top-th largest of the lanes' maxima is a lower bound of the top-th
    // largest logit: the logits from there up are few (ties aside), are
    // collected, and find their places by counting.
    if (plain && top > 1) {
      const float bound = top_bound(mine, top);
      if (bound > -INFINITY) {
        Found* list = found + (threadIdx.x & ~63);
        int total = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (__ballot(most[r] >= bound) == 0) continue;
#pragma unroll
          for (int v = 0; v < kVec<T>; ++v) {
            const float f = to_float(x.x[r][v]);
            const uint64_t hit = __ballot(f >= bound);
            if (hit == 0) continue;
            const int at = total + __builtin_amdgcn_mbcnt_hi(
                                       (uint32_t)(hit >> 32),
                                       __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0));
            if (f >= bound && at < 64) list[at] = Found{f, (uint32_t)x.column(r, v)};
            total += __popcll(hit);
          }
        }
        if (total <= 64) {
          __builtin_amdgcn_wave_barrier();
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          const Found mine = lane < total ? list[lane] : Found{-INFINITY, ~0u};
          const int place = place_among(rank_key(mine.x, mine.i), total);
          if (lane < total && place < top) put(place, mine.i, mine.x);
          return;
        }
      }
    }
  }
  uint64_t last = ~0ull;
  if (plain) last = rank_key(p.m, x.first_equal(p.m, most));
  for (int j = from; j < top; ++j) {
    last = team_best<TL>(x.best_below(last));
    const uint32_t i = ~(uint32_t)last;
    if (lane == 0) put(j, i, to_float(row[i]));
  }
}

// ---- longer rows: a workgroup per part of a row
//
// (64K rows of 16384 in bf16, one build against the other: 64 elements a thread
// take 448 us, 512 threads of 32 elements 629: reductions and the search for the
// bound are per wavefront.  Five wavefronts per SIMD: with four 559 us.)

// One part of a row per workgroup.  parts = 1: the row's outputs; else its
// statistics and best keys go to partials, for probs_join_kernel.
struct Split {
  int parts;    // per row
  int length;   // elements of a part (the last may be shorter)
  Part* stats;  // [rows][parts]
  uint64_t* best;  // [rows][parts][top]
  bool stream;     // past_caches
};

constexpr int kFound = 256;  // logits collected for the best ones

template <typename T, int W, int R, bool Even>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(5))) void probs_parts_kernel(
    ProbsParams P, const T* __restrict__ logits, ProbsOut out, Split split) {
  constexpr int kThreads = 64 * W;
  __shared__ Part parts[W];
  __shared__ float groups[64];  // largest logits of groups of W lanes
  __shared__ Found found[kFound];
  __shared__ uint64_t best[W];
  __shared__ int total;
  const int64_t n = blockIdx.x / (unsigned)split.parts;
  const int part = (int)(blockIdx.x - (uint32_t)n * (unsigned)split.parts);
  const int first = part * split.length;
  const int len = min(split.length, P.K - first);
  const T* row = logits + n * P.stride;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  Held<T, kThreads, R, Even> x;
  if (split.stream)
    x.template load<true>(row + first, threadIdx.x, len);
  else
    x.load(row + first, threadIdx.x, len);
  const int code = P.codes.p && split.parts == 1 ? P.codes.at(n, P.K) : kNoCode;
  float most[R];  // of each vector
#pragma unroll
  for (int r = 0; r < R; ++r) most[r] = x.max_of(r);
  float mine = most[0];
#pragma unroll
  for (int r = 1; r < R; ++r) mine = fmaxf(mine, most[r]);
  const float c = P.inv_t * kLog2e;
  const float m = wave_max(mine);
  T code_logit = static_cast<T>(0.0f);
  if (code >= 0) code_logit = row[code];
  const Exponent ex(base_of(m), 0.0f, c);
  Part p = x.part(ex);
  p.m = m;
  p.s = wave_sum(p.s);
  p.st = wave_sum(p.st);
  p = shifted(p, ex.shift);
  const int top = min(P.top, len);
  const float group = team_max<W>(mine);
  if ((lane & (W - 1)) == 0) groups[threadIdx.x / W] = group;
  if (lane == 0) parts[w] = p;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  // (joined by teams of W lanes, each lane a wavefront's part)
  p = parts[lane & (W - 1)];
  const float all = team_max<W>(p.m);
  const float d = bounded((p.m - base_of(all)) * c), f = exp2_fast(d);
  p.st = team_sum<W>(f * (p.st + d * p.s));
  p.s = team_sum<W>(f * p.s);
  p.m = all;
  const RowEnd e(p, P.inv_t);
  if (threadIdx.x == 0) {
    if (split.parts == 1)
      write_row(out, n, p, e, code, to_float(code_logit));
    else
      split.stats[(int64_t)blockIdx.x] = p;
  }
  if (P.top == 0) return;
  auto put = [&](int j, uint64_t key, float x) {
    if (split.parts == 1) {
      out.top_codes[n * P.top + j] = (int)~(uint32_t)key;
      out.top_log_probs[n * P.top + j] = e.log_prob(x);
    } else {
      // (columns of the whole row; 0 where the part has fewer than top)
      split.best[(int64_t)blockIdx.x * P.top + j] = key == 0 ? 0 : key - (uint32_t)first;
    }
  };
  for (int j = top + threadIdx.x; j < P.top; j += kThreads) put(j, 0, 0.0f);
  // (64 groups: the top-th largest of their largest logits is a lower bound)
  const float bound = top == 1 ? all : top_bound(groups[lane], top);
  if (p.s == p.s && bound > -INFINITY) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (most[r] < bound) continue;
      gs::forget<T>(x.x[r]);
#pragma unroll
      for (int v = 0; v < kVec<T>; ++v) {
        const float f = to_float(x.x[r][v]);
        if (f >= bound) {
          const int at = atomicAdd(&total, 1);
          if (at < kFound) found[at] = Found{f, (uint32_t)x.column(r, v)};
        }
      }
    }
    __syncthreads();
    const int count = total;
    // (the list's order depends on the run, the places do not)
    if (count <= 64) {
      if (w != 0) return;
      const Found mine = lane < count ? found[lane] : Found{-INFINITY, ~0u};
      const uint64_t k = rank_key(mine.x, mine.i);
      const int place = place_among(k, count);
      if (lane < count && place < top) put(place, k, mine.x);
      return;
    }
    if (count <= kFound) {
      if ((int)threadIdx.x < count) {
        const Found mine = found[threadIdx.x];
        const uint64_t k = rank_key(mine.x, mine.i);
        int place = 0;
        for (int j = 0; j < count; ++j) place += rank_key(found[j].x, found[j].i) > k;
        if (place < top) put(place, k, mine.x);
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
    for (int q = 1; q < W; ++q) k = max64(k, best[q]);
    last = k;
    if (threadIdx.x == 0) put(j, k, to_float(row[~(uint32_t)k]));
  }
}

// A wavefront per row joins the row's parts: the keys and the best codes' logits
// are each loaded at once (one row of 131072 codes in 64 parts, 8 best: 10.7 us
// with a load waited for in every step, 4.0 so).
constexpr int kKeys = 8;  // keys that a lane holds at a time

template <typename T>
__global__ __launch_bounds__(64) void probs_join_kernel(
    ProbsParams P, const T* __restrict__ logits, ProbsOut out, Split split) {
  const int64_t n = blockIdx.x;
  const int lane = threadIdx.x;
  const T* row = logits + n * P.stride;
  const float c = P.inv_t * kLog2e;
  const int total = split.parts * P.top;
  const uint64_t* keys = split.best + n * total;
  uint64_t held[kKeys];
#pragma unroll
  for (int q = 0; q < kKeys; ++q)
    held[q] = q * 64 + lane < total ? keys[q * 64 + lane] : 0;
  T code_logit = static_cast<T>(0.0f);
  int code = kNoCode;
  if (P.codes.p) {
    code = P.codes.at(n, P.K);
    if (code >= 0) code_logit = row[code];
  }
  Part p{-INFINITY, 0.0f, 0.0f};
  for (int j = lane; j < split.parts; j += 64) p = joined(p, split.stats[n * split.parts + j], c);
  const float all = wave_max(p.m);
  const float d = bounded((p.m - base_of(all)) * c), f = exp2_fast(d);
  p.st = wave_sum(f * (p.st + d * p.s));
  p.s = wave_sum(f * p.s);
  p.m = all;
  const RowEnd e(p, P.inv_t);
  if (lane == 0) write_row(out, n, p, e, code, to_float(code_logit));
  uint64_t last = ~0ull, mine = 0;
  for (int j = 0; j < P.top; ++j) {
    uint64_t k = 0;
#pragma unroll
    for (int q = 0; q < kKeys; ++q)
      if (held[q] < last) k = max64(k, held[q]);
    for (int i = kKeys * 64 + lane; i < total; i += 64)
      if (keys[i] < last) k = max64(k, keys[i]);
    last = team_best<64>(k);
    if (lane == j) mine = last;
  }
  if (lane < P.top) {
    const uint32_t i = ~(uint32_t)mine;
    out.top_codes[n * P.top + lane] = (int)i;
    out.top_log_probs[n * P.top + lane] = e.log_prob(to_float(row[i]));
  }
}

// ---- backward

// dL/dx = -p (total + gH (log p + H)) + gl at the code + gt at the
// alternatives, over T.  Per element two fused multiply-adds, a base-2
// exponential and a product: p = 2^(t + down), log p = (t + down) ln 2 with t from
// Exponent, and everything that is the same for the row is in two constants.
// A team of TL lanes per part of a row of TL * kVec * R columns (`parts` of
// them per row).  (Two or three vectors a lane: 1M rows of 104 floats 277 us with
// one, 186 with two; of 96 in bf16 139 and, with three, 97.)
template <typename T, int TL, int R, bool Even>
__global__ __launch_bounds__(kThreads) void probs_bwd_kernel(
    ProbsParams P, const T* __restrict__ logits,
    const int32_t* __restrict__ top_codes, const float2* __restrict__ stats,
    const float* __restrict__ entropy, const float* __restrict__ g_log_probs,
    const float* __restrict__ g_entropy, const float* __restrict__ g_top,
    T* __restrict__ g_logits, int parts) {
  constexpr int kTeams = kThreads / TL, V = kVec<T>, kSpan = TL * V * R;
  // Gradients of single columns: rows of one team add them up in LDS, a lane per
  // alternative (R = 4: rows of several parts, whose few columns are compared).
  constexpr bool kSpread = R < 4;
  __shared__ alignas(16) float spread[kSpread ? kThreads * V * R : 1];
  const int lane = threadIdx.x & (TL - 1);
  const int team = TL == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TL) : threadIdx.x / TL;
  const int64_t i = (int64_t)blockIdx.x * kTeams + team;
  if (i >= P.rows * parts) return;
  const int64_t n = parts == 1 ? i : i / parts;
  const int first = (int)(i - n * parts) * kSpan;
  const T* row = logits + n * P.stride;
  T* out = g_logits + n * P.K;
  vec_t<T> x[R];
  load_row<T, R, Even, true>(x, row, first + lane * V, TL * V, P.K, static_cast<T>(-INFINITY));
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
  float* mine = spread + (threadIdx.x - lane) * (V * R);  // (the team's columns)
  if constexpr (kSpread) {
    if (top > 0) {
#pragma unroll
      for (int v = 0; v < V * R; v += 4)
        *reinterpret_cast<float4*>(&mine[lane * (V * R) + v]) = make_float4(0, 0, 0, 0);
      __builtin_amdgcn_wave_barrier();
      float sum = 0.0f;
      for (int j = lane; j < top; j += TL) {
        const float w = gt[j];
        const unsigned col = (unsigned)(tc[j] - first);
        sum += w;
        // (a column may also be the code's: two additions, in either order)
        if (col < (unsigned)kSpan) atomicAdd(&mine[col], w * P.inv_t);
      }
      total += team_sum<TL>(sum);
      __builtin_amdgcn_wave_barrier();
    }
  } else {
    for (int j = 0; j < top; ++j) total += gt[j];
  }
  // 16 bits of a result: exponents 32 up, so that probabilities that the
  // hardware's exponential flushes are far below the type's smallest step (the
  // exponents' own steps, 4e-6 there, are lost in 16 bits).  32 bits: exp2_full.
  fix_row<T, R, Even>(x, first + lane * V, TL * V, P.K, static_cast<T>(-INFINITY));
  constexpr float kUp = sizeof(T) == 2 ? 32.0f : 0.0f;
  const Exponent e(st.x, st.y - kUp, P.inv_t * kLog2e);
  const float down = e.shift - kUp;
  const float f = -P.inv_t * exp2_fast(down);
  const float fixed = f * (total + ge * (entropy[n] + down * kLn2));
  const float per_t = f * ge * kLn2;
  gl *= P.inv_t;
  float g[R * V];
  auto products = [&](auto exponent) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        // (a masked logit: 0.  A row with a NaN has NaN constants.)
        const float t = bounded(exponent(to_float(x[r][v])));
        const float y = sizeof(T) == 2 ? exp2_fast(t) : exp2_full(t);
        g[r * V + v] = y * __builtin_fmaf(per_t, t, fixed);
      }
  };
  if (e.plain)
    products([&](float x) { return e.fast(x); });
  else
    products([&](float x) { return e.slow(x); });
  auto add = [&](int col, float w) {
    const unsigned rel = (unsigned)(col - first);
    if (rel >= (unsigned)kSpan) return;
    // (of a wavefront's row the place is the same for all lanes: one vector's
    // elements are looked at)
    const float own = lane == (int)(rel / V & (TL - 1)) ? w : 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned in = rel - r * (V * TL);
      if (R > 1 && in >= (unsigned)(V * TL)) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) g[r * V + v] += in % V == (unsigned)v ? own : 0.0f;
    }
  };
  if (code >= 0) add(code, gl);
  if constexpr (kSpread) {
    if (top > 0)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int v = 0; v < V; v += 4) {
          const float4 w = *reinterpret_cast<const float4*>(&mine[(r * TL + lane) * V + v]);
          g[r * V + v] += w.x;
          g[r * V + v + 1] += w.y;
          g[r * V + v + 2] += w.z;
          g[r * V + v + 3] += w.w;
        }
  } else {
    for (int j = 0; j < top; ++j) add(tc[j], gt[j] * P.inv_t);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    vec_t<T> o;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = static_cast<T>(g[r * V + v]);
    store_part<T, Even, true>(out, first + (r * TL + lane) * V, P.K, o);
  }
}

// Rows of at most this many codes are one workgroup's; longer ones are cut.
constexpr int kPartLong = 16384;

Split split_of(const ProbsParams& P) {
  Split s{1, P.K, nullptr, nullptr, past_caches(P.rows, P.K, P.dtype)};
  if (P.K <= kPartLong) return s;
  // Few rows: shorter parts, until there is one for each of 512 workgroups (one
  // row of 131072: 8.0 us against 9.6, 64 rows of 32768 8.7 against 10.1).
  int64_t length = kPartLong;
  while (length > 2048 && P.rows * ((P.K + length - 1) / length) < 512) length /= 2;
  s.length = (int)length;
  s.parts = (int)((P.K + length - 1) / length);
  return s;
}

template <typename T, bool Even>
int forward_of(const ProbsParams& P, const void* logits, const ProbsOut& out,
               void* workspace, hipStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  constexpr int V = kVec<T>;
  const int vecs = (P.K + V - 1) / V;
#define GS_ROWS(TL, R)                                                           \
  if (vecs <= TL * R) {                                                          \
    constexpr int kTeams = kThreads / TL;                                        \
    return in_launches(P.rows, kMostBlocks * kTeams, [&](int64_t n, int64_t rows) { \
      launch_traced("probs_rows_kernel", (probs_rows_kernel<T, TL, R, Even>),    \
                    dim3((unsigned)((rows + kTeams - 1) / kTeams)),              \
                    dim3(kThreads), 0, stream, rows_of(P, n, rows),              \
                    x + n * P.stride, out.from(n, P.top));                       \
      return check_launch("probs_rows_kernel");                                  \
    });                                                                          \
  }
  // (several codes of rows above 128 floats or 256 elements of 16 bits are found by
  // a whole wavefront's ballots: 524K rows of 256 floats, 8 best, 245 us so and 268 from
  // teams of 32 lanes' sorted keys)
  if (P.top <= 1) {
    GS_ROWS(2, 1)
    if constexpr (sizeof(T) == 2) {
      GS_ROWS(2, 3) GS_ROWS(4, 2) GS_ROWS(4, 3) GS_ROWS(8, 2) GS_ROWS(8, 3) GS_ROWS(16, 2)
      GS_ROWS(16, 3) GS_ROWS(32, 2) GS_ROWS(32, 3) GS_ROWS(32, 4) GS_ROWS(64, 3) GS_ROWS(64, 4)
    } else {
      GS_ROWS(2, 2) GS_ROWS(2, 3) GS_ROWS(4, 2) GS_ROWS(4, 3) GS_ROWS(4, 4) GS_ROWS(8, 3) GS_ROWS(8, 4)
      GS_ROWS(16, 3) GS_ROWS(16, 4) GS_ROWS(32, 3) GS_ROWS(32, 4) GS_ROWS(64, 3) GS_ROWS(64, 4)
    }
  }
  if constexpr (sizeof(T) == 2) {
    GS_ROWS(2, 1) GS_ROWS(4, 1) GS_ROWS(8, 1) GS_ROWS(16, 1) GS_ROWS(32, 1)
  } else {
    GS_ROWS(2, 1) GS_ROWS(2, 2) GS_ROWS(4, 2) GS_ROWS(8, 2) GS_ROWS(16, 2)
  }
  GS_ROWS(64, 1) GS_ROWS(64, 2) GS_ROWS(64, 4)
#undef GS_ROWS
  Split s = split_of(P);
  if (s.parts > 1) {
    s.stats = static_cast<Part*>(workspace);
    s.best = reinterpret_cast<uint64_t*>(
        static_cast<char*>(workspace) +
        align_up((size_t)P.rows * s.parts * sizeof(Part), 256));
  }
  const int len = (s.length + V - 1) / V;
  constexpr int kR = 16 / V;  // vectors of 16 elements
  // (launches of one after another use the same workspace)
  return in_launches(P.rows, kMostBlocks / s.parts, [&](int64_t n, int64_t rows) {
    const ProbsParams Q = rows_of(P, n, rows);
    const T* from = x + n * P.stride;
    const ProbsOut to = out.from(n, P.top);
#define GS_PARTS(W, R)                                                         \
  launch_traced("probs_parts_kernel", (probs_parts_kernel<T, W, R, Even>),     \
                dim3((unsigned)(rows * s.parts)), dim3(64 * W), 0, stream, Q, from, to, s)
    if (len <= 256 * kR) GS_PARTS(4, kR);
    else if (len <= 512 * kR) GS_PARTS(4, 2 * kR);
    else GS_PARTS(4, 4 * kR);
#undef GS_PARTS
    const int rc = check_launch("probs_parts_kernel");
    if (rc || s.parts == 1) return rc;
    launch_traced("probs_join_kernel", (probs_join_kernel<T>), dim3((unsigned)rows),
                  dim3(64), 0, stream, Q, from, to, s);
    return check_launch("probs_join_kernel");
  });
}

template <typename T, bool Even>
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
    constexpr int kTeams = kThreads / TL;                                      \
    return in_launches(P.rows, kMostBlocks * kTeams / parts, [&](int64_t n, int64_t rows) { \
      auto from = [&](const float* q, int per) { return q ? q + n * per : nullptr; }; \
      launch_traced("probs_bwd_kernel", (probs_bwd_kernel<T, TL, R, Even>),    \
                    dim3((unsigned)((rows * parts + kTeams - 1) / kTeams)),    \
                    dim3(kThreads), 0, stream, rows_of(P, n, rows),            \
                    x + n * P.stride, top_codes ? top_codes + n * P.top : nullptr, \
                    stats + n, entropy + n, from(g_log_probs, 1),              \
                    from(g_entropy, 1), from(g_top, P.top), g + n * P.K, parts); \
      return check_launch("probs_bwd_kernel");                                 \
    });                                                                        \
  }
  if (vecs <= 2) GS_BWD(2, 1)
  if (vecs <= 4) GS_BWD(4, 1)
  if (vecs <= 8) GS_BWD(8, 1)
  if (vecs <= 16) GS_BWD(8, 2)
  if (vecs <= 24) GS_BWD(8, 3)
  if (vecs <= 32) GS_BWD(16, 2)
  if (vecs <= 48) GS_BWD(16, 3)
  if (vecs <= 64) GS_BWD(32, 2)
  if (vecs <= 96) GS_BWD(32, 3)
  if (vecs <= 128) GS_BWD(64, 2)
  if (vecs <= 192) GS_BWD(64, 3)
  GS_BWD(64, 4)
#undef GS_BWD
}

}  // namespace

size_t probs_workspace_bytes(const ProbsParams& P) {
  const Split s = split_of(P);
  if (s.parts == 1) return 0;
  return align_up((size_t)P.rows * s.parts * sizeof(Part), 256) +
         (size_t)P.rows * s.parts * P.top * sizeof(uint64_t);
}

int launch_probs_forward(const ProbsParams& P, const void* logits,
                         float* log_probs, float* entropy, float* top_log_probs,
                         int32_t* top_codes, float2* stats, void* workspace,
                         hipStream_t stream) {
  if (P.rows == 0) return GSPLAT_OK;
  const bool even = P.K % (P.dtype == GSPLAT_F32 ? 4 : 8) == 0;
  auto f = P.dtype == GSPLAT_F32    ? (even ? forward_of<float, true> : forward_of<float, false>)
           : P.dtype == GSPLAT_BF16 ? (even ? forward_of<__bf16, true> : forward_of<__bf16, false>)
                                    : (even ? forward_of<_Float16, true> : forward_of<_Float16, false>);
  return f(P, logits, ProbsOut{log_probs, entropy, top_log_probs, top_codes, stats},
           workspace, stream);
}

int launch_probs_backward(const ProbsParams& P, const void* logits,
                          const int32_t* top_codes, const float2* stats,
                          const float* entropy, const float* g_log_probs,
                          const float* g_entropy, const float* g_top,
                          void* g_logits, hipStream_t stream) {
  if (P.rows == 0) return GSPLAT_OK;
  const bool even = P.K % (P.dtype == GSPLAT_F32 ? 4 : 8) == 0;
  auto f = P.dtype == GSPLAT_F32    ? (even ? backward_of<float, true> : backward_of<float, false>)
           : P.dtype == GSPLAT_BF16 ? (even ? backward_of<__bf16, true> : backward_of<__bf16, false>)
                                    : (even ? backward_of<_Float16, true> : backward_of<_Float16, false>);
  return f(P, logits, top_codes, stats, entropy, g_log_probs, g_entropy, g_top,
           g_logits, stream);
}

}  // namespace gs
