// code_adapters.h -- low-rank maps of splats' rows, each by its code's own.
//
//   h[j]   = down[c] x[n]                  (n: the splat at place j, c its code)
//   out[n] = base[n] + scale * up[c] h[j]
//   dh[j]  = scale * up[c]^T g[n]
//   gx[n]  = down[c]^T dh[j]
//   gdown[c] = sum over c's places of dh[j] x[n]^T,  gup[c] = scale * sum of g[n] h[j]^T
//
// A splat without a code has out = base and no gradient; one with a code out of
// range is NaN.
//
// A workgroup takes a tile: up to M places of one code, whose rows it reads
// once.  Its four wavefronts share out the rows' values, D, for the hidden
// values (which meet in LDS) and then the results' values, E.  The gradient of
// the rows is the same with up^T and down^T, turned on their way through LDS.
// Gradients of the maps: a workgroup takes up to L places of a code and a block
// of columns; longer codes' sums are joined by another launch, in order.
//
// Everything is a matrix product of 16 x 16 tiles.  In 16 bits the hidden values
// go into the second product as the sum of three bfloat16, and float16 factors beside
// them as that of two: exactly, and without a range to leave.  Each part of one is
// multiplied with each of the other.
// (An infinite value of a row or a map makes what depends on it infinite or NaN.)
//
// What bounds it, on an MI355X: 131072 rows of 1024 -> 1024 values of bfloat16,
// rank 32, 256 codes: the forward 174 us for 805 MB (4.6 TB/s; a large copy
// reaches 4.9), the rows' gradient 130 us for 537 MB, the maps' gradients 117 us
// for 537 MB and the hidden values (4.6 TB/s).  They wait on loads: two to three
// wavefronts a SIMD, 6 to 12 KB on their way each.  65536 rows of 128 -> 59 floats, rank 8:
// 22, 21 and 20 us for 49 MB each: one and a half rounds of workgroups, each a
// chain of dependent loads (starts, order, rows, maps).  What took the first case's
// step from 785 us to 442 (445 with all bits of the hidden values): coalesced rows of the factors (turned in LDS), rows
// without a code in all threads, loads without a mask, a branch or a use behind
// them, and stores and last reads past the caches (the maps' gradients 155 us
// without, as what they read was no longer there).
//
// Tiles: 64 places up to rank 64 once codes have 32 on average and tiles fill the card,
// otherwise 16 (both sides at rows_plan).  Measured and not kept: 32 places for narrow
// rows (22 us for 21) and above rank 64 (131072 rows, 256 a code: 416 and 446 us at
// 1024 -> 1024, rank 128, 132 and 156 at 128 -> 59, rank 96; the rows' gradient 518 and
// 493, 144 and 200), three wavefronts a SIMD for the maps' gradients at rank 32, which
// spill (155 us as two took at that time).
#pragma once

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "codes.h"

namespace gs {
namespace {

constexpr int kThreads = 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- tiles

// Of the places [0, rows), code k's are [start(k), start(k + 1)); k = K: those
// without a code.
__device__ __forceinline__ int64_t start_of(const AdapterParams& P, int64_t k) {
  if (k > P.K) return P.rows;
  return min(max((int64_t)P.starts[k], (int64_t)0), P.rows);
}

// Slots of tiles of M places: code k's begin at start(k) / M + k, room for
// ceil(count / M) of them whatever the start.  With many more codes than places
// a slot is a place instead, the first of its tile or none's.
struct Slots {
  int M;
  bool by_place;
  int64_t begin;  // the launch's first (a launch has fewer than 2^32 threads)
  __device__ __forceinline__ int64_t first(int64_t start, int64_t k) const {
    return by_place ? start : start / M + k;
  }
};
inline int64_t slots_of(const AdapterParams& P, int M, bool by_place) {
  return by_place ? P.rows : P.rows / M + P.K + 1;
}
// (fewer slots, of those that both ways have)
inline bool by_place(const AdapterParams& P, int M) {
  return P.rows < P.rows / M + P.K + 1;
}

struct Tile {
  int64_t code, first, index;  // index: of the code's tiles
  int count;                   // 0: the slot is nobody's
};

// The wavefront's 64 lanes look at 64 codes at a time.
__device__ __forceinline__ Tile tile_at(const AdapterParams& P, Slots S, int64_t slot) {
  int64_t lo = 0, len = (int64_t)P.K + 1;
  const int lane = threadIdx.x & 63;
  while (len > 1) {
    const int64_t step = (len + 63) / 64, k = lo + lane * step;
    const bool before = lane * step < len && S.first(start_of(P, k), k) <= slot;
    const int found = max(__popcll(__ballot(before)), 1) - 1;
    lo += found * step;
    len = min(step, len - found * step);
  }
  const int64_t from = start_of(P, lo), to = start_of(P, lo + 1);
  Tile t{lo, slot, 0, 0};
  const int64_t at = slot - S.first(from, lo);
  if (S.by_place) {
    if (at % S.M != 0) return t;
    t.index = at / S.M;
  } else {
    t.index = at;
    t.first = from + at * S.M;
  }
  if (at >= 0 && t.first < to) t.count = (int)min((int64_t)S.M, to - t.first);
  return t;
}

// The row of place j (-1: out of range).
__device__ __forceinline__ int row_at(const AdapterParams& P, int64_t j) {
  if (P.by_code) return (int)j;
  const int n = P.order[j];
  return n >= 0 && n < P.rows ? n : -1;
}

// ---- 16 x 16 tiles

// A lane has 16 bytes of a factor: of its row lane % 16, the quarter lane / 16 of 4 *
// kVec values.  Of the product of two, lane l has elements 4 (l / 16) + 0..3 of
// column l % 16.
template <typename T>
__device__ __forceinline__ void mma(f32x4& acc, vec_t<T> a, vec_t<T> b) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
  } else if constexpr (__is_same(T, __bf16)) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
  }
}

// x as the sum of N bfloat16, each what the ones before leave, cut off after 8 bits (so
// that it stays in range): three hold a float, two a float16, exactly.  An infinity and
// a NaN have no smaller parts.
constexpr int kParts = 3;
template <int N>
__device__ __forceinline__ void split(float x, uint32_t (&part)[N]) {
  const bool whole = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t u = __float_as_uint(x);
    part[i] = u >> 16;
    x = whole ? x - __uint_as_float(u & 0xffff0000u) : 0.0f;
  }
}
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8 (&part)[N]) {
  u32x4 w[N];
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint32_t a[N], b[N];
    split(x[2 * p], a);
    split(x[2 * p + 1], b);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i][p] = a[i] | b[i] << 16;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) part[i] = __builtin_bit_cast(bf16x8, w[i]);
}
// Eight values of a map or a row as bfloat16: themselves, or a float16's two parts.
template <typename T>
constexpr int kOfMap = __is_same(T, __bf16) ? 1 : 2;
template <typename T>
__device__ __forceinline__ void parts(vec_t<T> x, bf16x8 (&part)[kOfMap<T>]) {
  if constexpr (__is_same(T, __bf16)) {
    part[0] = x;
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_float(x[i]);
    split8(f, part);
  }
}

// How widths fit the 16-byte vectors: all are whole ones, at least one, or some less.
constexpr int kShort = 0, kRagged = 1, kWhole = 2;
inline int fit_of(std::initializer_list<int> widths, int vec) {
  int fit = kWhole;
  for (const int n : widths) fit = std::min(fit, n % vec == 0 ? kWhole : n > vec ? kRagged : kShort);
  return fit;
}

// Values i .. i + kVec - 1 of a row of n as one load, and later brought to their
// place, zeros past the row's end.  Apart, since a value that is looked at as it is
// loaded, or loaded behind a branch, is waited for: the loads after it would start
// only then.
// Stream: past the caches, for what nothing reads again.
template <typename T, int Fit, bool Stream = false>
__device__ __forceinline__ vec_t<T> load_raw(const T* row, int i, int n) {
  if (Fit != kShort || n >= kVec<T>) {
    const T* at = row + min(i, n - kVec<T>);
    return Stream ? load_vec_stream(at) : load_vec(at);
  }
  return load_part(row, i, n, static_cast<T>(0.0f));
}
template <typename T, int Fit>
__device__ __forceinline__ void bring(vec_t<T>& v, int i, int n) {
  vec_t<T> x[1] = {v};
  fix_row<T, 1, Fit == kWhole>(x, i, 0, n, static_cast<T>(0.0f));
  v = i < n ? x[0] : vec_t<T>{};
}

// N adjacent values of a row of n from i on.  (Whole: n is a multiple of N.)
template <int N, typename T, bool Whole>
__device__ __forceinline__ void store_n(T* row, int i, int n, const T (&v)[N]) {
  if (Whole ? i < n : i + N <= n) {
    if constexpr (sizeof(v) == 16) {
      vec_t<T> x;
      __builtin_memcpy(&x, v, 16);
      store_vec_stream(row + i, x);
    } else {
      __builtin_memcpy(row + i, v, sizeof(v));
    }
    return;
  }
  if (Whole) return;
#pragma unroll
  for (int q = 0; q < N; ++q)
    if (i + q < n) row[i + q] = v[q];
}

// Eight rows of eight 16-bit values (four of four in 32 bits) turned.
template <typename T>
__device__ __forceinline__ void turn(vec_t<T> (&x)[kVec<T>]) {
  constexpr int V = kVec<T>;
  vec_t<T> y[V];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) y[i][j] = x[j][i];
  } else {
    u32x4 w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __builtin_bit_cast(u32x4, x[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u32x4 z;
#pragma unroll
      for (int p = 0; p < 4; ++p)
        z[p] = __builtin_amdgcn_perm(w[2 * p + 1][i / 2], w[2 * p][i / 2],
                                     i % 2 ? 0x07060302u : 0x05040100u);
      y[i] = __builtin_bit_cast(vec_t<T>, z);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = y[i];
}

// A factor on its way to the tiles.  The matrix instructions take a lane's 16
// bytes from row lane % 16: loaded so, every lane would be a request of its own (64 a
// load, where 8 lanes of a row make one).  So a wavefront loads rows of adjacent
// chunks of 16 bytes, and turns them over in its own part of LDS, no barrier needed.
// Chunk c of row i lies at c ^ (a few bits of i): both ways touch every bank once.
template <int Chunks>
__device__ __forceinline__ int swizzled(int row, int chunk) {
  constexpr int kMask = Chunks < 8 ? Chunks - 1 : 7, kRows = Chunks < 8 ? 8 / Chunks : 1;
  return row * Chunks + (chunk ^ (row / kRows & kMask));
}
__device__ __forceinline__ void wavefront_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// kRows x kChunks chunks of a map of `rows` x `depth` values, ld apart: rows of
// adjacent values, or (Turned) the values of adjacent rows side by side.  Values
// past the depth are zeros, rows past the last repeat it.
template <typename T, bool Turned, int Fit, int kRows, int kChunks>
struct MapChunks {
  static constexpr int V = kVec<T>, kEach = Turned ? V : 1;
  static constexpr int kTasks = kRows / kEach * kChunks, kTurns = (kTasks + 63) / 64;
  vec_t<T> v[kTurns][kEach];
  __device__ __forceinline__ void load(const T* map, int ld, int rows, int depth, int row0, int k0) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int task = u * 64 + lane;
      if constexpr (Turned) {
        const int row = row0 + task % (kRows / V) * V, k = k0 + task / (kRows / V) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const T* at = map + (int64_t)min(k + j, depth - 1) * ld;
          v[u][j] = load_raw<T, Fit>(at, row, rows);
        }
      } else {
        const int row = row0 + task / kChunks, k = k0 + task % kChunks * V;
        v[u][0] = load_raw<T, Fit>(map + (int64_t)min(row, rows - 1) * ld, k, depth);
      }
    }
  }
  // What lies past the ends, zeros past the depth.
  __device__ __forceinline__ void finish(int rows, int depth, int row0, int k0) {
    if (k0 + kChunks * V <= depth && (!Turned || Fit == kWhole || row0 + kRows <= rows)) return;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int task = u * 64 + lane;
      if constexpr (Turned) {
        const int row = row0 + task % (kRows / V) * V, k = k0 + task / (kRows / V) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (Fit != kWhole) bring<T, Fit>(v[u][j], row, rows);
          if (k + j >= depth) v[u][j] = vec_t<T>{};
        }
      } else {
        bring<T, Fit>(v[u][0], k0 + task % kChunks * V, depth);
      }
    }
  }
  // place(row, chunk): where it lies
  template <typename Place>
  __device__ __forceinline__ void store(u32x4* lds, Place place, int rows, int depth, int row0, int k0) {
    finish(rows, depth, row0, k0);
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
      const int task = u * 64 + lane;
      if (kTasks % 64 != 0 && task >= kTasks) continue;
      if constexpr (Turned) {
        turn<T>(v[u]);
#pragma unroll
        for (int i = 0; i < V; ++i)
          lds[place(task % (kRows / V) * V + i, task / (kRows / V))] = __builtin_bit_cast(u32x4, v[u][i]);
      } else {
        lds[place(task / kChunks, task % kChunks)] = __builtin_bit_cast(u32x4, v[u][0]);
      }
    }
  }
};

// Hidden values of a tile as the second product's factors.  Rank blocks of 16 in
// 32 bits, of 32 in 16 bits, a factor for each part; a single block of 16 ranks is there
// twice instead, for the first two parts side by side and for the halves of the third.
template <typename T, int RT>
struct Hidden {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr bool kBoth = !kWide && RT == 1;
  static constexpr int kBlocks = kWide || RT == 1 ? RT : RT / 2;
  static constexpr int kRow = kWide ? 16 * RT + 4 : 16 * RT + 8;  // of LDS, elements
  static constexpr int kChunks = 16 * RT / kVec<T>;               // of a map's row
  static constexpr int kHeld = kWide ? 1 : kParts;                // in LDS
  static constexpr int kFactors = kWide ? 1 : kBoth ? 2 : kParts;
  using Factor = std::conditional_t<kWide, vec_t<float>, bf16x8>;
  using Element = std::conditional_t<kWide, float, uint16_t>;
  // the map's chunk that a lane's quarter multiplies in rank block k
  static __device__ __forceinline__ int chunk(int k, int quarter) {
    return kBoth ? quarter & 1 : 4 * k + quarter;
  }
  // the part that a lane's quarter has of factor i
  static __device__ __forceinline__ int part(int i, int quarter) {
    return !kBoth ? i : i == 0 ? quarter >> 1 : 2;
  }
};

// acc += h * up for one rank block.
template <typename T, int RT>
__device__ __forceinline__ void mma_hidden(f32x4& acc,
                                           const typename Hidden<T, RT>::Factor (&h)[Hidden<T, RT>::kFactors],
                                           vec_t<T> up) {
  if constexpr (sizeof(T) == 4) {
    mma<float>(acc, h[0], up);
  } else {
    bf16x8 u[kOfMap<T>];
    parts<T>(up, u);
#pragma unroll
    for (int p = 0; p < kOfMap<T>; ++p)
#pragma unroll
      for (int i = 0; i < Hidden<T, RT>::kFactors; ++i) mma<__bf16>(acc, h[i], u[p]);
  }
}

// ---- rows

struct RowsArgs {
  const void* rows;
  int64_t stride;
  int D, E;
  const void* down;  // [K][r][D], or turned: [K][D][r]
  const void* up;    // [K][E][r], or turned: [K][r][E]
  const void* base;  // [rows][E], or null
  float f_hidden, f_out;
  void* out;         // or null: the hidden values only
  float* hidden;     // [rows][r], or null
  float* parts;      // [splits][rows][r]: sums over parts of D
  int splits;
};

// The LDS of a workgroup.
template <typename T, int MT, int RT>
struct RowsLds {
  using H = Hidden<T, RT>;
  static constexpr int V = kVec<T>, M = 16 * MT, R = 16 * RT;
  // columns of a lane in the second product
  static constexpr int kCols = RT >= (sizeof(T) == 4 ? 8 : 4) ? V / 2 : V;
  static constexpr int kFirst = (M + R) * 8, kSecond = 16 * kCols * H::kChunks;  // chunks of a wavefront
  // (the hidden values lie where the first product's factors were: at rank 32 three
  // workgroups of 49 KB a compute unit instead of two of 60)
  union {
    u32x4 first[4][kFirst];
    struct {
      union {
        u32x4 second[4][kSecond];
        float red[2][M][R + 4];
      };
      __attribute__((aligned(16))) typename H::Element hidden[H::kHeld][M][H::kRow];
    };
  };
  int rows[M];
};

// Sums of a wavefront's rows m0 .. m0 + 16 MW over chunks first, first + step, ... of
// D: 128 bytes of each row.
template <typename T, int MW, int RT, bool Turned, int Fit>
__device__ __forceinline__ void first_product(f32x4 (&acc)[MW][RT], const RowsArgs& A, int r,
                                              const T* down, u32x4* stage, const int* ids, int first,
                                              int step) {
  constexpr int V = kVec<T>, kChunk = 8 * V;
  const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const int row = lane >> 3, c = lane & 7;
  const T* x[2 * MW];
#pragma unroll
  for (int i = 0; i < 2 * MW; ++i)
    x[i] = static_cast<const T*>(A.rows) + (int64_t)max(ids[8 * i + row], 0) * A.stride;
  u32x4 *rows_at = stage, *map_at = stage + 16 * MW * 8;
  vec_t<T> v[2 * MW];
  MapChunks<T, Turned, Fit, 16 * RT, 8> map;
  const int ld = Turned ? r : A.D;
  auto load = [&](int at) {
#pragma unroll
    for (int i = 0; i < 2 * MW; ++i) v[i] = load_raw<T, Fit>(x[i], at * kChunk + c * V, A.D);
    map.load(down, ld, r, A.D, 0, at * kChunk);
  };
  int at = first;
  if (at * kChunk < A.D) load(at);
  for (; at * kChunk < A.D; at += step) {
    if ((at + 1) * kChunk > A.D)
#pragma unroll
      for (int i = 0; i < 2 * MW; ++i) bring<T, Fit>(v[i], at * kChunk + c * V, A.D);
#pragma unroll
    for (int i = 0; i < 2 * MW; ++i)
      rows_at[swizzled<8>(8 * i + row, c)] = __builtin_bit_cast(u32x4, v[i]);
    map.store(map_at, swizzled<8>, r, A.D, 0, at * kChunk);
    wavefront_sync();
    if ((at + step) * kChunk < A.D) load(at + step);  // (on its way during the products)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      vec_t<T> a[RT];
#pragma unroll
      for (int k = 0; k < RT; ++k)
        a[k] = __builtin_bit_cast(vec_t<T>, map_at[swizzled<8>(16 * k + col, 4 * u + quarter)]);
#pragma unroll
      for (int m = 0; m < MW; ++m) {
        const auto b = __builtin_bit_cast(vec_t<T>, rows_at[swizzled<8>(16 * m + col, 4 * u + quarter)]);
#pragma unroll
        for (int k = 0; k < RT; ++k) mma<T>(acc[m][k], a[k], b);
      }
    }
    wavefront_sync();
  }
}

// Results of rows m0 .. m0 + 16 MW in column blocks first, first + step, ...: lane l
// has kCols adjacent columns of rows 4 (l / 16) + 0..3, so that 16 lanes write
// 16 kCols adjacent ones.
template <typename T, int MT, int RT, int MW, bool Turned, int Fit>
__device__ __forceinline__ void second_product(const RowsArgs& A, int r, const T* up,
                                               RowsLds<T, MT, RT>& lds, u32x4* stage, int m0,
                                               int count, int first, int step) {
  using L = RowsLds<T, MT, RT>;
  using H = Hidden<T, RT>;
  constexpr int N = L::kCols, kBlock = 16 * N;
  const int lane = threadIdx.x & 63, col = lane & 15, quarter = lane >> 4;
  const T* base = Turned ? nullptr : static_cast<const T*>(A.base);  // (no gradient has one)
  T* out = static_cast<T*>(A.out);
  // (what is read without a base is of the map, which has E values and more, and unused:
  // no branch)
  const T* from = base ? base : up;
  const int64_t from_row = base ? A.E : 0;
  const int ld = Turned ? A.E : r;
  auto place = [](int row, int chunk) {
    const int n = row / N, t = row % N;
    return t * 16 * H::kChunks + swizzled<H::kChunks>(n, chunk);
  };
  MapChunks<T, Turned, Fit, kBlock, H::kChunks> map;
  if (first * kBlock < A.E) map.load(up, ld, A.E, r, first * kBlock, 0);
  for (int at = first; at * kBlock < A.E; at += step) {
    const int e = at * kBlock + N * col;
    T y[2][4][N];
    // (a last block that is not whole takes its values one by one, where they are used)
    const bool cut = Fit != kWhole && (at + 1) * kBlock > A.E;
    auto base_row = [&](int m, int i) {
      return from + max(lds.rows[m0 + 16 * m + 4 * quarter + i], 0) * from_row;
    };
    auto load_base = [&](int m, T (&to)[4][N]) {
      if constexpr (Turned) return;
      if (Fit != kShort || (base && !cut))
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_memcpy(to[i], base_row(m, i) + min(e, A.E - N), sizeof(to[i]));
    };
    load_base(0, y[0]);
    map.store(stage, place, A.E, r, at * kBlock, 0);
    wavefront_sync();
    if ((at + step) * kBlock < A.E) map.load(up, ld, A.E, r, (at + step) * kBlock, 0);
#pragma unroll
    for (int m = 0; m < MW; ++m) {
      if (m + 1 < MW) load_base(m + 1, y[(m + 1) & 1]);
      typename H::Factor h[H::kBlocks][H::kFactors];
      const int row = m0 + 16 * m + col;
#pragma unroll
      for (int k = 0; k < H::kBlocks; ++k)
#pragma unroll
        for (int i = 0; i < H::kFactors; ++i)
          h[k][i] = __builtin_bit_cast(
              typename H::Factor,
              *reinterpret_cast<const u32x4*>(&lds.hidden[H::part(i, quarter)][row][kVec<T> * H::chunk(k, quarter)]));
      f32x4 acc[N];
#pragma unroll
      for (int t = 0; t < N; ++t) {
        acc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < H::kBlocks; ++k)
          mma_hidden<T, RT>(acc[t], h[k],
                            __builtin_bit_cast(vec_t<T>, stage[place(N * col + t, H::chunk(k, quarter))]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = lds.rows[m0 + 16 * m + 4 * quarter + i];
        if (m0 + 16 * m + 4 * quarter + i >= count || n < 0) continue;
        T z[N];
        if (cut && base)
#pragma unroll
          for (int t = 0; t < N; ++t) y[m & 1][i][t] = base_row(m, i)[min(e + t, A.E - 1)];
#pragma unroll
        for (int t = 0; t < N; ++t) {
          const float f = acc[t][i] * A.f_out;
          z[t] = static_cast<T>(base ? to_float(y[m & 1][i][t]) + f : f);
        }
        store_n<N, T, Fit == kWhole>(out + (int64_t)n * A.E, e, A.E, z);
      }
    }
    wavefront_sync();
  }
}

// A tile of rows without a code: base, or zeros; NaN for codes out of range.  ids:
// the rows in LDS, those with codes out of range at -2 - row.
template <typename T, int Fit>
__device__ __forceinline__ void rows_without_code(const RowsArgs& A, const int* ids, int count,
                                                  int part, int parts) {
  constexpr int V = kVec<T>, kAhead = 4;
  const T* base = static_cast<const T*>(A.base);
  T* out = static_cast<T*>(A.out);
  const int vecs = (A.E + V - 1) / V, all = count * vecs, step = kThreads * parts;
  for (int i0 = kThreads * part + threadIdx.x; i0 < all; i0 += step * kAhead) {
    vec_t<T> y[kAhead];
    int n[kAhead], e[kAhead];
    bool bad[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = min(i0 + u * step, all - 1), m = i / vecs;
      e[u] = (i - m * vecs) * V;
      n[u] = ids[m];
      bad[u] = n[u] < -1;
      if (bad[u]) n[u] = -2 - n[u];
      if (base) y[u] = load_raw<T, Fit>(base + (int64_t)max(n[u], 0) * A.E, e[u], A.E);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (base && Fit != kWhole) bring<T, Fit>(y[u], e[u], A.E);
      if (!base || bad[u])
#pragma unroll
        for (int v = 0; v < V; ++v) y[u][v] = static_cast<T>(bad[u] ? __builtin_nanf("") : 0.0f);
      if (n[u] >= 0) store_part<T, Fit == kWhole>(out + (int64_t)n[u] * A.E, e[u], A.E, y[u]);
    }
  }
}

// Wavefronts a SIMD that the compiler keeps room for: three where it takes them without
// spills and would have two registers too many.
template <typename T, int MT, int RT, int Fit>
constexpr int kRowsWaves = MT == 4 && RT == 2 && Fit == kWhole && __is_same(T, __bf16) ? 3 : 2;

// Phase 1: hidden values, over part blockIdx.y of D, left in `parts`; 2: results
// from them, over part blockIdx.y of E; 3: both.  Fit: that of D, E and r.
template <typename T, int MT, int RT, int Phase, bool Turned, int Fit>
__global__ __launch_bounds__(kThreads, (kRowsWaves<T, MT, RT, Fit>)) void adapters_rows_kernel(AdapterParams P, RowsArgs A,
                                                                    Slots S) {
  using L = RowsLds<T, MT, RT>;
  using H = Hidden<T, RT>;
  constexpr int V = kVec<T>, M = L::M, R = L::R;
  __shared__ L lds;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = lane & 15, quarter = lane >> 4;
  // (the last first: those without a code have the most to wait for)
  const Tile t = tile_at(P, S, S.begin + gridDim.x - 1 - xcd_remap(blockIdx.x, gridDim.x));
  if (t.count == 0) return;
  const bool none = t.code >= P.K;
  if (none && (Phase == 1 || A.out == nullptr)) return;
  if (threadIdx.x < M) {
    const int64_t j = t.first + min((int)threadIdx.x, t.count - 1);
    int n = row_at(P, j);
    if (none && n >= 0) {
      const int i = P.order[j];
      if (i < 0 || i >= P.rows || P.places[i] != kNoCode) n = -2 - n;
    }
    lds.rows[threadIdx.x] = n;
  }
  __syncthreads();
  const int parts = Phase == 3 ? 1 : gridDim.y, part = Phase == 3 ? 0 : blockIdx.y;
  if (none) {
    rows_without_code<T, Fit>(A, lds.rows, t.count, part, parts);
    // (the forward's are an output)
    if (!Turned && A.hidden && part == 0)
      for (int i = threadIdx.x; i < t.count * P.r; i += kThreads) A.hidden[t.first * P.r + i] = 0.0f;
    return;
  }

  // Rows of four chunks and more go over the wavefronts by chunks, whose sums meet;
  // shorter ones by tiles.
  const bool by_rows = MT > 1 && A.D <= 3 * 8 * V;
  if constexpr (Phase & 1) {
    const T* down = static_cast<const T*>(A.down) + t.code * P.r * A.D;
    if (by_rows) {
      f32x4 acc[1][RT];
#pragma unroll
      for (int k = 0; k < RT; ++k) acc[0][k] = f32x4{0, 0, 0, 0};
      if (w < MT)
        first_product<T, 1, RT, Turned, Fit>(acc, A, P.r, down, lds.first[w], lds.rows + 16 * w, 0, 1);
      __syncthreads();
      if (w < MT)
#pragma unroll
        for (int k = 0; k < RT; ++k)
          *reinterpret_cast<f32x4*>(&lds.red[0][16 * w + col][16 * k + 4 * quarter]) = acc[0][k];
      __syncthreads();
    } else {
      f32x4 acc[MT][RT];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < RT; ++k) acc[m][k] = f32x4{0, 0, 0, 0};
      first_product<T, MT, RT, Turned, Fit>(acc, A, P.r, down, lds.first[w], lds.rows, w + 4 * part,
                                              4 * parts);
      __syncthreads();
      // Wavefronts 2 and 3's sums to 0 and 1's, whose two are added where they are read.
      auto at = [&](int which, int m, int k) {
        return reinterpret_cast<f32x4*>(&lds.red[which][16 * m + col][16 * k + 4 * quarter]);
      };
      if (w >= 2)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int k = 0; k < RT; ++k) *at(w - 2, m, k) = acc[m][k];
      __syncthreads();
      if (w < 2)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int k = 0; k < RT; ++k) *at(w, m, k) += acc[m][k];
      __syncthreads();
    }
  }
  // Hidden values: summed, kept, and as the next product's factor.
  for (int i = threadIdx.x; i < M * R; i += kThreads) {
    const int m = i / R, k = i % R;
    float h = 0.0f;
    if (m < t.count && k < P.r) {
      const int64_t at = (t.first + m) * P.r + k;
      if constexpr (Phase == 2) {
#pragma unroll 8
        for (int p = 0; p < A.splits; ++p) h += A.parts[p * P.rows * P.r + at];
        h *= A.f_hidden;
        if (A.hidden && part == 0) A.hidden[at] = h;
      } else {
        h = lds.red[0][m][k];
        if (!by_rows) h += lds.red[1][m][k];
        if constexpr (Phase == 1) {
          A.parts[part * P.rows * P.r + at] = h;
        } else {
          h *= A.f_hidden;
          if (A.hidden) A.hidden[at] = h;
        }
      }
    }
    if constexpr (Phase != 1) {
      if constexpr (H::kWide) {
        lds.hidden[0][m][k] = h;
      } else {
        uint32_t part[kParts];
        split(h, part);
        if (H::kBoth) part[2] = __float_as_uint(0.5f * __uint_as_float(part[2] << 16)) >> 16;
#pragma unroll
        for (int i = 0; i < kParts; ++i) lds.hidden[i][m][k] = (uint16_t)part[i];
      }
    }
  }
  if constexpr (Phase != 1) {
    if (A.out == nullptr) return;
    __syncthreads();
    const T* up = static_cast<const T*>(A.up) + t.code * P.r * A.E;
    if (MT > 1 && A.E <= 3 * 16 * L::kCols) {
      if (w < MT)
        second_product<T, MT, RT, 1, Turned, Fit>(A, P.r, up, lds, lds.second[w], 16 * w, t.count, 0, 1);
    } else {
      second_product<T, MT, RT, MT, Turned, Fit>(A, P.r, up, lds, lds.second[w], 0, t.count,
                                                   w + 4 * part, 4 * parts);
    }
  }
}

// ---- gradients of the maps

struct MapsArgs {
  const void* rows[2];     // x and g
  int64_t stride[2];
  int width[2];            // D and E
  const float* hidden[2];  // dh and h
  void* out[2];            // gdown [K][r][D] and gup [K][E][r], either null
  float factor[2];
  float* sums[2];          // [2 rows / L + 2][r * width]: of codes with several chunks
  int blocks[2];           // of columns (0: not wanted)
  int rank_blocks;
};

// Where the sums of chunk `index` of a code with several go: codes with several
// have more than L places, so that twice their starts over L leaves room.
__device__ __forceinline__ int64_t sums_at(int64_t start, int64_t index, int L) {
  return 2 * start / L + index;
}

template <typename T, int RT, int Fit, int Waves>
__global__ __launch_bounds__(64 * Waves) void adapters_maps_kernel(AdapterParams P, MapsArgs A,
                                                                 Slots S) {
  constexpr int V = kVec<T>, W = 16 * V, R = 16 * RT;
  __shared__ __attribute__((aligned(16))) float red[Waves == 1 ? 1 : 2][R][W + 4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = lane & 15, quarter = lane >> 4;
  const int per_slot = (A.blocks[0] + A.blocks[1]) * A.rank_blocks;
  // (a slot's blocks on one XCD: all of them read its hidden values)
  const int block = xcd_remap(blockIdx.x, gridDim.x);
  const int64_t slot = S.begin + block / per_slot;
  int at = block % per_slot;
  const int r0 = at % A.rank_blocks * R;
  at /= A.rank_blocks;
  const int which = at < A.blocks[0] ? 0 : 1;
  const int c0 = (at - (which ? A.blocks[0] : 0)) * W;
  const Tile t = tile_at(P, S, slot);
  if (t.code >= P.K || (t.count == 0 && t.index > 0)) return;
  const int width = A.width[which];
  const int64_t stride = A.stride[which];
  const T* rows = static_cast<const T*>(A.rows[which]);
  const float* hidden = A.hidden[which];
  f32x4 acc[RT][V];
#pragma unroll
  for (int k = 0; k < RT; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[k][v] = f32x4{0, 0, 0, 0};
  const int d = c0 + V * col, end = t.count;  // (places from the tile's first on)
  // A step has kRows places; a lane has kVec of them, each 16 bytes of a row and the
  // hidden values of a rank.  The next step's rows and the places after that are
  // loaded during this step's products.
  constexpr int kRows = 4 * V;
  auto place = [&](int j0, int q) { return sizeof(T) == 4 ? j0 + 4 * q + quarter : j0 + 8 * quarter + q; };
  int n[V];
  vec_t<T> x[V];
  float h[RT][V];
  auto ids = [&](int j0) {
#pragma unroll
    for (int q = 0; q < V; ++q) n[q] = P.order[t.first + min(place(j0, q), end - 1)];
  };
  // (ranks past the last make sums that nobody writes)
  auto load = [&](int j0) {
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int64_t at = t.first + min(place(j0, q), end - 1);
      const int64_t row = P.by_code ? at : (uint32_t)n[q] < (uint32_t)P.rows ? n[q] : 0;
      x[q] = load_raw<T, Fit, true>(rows + row * stride, d, width);
      const float* from = hidden + at * P.r + r0;
#pragma unroll
      for (int k = 0; k < RT; ++k) h[k][q] = from[min(16 * k + col, P.r - 1 - r0)];
    }
  };
  // What stands in for places past the tile's end.  (Only there and only now: a
  // value that is looked at as it is loaded is waited for.)
  auto cut = [&](int j0) {
    if (Fit != kWhole && c0 + W > width)
#pragma unroll
      for (int q = 0; q < V; ++q) bring<T, Fit>(x[q], d, width);
    if (j0 + kRows <= end) return;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      if (place(j0, q) < end) continue;
      x[q] = vec_t<T>{};
#pragma unroll
      for (int k = 0; k < RT; ++k) h[k][q] = 0.0f;
    }
  };
  int j0 = kRows * w;
  if (j0 < end) {
    ids(j0);
    load(j0);
    ids(j0 + Waves * kRows);
  }
  for (; j0 < end; j0 += Waves * kRows) {
    cut(j0);
    if constexpr (sizeof(T) == 4) {
      float g[RT][V];
      vec_t<T> y[V];
#pragma unroll
      for (int q = 0; q < V; ++q) {
        y[q] = x[q];
#pragma unroll
        for (int k = 0; k < RT; ++k) g[k][q] = h[k][q];
      }
      load(j0 + Waves * kRows);  // (the last row again, past the end)
      ids(j0 + 2 * Waves * kRows);
      // (four places a product: 4 q + quarter)
#pragma unroll
      for (int q = 0; q < V; ++q)
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v)
            acc[k][v] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[k][q], y[q][v], acc[k][v], 0, 0, 0);
    } else {
      // (a lane's eight rows turned into eight columns' values)
      vec_t<T> y[V];
#pragma unroll
      for (int q = 0; q < V; ++q) y[q] = x[q];
      turn<T>(y);
      bf16x8 g[RT][kParts];
#pragma unroll
      for (int k = 0; k < RT; ++k) split8(h[k], g[k]);
      load(j0 + Waves * kRows);  // (the last row again, past the end)
      ids(j0 + 2 * Waves * kRows);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        bf16x8 z[kOfMap<T>];
        parts<T>(y[v], z);
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
          for (int p = 0; p < kOfMap<T>; ++p)
#pragma unroll
            for (int i = 0; i < kParts; ++i) mma<__bf16>(acc[k][v], g[k][i], z[p]);
      }
    }
  }
  // Of four, wavefronts 2 and 3's sums to 0 and 1's, whose two are added where they
  // are read.
  auto red_at = [&](int half, int k, int i) { return &red[half][16 * k + 4 * quarter + i][V * col]; };
  if (Waves == 1 || w >= 2)
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < V; v += 4)
          *reinterpret_cast<f32x4*>(red_at(Waves == 1 ? 0 : w - 2, k, i) + v) =
              f32x4{acc[k][v][i], acc[k][v + 1][i], acc[k][v + 2][i], acc[k][v + 3][i]};
  __syncthreads();
  if (Waves > 1 && w < 2)
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int v = 0; v < V; v += 4)
          *reinterpret_cast<f32x4*>(red_at(w, k, i) + v) +=
              f32x4{acc[k][v][i], acc[k][v + 1][i], acc[k][v + 2][i], acc[k][v + 3][i]};
  if (Waves > 1) __syncthreads();
  const int64_t from = start_of(P, t.code), to = start_of(P, t.code + 1);
  const bool alone = to - from <= S.M;
  const int64_t values = (int64_t)P.r * width;
  T* out = static_cast<T*>(A.out[which]) + t.code * values;
  float* sums = alone ? nullptr : A.sums[which] + sums_at(from, t.index, S.M) * values;
  const float factor = A.factor[which];
  // Down's gradient has the columns adjacent, up's the ranks: kVec of them a thread.
  constexpr int kAcross = R / V;
  for (int i = threadIdx.x; i < R * 16; i += 64 * Waves) {
    const int k = which ? i % kAcross * V : i / 16, c = which ? i / kAcross : i % 16 * V;
    if (r0 + k >= P.r || c0 + c >= width) continue;
    float f[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int y = which ? k + v : k, x = which ? c : c + v;
      f[v] = (Waves == 1 ? red[0][y][x] : red[0][y][x] + red[Waves > 1][y][x]) * factor;
    }
    const int first = which ? r0 + k : c0 + c, n = which ? P.r : width;
    const int64_t row = (int64_t)(which ? c0 + c : r0 + k) * n;
    if (alone) {
      vec_t<T> z;
#pragma unroll
      for (int v = 0; v < V; ++v) z[v] = static_cast<T>(f[v]);
      store_part(out + row, first, n, z);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (first + v < n) sums[row + first + v] = f[v];
    }
  }
}

// The chunks' sums of the codes that have several, in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapters_join_kernel(AdapterParams P, MapsArgs A,
                                                                 Slots S) {
  const Tile t = tile_at(P, S, S.begin + blockIdx.x);
  if (t.code >= P.K || t.index > 0) return;
  const int64_t from = start_of(P, t.code), to = start_of(P, t.code + 1);
  if (to - from <= S.M) return;
  const int64_t chunks = (to - from + S.M - 1) / S.M;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (A.blocks[which] == 0) continue;
    const int64_t values = (int64_t)P.r * A.width[which];
    const float* sums = A.sums[which] + sums_at(from, 0, S.M) * values;
    T* out = static_cast<T*>(A.out[which]) + t.code * values;
    for (int64_t i = blockIdx.y * kThreads + threadIdx.x; i < values; i += gridDim.y * kThreads) {
      float a = 0.0f;
#pragma unroll 8
      for (int64_t c = 0; c < chunks; ++c) a += sums[c * values + i];
      out[i] = static_cast<T>(a);
    }
  }
}

// ---- host

// Rank tiles, a power of two of 16 ranks.
int rank_tiles(int r) { return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : 8; }

// How rows go: tiles of 16 * row_tiles places; splits > 1: hidden values and
// results in launches of their own, each over parts of a row.
//
// Tiles, us of a forward of 131072 rows in tiles of 16 and of 64 places, by the rows a
// code has on average: bfloat16 128 -> 59, rank 8: 16 rows 77 and 97, 32 rows 62 and 57,
// 256 rows 44 and 34; 1024 -> 1024, rank 32: 381 and 381, 274 and 272, 194 and 181; floats
// 128 -> 59: 70 and 108, 57 and 63, 42 and 39.  The rows' gradient gains more (bfloat16 at
// 1024: 336 and 328, 236 and 219, 184 and 136).  Fewer rows, 256 a code: 32768 rows 14.4
// and 11.9, 8192 rows 7.6 and 8.1.
//
// Splits, us of a forward at rank 16 in one launch and in two: bfloat16, one row of
// 1024 -> 1024 6.2 and 7.6, of 2048 8.9 and 7.3, of 4096 14.3 and 7.8; 256 rows 8.0 and
// 9.2, 12.0 and 9.0, 19.9 and 10.8; 4000 rows 9.6 and 11.9, 16.6 and 16.8, 28.5 and 26.1.
// Floats of 1024 gain too (9.1 and 7.2), but the second launch takes the host 3 us.
struct RowsPlan {
  int row_tiles, splits_down, splits_up;
};
RowsPlan rows_plan(const AdapterParams& P, int D, int E) {
  RowsPlan L{4, 1, 1};
  if (rank_tiles(P.r) < 8 && P.rows >= 32 * (int64_t)P.K && P.rows >= 512 * 64) return L;
  L.row_tiles = 1;
  const int64_t tiles = std::min<int64_t>(P.rows, P.rows / 16 + P.K);
  if (tiles < 512 && std::max(D, E) >= 2048) {
    const int64_t most = 512 / std::max<int64_t>(tiles, 1) + 1;
    // (a chunk of a row, a block of columns for each of the four wavefronts)
    const int wide = P.dtype == GSPLAT_F32 ? 1 : 2;
    L.splits_down = (int)std::clamp<int64_t>(D / (128 * wide), 1, most);
    L.splits_up = (int)std::clamp<int64_t>(E / (256 * wide), 1, most);
  }
  return L;
}
bool is_split(const RowsPlan& L) { return L.splits_down > 1 || L.splits_up > 1; }

template <typename T, int MT, int RT, int Phase, bool Turned, int Fit>
int launch_rows(const AdapterParams& P, const RowsArgs& A, int parts, hipStream_t stream) {
  Slots S{16 * MT, by_place(P, 16 * MT), 0};
  return in_launches(slots_of(P, S.M, S.by_place), kMostBlocks, [&](int64_t first, int64_t n) {
    S.begin = first;
    launch_traced("adapters_rows_kernel", (adapters_rows_kernel<T, MT, RT, Phase, Turned, Fit>),
                  dim3((unsigned)n, parts), dim3(kThreads), 0, stream, P, A, S);
    return check_launch("adapters_rows_kernel");
  });
}

template <typename T, int RT, bool Turned, int Fit>
int rows_of_rank(const AdapterParams& P, RowsArgs A, const RowsPlan& L, hipStream_t stream) {
  if (is_split(L)) {
    const int rc = launch_rows<T, 1, RT, 1, Turned, Fit>(P, A, L.splits_down, stream);
    return rc ? rc : launch_rows<T, 1, RT, 2, Turned, Fit>(P, A, A.out ? L.splits_up : 1, stream);
  }
  if constexpr (RT < 8)
    if (L.row_tiles > 1) return launch_rows<T, 4, RT, 3, Turned, Fit>(P, A, 1, stream);
  return launch_rows<T, 1, RT, 3, Turned, Fit>(P, A, 1, stream);
}

template <typename T, bool Turned>
int rows_of(const AdapterParams& P, RowsArgs A, float* parts, hipStream_t stream) {
  const RowsPlan L = rows_plan(P, A.D, A.E);
  A.parts = parts;
  A.splits = L.splits_down;
  const int fit = fit_of({A.D, A.E, P.r}, kVec<T>);
  switch (rank_tiles(P.r)) {
#define GS_RANK(RT)                                                           \
  case RT:                                                                    \
    return fit == kWhole    ? rows_of_rank<T, RT, Turned, kWhole>(P, A, L, stream)  \
           : fit == kRagged ? rows_of_rank<T, RT, Turned, kRagged>(P, A, L, stream) \
                            : rows_of_rank<T, RT, Turned, kShort>(P, A, L, stream);
    GS_RANK(1) GS_RANK(2) GS_RANK(4)
    default: GS_RANK(8)
#undef GS_RANK
  }
}

// Places of a chunk: enough workgroups for the card, and sums that are few beside
// the rows they come from (4 r / (places * bytes of a value) of them: at 512 places and
// rank 32 in 16 bits an eighth).  Both gradients in bfloat16, us in chunks of 256, 512,
// 1024, 2048 and 4096 places (in brackets the one taken): 131072 rows of 1024 -> 1024,
// rank 32, 256 codes 337 267 189 (188) 187, 8 codes 362 260 218 (205) 248, one code 848
// 516 340 (260) 236; 128 -> 128, rank 16, 256 codes 69 (65) 49 49 49, 8 codes 55 (52) 47
// 51 70; 16384 rows of 128 -> 128, 8 codes 20 (22) 25 33 31; 65536 rows of 256 -> 256, rank
// 128, 8 codes 260 (203) 181 205 182.
int chunk_of(const AdapterParams& P, int dtype_bytes) {
  const int64_t blocks = (P.D + P.E) * dtype_bytes / 256 + 1;
  int L = 512;
  while (L < 65536 && P.rows * blocks > (int64_t)L * 2048) L *= 2;
  return L;
}

struct BackwardLayout {
  size_t dh, parts, sums[2], total;
  int chunk;
};
BackwardLayout backward_layout(const AdapterParams& P) {
  BackwardLayout L{};
  const int bytes = P.dtype == GSPLAT_F32 ? 4 : 2;
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t at = off;
    off += align_up(n, 256);
    return at;
  };
  L.chunk = chunk_of(P, bytes);
  L.dh = take((size_t)P.rows * P.r * 4);
  const RowsPlan R = rows_plan(P, P.E, P.D);
  L.parts = take(is_split(R) ? (size_t)R.splits_down * P.rows * P.r * 4 : 0);
  if (P.rows > L.chunk) {
    const size_t n = (size_t)(2 * P.rows / L.chunk + 2) * P.r * 4;
    L.sums[0] = take(n * P.D);
    L.sums[1] = take(n * P.E);
  }
  L.total = off;
  return L;
}

}  // namespace

// A file of its own for each type (they are compiled side by side).
template <typename T>
int adapters_forward_of(const AdapterParams& P, const void* rows, const void* down,
               const void* up, const void* base, void* out, float* hidden,
               void* workspace, hipStream_t stream) {
  return rows_of<T, false>(P, RowsArgs{rows, P.stride, P.D, P.E, down, up, base, 1.0f, P.scale, out,
                                       hidden, nullptr, 0},
                           static_cast<float*>(workspace), stream);
}

template <typename T>
int adapters_backward_of(const AdapterParams& P, const void* grad, const void* rows,
                const void* down, const void* up, const float* hidden,
                void* g_rows, void* g_down, void* g_up, void* workspace,
                hipStream_t stream) {
  char* ws = static_cast<char*>(workspace);
  const BackwardLayout L = backward_layout(P);
  auto* dh = reinterpret_cast<float*>(ws + L.dh);
  int rc = GSPLAT_OK;
  if ((g_rows || g_down) && P.rows > 0) {
    rc = rows_of<T, true>(P, RowsArgs{grad, P.E, P.E, P.D, up, down, nullptr, P.scale, 1.0f, g_rows,
                                      dh, nullptr, 0},
                          reinterpret_cast<float*>(ws + L.parts), stream);
    if (rc) return rc;
  }
  if (!g_down && !g_up) return rc;
  constexpr int W = 16 * kVec<T>;
  const int rt = std::min(rank_tiles(P.r), 4);
  const MapsArgs A{{rows, grad}, {P.stride, P.E}, {P.D, P.E}, {dh, hidden}, {g_down, g_up},
                   {1.0f, P.scale},
                   {reinterpret_cast<float*>(ws + L.sums[0]), reinterpret_cast<float*>(ws + L.sums[1])},
                   {g_down ? (P.D + W - 1) / W : 0, g_up ? (P.E + W - 1) / W : 0},
                   rank_tiles(P.r) == 8 ? 2 : 1};
  const int fit = fit_of({P.D, P.E}, kVec<T>);
  // One wavefront a workgroup where that makes enough of them: nothing to join.  us in
  // four and in one, by the number below, bfloat16 of rank 32: 131072 rows of 1024 -> 1024,
  // 64 codes (2048) 219 and 253, 256 codes (5120) 195 and 187, 1024 codes (17408) 348 and
  // 240; 128 -> 128, 256 codes (1024) 77 and 87, 4096 codes (4096) 207 and 144; floats
  // 512 -> 512, 16384 rows: 64 codes (1536) 50 and 56, 256 codes (4096) 64 and 54.
  const bool single = std::min<int64_t>(P.rows / 64, P.K + P.rows / L.chunk) *
                          (A.blocks[0] + A.blocks[1]) * A.rank_blocks >= 4096;
  Slots S{L.chunk, false, 0};
  const int64_t slots = P.rows / L.chunk + P.K;
  const int per_slot = (A.blocks[0] + A.blocks[1]) * A.rank_blocks;
  rc = in_launches(slots, kMostBlocks / per_slot, [&](int64_t first, int64_t n) {
    S.begin = first;
    const dim3 grid((unsigned)(n * per_slot));
#define GS_MAPS_OF(RT, FIT, WAVES)                                                      \
  launch_traced("adapters_maps_kernel", (adapters_maps_kernel<T, RT, FIT, WAVES>), grid, \
                dim3(64 * WAVES), 0, stream, P, A, S)
#define GS_MAPS_FIT(RT, FIT)                \
  if (rt == RT && fit == FIT) {             \
    if (single) GS_MAPS_OF(RT, FIT, 1);     \
    else GS_MAPS_OF(RT, FIT, 4);            \
  }
#define GS_MAPS(RT) GS_MAPS_FIT(RT, kWhole) GS_MAPS_FIT(RT, kRagged) GS_MAPS_FIT(RT, kShort)
    GS_MAPS(1) GS_MAPS(2) GS_MAPS(4)
#undef GS_MAPS
#undef GS_MAPS_FIT
#undef GS_MAPS_OF
    return check_launch("adapters_maps_kernel");
  });
  if (rc || P.rows <= L.chunk) return rc;
  return in_launches(slots, kMostBlocks, [&](int64_t first, int64_t n) {
    S.begin = first;
    launch_traced("adapters_join_kernel", (adapters_join_kernel<T>), dim3((unsigned)n, 8),
                  dim3(kThreads), 0, stream, P, A, S);
    return check_launch("adapters_join_kernel");
  });
}

}  // namespace gs
