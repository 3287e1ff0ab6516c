// code_adapters.hip -- low-rank maps of splats' rows, each by its code's own.
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
// the rows is the same with up^T and down^T, laid out by a launch before it.
// Gradients of the maps: a workgroup takes up to L places of a code and a block
// of columns; longer codes' sums are joined by another launch, in order.
//
// Everything is a matrix product of 16 x 16 tiles.  In 16 bits the hidden values
// go into the second product as two bfloat16, h = hi + lo (16 bits of them, so
// that the result's rounding is the only one that counts), and float16 factors
// beside them as two bfloat16 too, exactly: hidden values have no range to leave.
#include <algorithm>

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

// A lane's 16 bytes of a factor: row lane % 16, values 4 v + ... of the quarter
// lane / 16.  A product of two takes 4 * kVec values of the rows; lane l has its
// elements 4 (l / 16) + 0..3 of column l % 16.
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

// x = hi + lo, the larger part cut off after 8 bits (it stays in range), the
// smaller one rounded to 8; an infinity has no smaller part.
__device__ __forceinline__ void split(float x, uint32_t& hi, float& lo) {
  const uint32_t u = __float_as_uint(x);
  hi = u >> 16;
  lo = x - __uint_as_float(u & 0xffff0000u);
  if ((u & 0x7f800000u) == 0x7f800000u) lo = 0.0f;
}
__device__ __forceinline__ uint32_t bf16_bits(float x) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
}
__device__ __forceinline__ void split8(const float (&x)[8], bf16x8& hi, bf16x8& lo) {
  u32x4 h, l;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    uint32_t h0, h1;
    float l0, l1;
    split(x[2 * p], h0, l0);
    split(x[2 * p + 1], h1, l1);
    h[p] = h0 | h1 << 16;
    l[p] = bf16_bits(l0) | bf16_bits(l1) << 16;
  }
  hi = __builtin_bit_cast(bf16x8, h);
  lo = __builtin_bit_cast(bf16x8, l);
}
// Eight values of a map or a row as bfloat16: themselves, or a float16's two parts.
template <typename T>
__device__ __forceinline__ void parts(vec_t<T> x, bf16x8& hi, bf16x8& lo) {
  if constexpr (__is_same(T, __bf16)) {
    hi = x;
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_float(x[i]);
    split8(f, hi, lo);
  }
}

// Hidden values of a tile as the second product's factor.  Rank blocks of 16 in
// 32 bits, of 32 in 16 bits; a single block of 16 ranks holds hi and lo side by
// side instead.
template <typename T, int RT>
struct Hidden {
  static constexpr bool kWide = sizeof(T) == 4;
  static constexpr bool kBoth = !kWide && RT == 1;
  static constexpr int kBlocks = kWide || RT == 1 ? RT : RT / 2;
  static constexpr int kRow = kWide ? 16 * RT + 4 : 16 * RT + 8;  // of LDS, elements
  using Factor = std::conditional_t<kWide, vec_t<float>, bf16x8>;
};

// acc += up * h for one rank block.
template <typename T, int RT>
__device__ __forceinline__ void mma_hidden(f32x4& acc, vec_t<T> up,
                                           typename Hidden<T, RT>::Factor hi,
                                           typename Hidden<T, RT>::Factor lo) {
  if constexpr (sizeof(T) == 4) {
    mma<float>(acc, up, hi);
  } else {
    bf16x8 u, v;
    parts<T>(up, u, v);
    mma<__bf16>(acc, u, hi);
    if constexpr (RT > 1) mma<__bf16>(acc, u, lo);
    if constexpr (!__is_same(T, __bf16)) mma<__bf16>(acc, v, hi);
  }
}

// ---- rows

struct RowsArgs {
  const void* rows;
  int64_t stride;
  int D, E;
  const void* down;  // [K][r][D]
  const void* up;    // [K][E][r]
  const void* base;  // [rows][E], or null
  float f_hidden, f_out;
  void* out;         // or null: the hidden values only
  float* hidden;     // [rows][r], or null
  float* parts;      // [splits][rows][r]: sums over parts of D
  int splits;
};

// Phase 1: hidden values, over part blockIdx.y of D, left in `parts`; 2: results
// from them, over part blockIdx.y of E; 3: both.
template <typename T, int MT, int RT, int Phase>
__global__ __launch_bounds__(kThreads) void adapters_rows_kernel(AdapterParams P, RowsArgs A,
                                                                 Slots S) {
  using H = Hidden<T, RT>;
  constexpr int V = kVec<T>, M = 16 * MT, R = 16 * RT, kStep = 4 * V, kPad = R + 4;
  __shared__ __attribute__((aligned(16))) float red[2][M][kPad];
  __shared__ __attribute__((aligned(16))) uint16_t parts16[H::kWide ? 1 : 2][H::kWide ? 1 : M][H::kWide ? 8 : H::kRow];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = lane & 15, quarter = lane >> 4;
  const Tile t = tile_at(P, S, S.begin + xcd_remap(blockIdx.x, gridDim.x));
  if (t.count == 0) return;
  const T* rows = static_cast<const T*>(A.rows);
  if (t.code >= P.K) {  // without a code
    if (Phase == 1 || A.out == nullptr) return;
    const T* base = static_cast<const T*>(A.base);
    T* out = static_cast<T*>(A.out);
    const int step = kThreads * (Phase == 2 ? gridDim.y : 1);
    for (int m = 0; m < t.count; ++m) {
      const int64_t j = t.first + m;
      const int i = P.order[j], n = row_at(P, j);
      if (n < 0) continue;
      const float rest =
          i >= 0 && i < P.rows && P.places[i] == kNoCode ? 0.0f : __builtin_nanf("");
      for (int e = (Phase == 2 ? blockIdx.y * kThreads : 0) + threadIdx.x; e < A.E; e += step)
        out[(int64_t)n * A.E + e] =
            base && rest == 0.0f ? base[(int64_t)n * A.E + e] : static_cast<T>(rest);
    }
    return;
  }
  int n[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) n[m] = row_at(P, t.first + min(16 * m + col, t.count - 1));

  if constexpr (Phase & 1) {
    f32x4 acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int k = 0; k < RT; ++k) acc[m][k] = f32x4{0, 0, 0, 0};
    const T *x[MT], *d[RT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = rows + (int64_t)max(n[m], 0) * A.stride;
    const T* down = static_cast<const T*>(A.down) + t.code * P.r * A.D;
#pragma unroll
    for (int k = 0; k < RT; ++k) d[k] = down + (int64_t)min(16 * k + col, P.r - 1) * A.D;
    constexpr int U = MT * RT > 8 ? 1 : MT + RT > 4 ? 2 : 4;
    const int full = A.D / kStep, turn = 4 * (Phase == 1 ? gridDim.y : 1);
    int s = w + 4 * (Phase == 1 ? blockIdx.y : 0);
    for (; s + (U - 1) * turn < full; s += U * turn) {
      vec_t<T> a[U][RT], b[U][MT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = (s + u * turn) * kStep + quarter * V;
#pragma unroll
        for (int m = 0; m < MT; ++m) b[u][m] = load_vec(x[m] + at);
#pragma unroll
        for (int k = 0; k < RT; ++k) a[u][k] = load_vec(d[k] + at);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int k = 0; k < RT; ++k) mma<T>(acc[m][k], a[u][k], b[u][m]);
    }
    for (; s * kStep < A.D; s += turn) {
      const int at = s * kStep + quarter * V;
      vec_t<T> a[RT], b[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) b[m] = load_part(x[m], at, A.D, static_cast<T>(0.0f));
#pragma unroll
      for (int k = 0; k < RT; ++k) a[k] = load_part(d[k], at, A.D, static_cast<T>(0.0f));
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < RT; ++k) mma<T>(acc[m][k], a[k], b[m]);
    }
    // The wavefronts' sums: 2 and 3 to 0 and 1, whose two are added where they are read.
    auto at = [&](int which, int m, int k) {
      return reinterpret_cast<f32x4*>(&red[which][16 * m + col][16 * k + 4 * quarter]);
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
  // Hidden values: summed, kept, and as the next product's factor.
  for (int i = threadIdx.x; i < M * R; i += kThreads) {
    const int m = i / R, k = i % R;
    float h = 0.0f;
    if (m < t.count && k < P.r) {
      const int64_t at = (t.first + m) * P.r + k;
      if constexpr (Phase == 2) {
        for (int p = 0; p < A.splits; ++p) h += A.parts[p * P.rows * P.r + at];
        h *= A.f_hidden;
        if (A.hidden && blockIdx.y == 0) A.hidden[at] = h;
      } else {
        h = red[0][m][k] + red[1][m][k];
        if constexpr (Phase == 1) {
          A.parts[blockIdx.y * P.rows * P.r + at] = h;
        } else {
          h *= A.f_hidden;
          if (A.hidden) A.hidden[at] = h;
        }
      }
    }
    if constexpr (Phase != 1) {
      if constexpr (H::kWide) {
        red[0][m][k] = h;
      } else {
        uint32_t hi;
        float lo;
        split(h, hi, lo);
        parts16[0][m][k] = (uint16_t)hi;
        parts16[1][m][k] = (uint16_t)bf16_bits(lo);
      }
    }
  }
  if constexpr (Phase != 1) {
    if (A.out == nullptr) return;
    __syncthreads();
    typename H::Factor hi[MT][H::kBlocks], lo[MT][H::kBlocks];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int k = 0; k < H::kBlocks; ++k) {
        const int row = 16 * m + col;
        if constexpr (H::kWide) {
          hi[m][k] = load_vec(&red[0][row][16 * k + 4 * quarter]);
        } else if constexpr (H::kBoth) {
          hi[m][k] = __builtin_bit_cast(
              bf16x8, *reinterpret_cast<const u32x4*>(&parts16[quarter >> 1][row][8 * (quarter & 1)]));
        } else {
          hi[m][k] = __builtin_bit_cast(
              bf16x8, *reinterpret_cast<const u32x4*>(&parts16[0][row][32 * k + 8 * quarter]));
          lo[m][k] = __builtin_bit_cast(
              bf16x8, *reinterpret_cast<const u32x4*>(&parts16[1][row][32 * k + 8 * quarter]));
        }
      }
    // 32 columns at a time: lane l's results are columns 8 (l / 16) + 0..7 of row
    // l % 16, four of either of two tiles.
    const T* up = static_cast<const T*>(A.up) + t.code * P.r * A.E;
    const T* base = static_cast<const T*>(A.base);
    T* out = static_cast<T*>(A.out);
    const int turn = 128 * (Phase == 2 ? gridDim.y : 1);
    for (int c0 = 32 * (w + 4 * (Phase == 2 ? blockIdx.y : 0)); c0 < A.E; c0 += turn) {
      f32x4 acc[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int e = min(c0 + 8 * (col >> 2) + 4 * v + (col & 3), A.E - 1);
        const T* row = up + (int64_t)e * P.r;
#pragma unroll
        for (int k = 0; k < H::kBlocks; ++k) {
          const int rank = H::kWide ? 16 * k + 4 * quarter
                                    : H::kBoth ? 8 * (quarter & 1) : 32 * k + 8 * quarter;
          const vec_t<T> u = load_part(row, rank, P.r, static_cast<T>(0.0f));
#pragma unroll
          for (int m = 0; m < MT; ++m) mma_hidden<T, RT>(acc[m][v], u, hi[m][k], lo[m][k]);
        }
      }
      const int e = c0 + 8 * quarter;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (16 * m + col >= t.count || n[m] < 0) continue;
        T* to = out + (int64_t)n[m] * A.E;
        const T* from = base + (int64_t)n[m] * A.E;
#pragma unroll
        for (int v = 0; v < 8 / V; ++v) {
          const int first = e + v * V;
          vec_t<T> y;
          if (base) y = load_part(from, first, A.E, static_cast<T>(0.0f));
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int q = v * V + i;
            const float z = acc[m][q / 4][q % 4] * A.f_out;
            y[i] = static_cast<T>(base ? to_float(y[i]) + z : z);
          }
          store_part(to, first, A.E, y);
        }
      }
    }
  }
}

// Maps transposed, [K][a][b] -> [K][b][a], of the codes that have places.
template <typename T>
__global__ __launch_bounds__(kThreads) void adapters_transpose_kernel(
    AdapterParams P, const T* __restrict__ from, T* __restrict__ to, int a, int b,
    int64_t first_code) {
  __shared__ T tile[32][34];
  const int64_t across = (b + 31) / 32, down = (a + 31) / 32, tiles = across * down;
  const int64_t i = blockIdx.x % tiles, k = first_code + blockIdx.x / tiles;
  if (start_of(P, k) >= start_of(P, k + 1)) return;
  const int a0 = (int)(i / across) * 32, b0 = (int)(i % across) * 32;
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  from += k * a * b;
  to += k * a * b;
  for (int v = y; v < 32; v += 8)
    if (a0 + v < a && b0 + x < b) tile[v][x] = from[(int64_t)(a0 + v) * b + b0 + x];
  __syncthreads();
  for (int v = y; v < 32; v += 8)
    if (b0 + v < b && a0 + x < a) to[(int64_t)(b0 + v) * a + a0 + x] = tile[x][v];
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

template <typename T, int RT>
__global__ __launch_bounds__(kThreads) void adapters_maps_kernel(AdapterParams P, MapsArgs A,
                                                                 Slots S) {
  constexpr int V = kVec<T>, W = 16 * V, R = 16 * RT;
  __shared__ __attribute__((aligned(16))) float red[R][W + 4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int col = lane & 15, quarter = lane >> 4;
  const int per_slot = (A.blocks[0] + A.blocks[1]) * A.rank_blocks;
  const int64_t slot = S.begin + blockIdx.x / per_slot;
  int at = (int)(blockIdx.x % per_slot);
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
  const int d = c0 + V * col;
  const int64_t end = t.first + t.count;
  if constexpr (sizeof(T) == 4) {
    // A step is 16 places, four a product: place 4 u + quarter.
    for (int64_t j0 = t.first + 16 * w; j0 < end; j0 += 64) {
      vec_t<T> x[4];
      float h[4][RT];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t j = j0 + 4 * u + quarter, safe = min(j, end - 1);
        const int n = row_at(P, safe);
        const bool in = j < end && n >= 0;
        x[u] = load_part(rows + (int64_t)max(n, 0) * stride, d, width, 0.0f);
        if (!in) x[u] = vec_t<T>{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < RT; ++k) {
          const int rank = r0 + 16 * k + col;
          h[u][k] = in && rank < P.r ? hidden[safe * P.r + rank] : 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int k = 0; k < RT; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v)
            acc[k][v] =
                __builtin_amdgcn_mfma_f32_16x16x4f32(h[u][k], x[u][v], acc[k][v], 0, 0, 0);
    }
  } else {
    // A step is 32 places: a lane's eight rows, places 8 quarter + 0..7, turned
    // into eight columns' values.
    for (int64_t j0 = t.first + 32 * w; j0 < end; j0 += 128) {
      u32x4 x[8];
      bool in[8];
      int64_t safe[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int64_t j = j0 + 8 * quarter + q;
        safe[q] = min(j, end - 1);
        const int n = row_at(P, safe[q]);
        in[q] = j < end && n >= 0;
        x[q] = __builtin_bit_cast(
            u32x4, load_part(rows + (int64_t)max(n, 0) * stride, d, width, static_cast<T>(0.0f)));
        if (!in[q]) x[q] = u32x4{0, 0, 0, 0};
      }
      bf16x8 hi[RT], lo[RT];
#pragma unroll
      for (int k = 0; k < RT; ++k) {
        const int rank = r0 + 16 * k + col;
        float h[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          h[q] = in[q] && rank < P.r ? hidden[safe[q] * P.r + rank] : 0.0f;
        split8(h, hi[k], lo[k]);
      }
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        u32x4 y;
#pragma unroll
        for (int p = 0; p < 4; ++p)
          y[p] = __builtin_amdgcn_perm(x[2 * p + 1][v / 2], x[2 * p][v / 2],
                                       v % 2 ? 0x07060302u : 0x05040100u);
        bf16x8 big, small;
        parts<T>(__builtin_bit_cast(vec_t<T>, y), big, small);
#pragma unroll
        for (int k = 0; k < RT; ++k) {
          mma<__bf16>(acc[k][v], hi[k], big);
          mma<__bf16>(acc[k][v], lo[k], big);
          if constexpr (!__is_same(T, __bf16)) mma<__bf16>(acc[k][v], hi[k], small);
        }
      }
    }
  }
  // The wavefronts' sums, one after another.
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (w == u)
#pragma unroll
      for (int k = 0; k < RT; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            float& s = red[16 * k + 4 * quarter + i][V * col + v];
            s = u == 0 ? acc[k][v][i] : s + acc[k][v][i];
          }
    __syncthreads();
  }
  const int64_t from = start_of(P, t.code), to = start_of(P, t.code + 1);
  const int ranks = min(R, P.r - r0), cols = min(W, width - c0);
  const bool alone = to - from <= S.M;
  const int64_t values = (int64_t)P.r * width;
  T* out = static_cast<T*>(A.out[which]) + t.code * values;
  float* sums = alone ? nullptr : A.sums[which] + sums_at(from, t.index, S.M) * values;
  for (int i = threadIdx.x; i < ranks * cols; i += kThreads) {
    // down's gradient has the columns adjacent, up's the ranks
    const int k = which ? i % ranks : i / cols, c = which ? i / ranks : i % cols;
    const int64_t to_at = which ? (int64_t)(c0 + c) * P.r + r0 + k : (int64_t)(r0 + k) * width + c0 + c;
    const float v = red[k][c] * A.factor[which];
    if (alone) out[to_at] = static_cast<T>(v);
    else sums[to_at] = v;
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
struct RowsPlan {
  int row_tiles, splits_down, splits_up;
};
RowsPlan rows_plan(const AdapterParams& P, int D, int E) {
  const int big = rank_tiles(P.r) == 8 ? 2 : 4;
  RowsPlan L{big, 1, 1};
  if (P.rows >= 32 * (int64_t)P.K && P.rows >= 512 * 16 * big) return L;
  L.row_tiles = 1;
  const int64_t tiles = std::min<int64_t>(P.rows, P.rows / 16 + P.K);
  if (tiles < 512 && std::max(D, E) >= 1024) {
    const int64_t most = 512 / std::max<int64_t>(tiles, 1) + 1;
    L.splits_down = (int)std::clamp<int64_t>(D / 256, 1, most);
    L.splits_up = (int)std::clamp<int64_t>(E / 256, 1, most);
  }
  return L;
}
bool is_split(const RowsPlan& L) { return L.splits_down > 1 || L.splits_up > 1; }

template <typename T, int MT, int RT, int Phase>
int launch_rows(const AdapterParams& P, const RowsArgs& A, int parts, hipStream_t stream) {
  Slots S{16 * MT, by_place(P, 16 * MT), 0};
  return in_launches(slots_of(P, S.M, S.by_place), kMostBlocks, [&](int64_t first, int64_t n) {
    S.begin = first;
    launch_traced("adapters_rows_kernel", (adapters_rows_kernel<T, MT, RT, Phase>),
                  dim3((unsigned)n, parts), dim3(kThreads), 0, stream, P, A, S);
    return check_launch("adapters_rows_kernel");
  });
}

template <typename T>
int rows_of(const AdapterParams& P, RowsArgs A, float* parts, hipStream_t stream) {
  const RowsPlan L = rows_plan(P, A.D, A.E);
  const int rt = rank_tiles(P.r);
  if (is_split(L)) {
    A.parts = parts;
    A.splits = L.splits_down;
#define GS_SPLIT(RT)                                                                   \
  if (rt == RT) {                                                                      \
    const int rc = launch_rows<T, 1, RT, 1>(P, A, L.splits_down, stream);              \
    return rc ? rc : launch_rows<T, 1, RT, 2>(P, A, A.out ? L.splits_up : 1, stream);  \
  }
    GS_SPLIT(1) GS_SPLIT(2) GS_SPLIT(4) GS_SPLIT(8)
#undef GS_SPLIT
  }
  if (L.row_tiles == 1) {
    if (rt == 1) return launch_rows<T, 1, 1, 3>(P, A, 1, stream);
    if (rt == 2) return launch_rows<T, 1, 2, 3>(P, A, 1, stream);
    if (rt == 4) return launch_rows<T, 1, 4, 3>(P, A, 1, stream);
    return launch_rows<T, 1, 8, 3>(P, A, 1, stream);
  }
  if (rt == 1) return launch_rows<T, 4, 1, 3>(P, A, 1, stream);
  if (rt == 2) return launch_rows<T, 4, 2, 3>(P, A, 1, stream);
  if (rt == 4) return launch_rows<T, 4, 4, 3>(P, A, 1, stream);
  return launch_rows<T, 2, 8, 3>(P, A, 1, stream);
}

template <typename T>
int forward_of(const AdapterParams& P, const void* rows, const void* down,
               const void* up, const void* base, void* out, float* hidden,
               void* workspace, hipStream_t stream) {
  return rows_of<T>(P, RowsArgs{rows, P.stride, P.D, P.E, down, up, base, 1.0f, P.scale, out,
                                hidden, nullptr, 0},
                    static_cast<float*>(workspace), stream);
}

// Places of a chunk: enough workgroups for the card, and sums that are few beside
// the rows they come from.
int chunk_of(const AdapterParams& P, int dtype_bytes) {
  const int64_t blocks = (P.D + P.E) * dtype_bytes / 256 + 1;
  int L = 512;
  while (L < 8192 && P.rows * blocks > (int64_t)L * 2048) L *= 2;
  return L;
}

struct BackwardLayout {
  size_t dh, parts, down_t, up_t, sums[2], total;
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
  L.down_t = take((size_t)P.K * P.r * P.D * bytes);
  L.up_t = take((size_t)P.K * P.r * P.E * bytes);
  if (P.rows > L.chunk) {
    const size_t n = (size_t)(2 * P.rows / L.chunk + 2) * P.r * 4;
    L.sums[0] = take(n * P.D);
    L.sums[1] = take(n * P.E);
  }
  L.total = off;
  return L;
}

template <typename T>
int transpose(const AdapterParams& P, const void* from, void* to, int a, int b,
              hipStream_t stream) {
  const int64_t tiles = (int64_t)((a + 31) / 32) * ((b + 31) / 32);
  return in_launches(P.K, kMostBlocks / tiles, [&](int64_t first, int64_t codes) {
    launch_traced("adapters_transpose_kernel", (adapters_transpose_kernel<T>),
                  dim3((unsigned)(tiles * codes)), dim3(kThreads), 0, stream, P,
                  static_cast<const T*>(from), static_cast<T*>(to), a, b, first);
    return check_launch("adapters_transpose_kernel");
  });
}

template <typename T>
int backward_of(const AdapterParams& P, const void* grad, const void* rows,
                const void* down, const void* up, const float* hidden,
                void* g_rows, void* g_down, void* g_up, void* workspace,
                hipStream_t stream) {
  char* ws = static_cast<char*>(workspace);
  const BackwardLayout L = backward_layout(P);
  auto* dh = reinterpret_cast<float*>(ws + L.dh);
  int rc = GSPLAT_OK;
  if ((g_rows || g_down) && P.rows > 0) {
    if ((rc = transpose<T>(P, up, ws + L.up_t, P.E, P.r, stream))) return rc;
    if (g_rows && (rc = transpose<T>(P, down, ws + L.down_t, P.r, P.D, stream))) return rc;
    rc = rows_of<T>(P, RowsArgs{grad, P.E, P.E, P.D, ws + L.up_t, ws + L.down_t, nullptr, P.scale,
                                1.0f, g_rows, dh, nullptr, 0},
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
  Slots S{L.chunk, false, 0};
  const int64_t slots = P.rows / L.chunk + P.K;
  const int per_slot = (A.blocks[0] + A.blocks[1]) * A.rank_blocks;
  rc = in_launches(slots, kMostBlocks / per_slot, [&](int64_t first, int64_t n) {
    S.begin = first;
    const dim3 grid((unsigned)(n * per_slot));
#define GS_MAPS(RT)                                                                     \
  if (rt == RT)                                                                         \
    launch_traced("adapters_maps_kernel", (adapters_maps_kernel<T, RT>), grid,          \
                  dim3(kThreads), 0, stream, P, A, S);
    GS_MAPS(1) GS_MAPS(2) GS_MAPS(4)
#undef GS_MAPS
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

}  // namespace

size_t adapters_forward_workspace_bytes(const AdapterParams& P) {
  const RowsPlan L = rows_plan(P, P.D, P.E);
  return is_split(L) ? (size_t)L.splits_down * P.rows * P.r * 4 : 0;
}
size_t adapters_backward_workspace_bytes(const AdapterParams& P) {
  return backward_layout(P).total;
}

#define GS_BY_TYPE(F)                                         \
  (P.dtype == GSPLAT_F32 ? F<float> : P.dtype == GSPLAT_BF16 ? F<__bf16> : F<_Float16>)

int launch_adapters_forward(const AdapterParams& P, const void* rows,
                            const void* down, const void* up, const void* base,
                            void* out, float* hidden, void* workspace,
                            hipStream_t stream) {
  return GS_BY_TYPE(forward_of)(P, rows, down, up, base, out, hidden, workspace, stream);
}

int launch_adapters_backward(const AdapterParams& P, const void* grad,
                             const void* rows, const void* down, const void* up,
                             const float* hidden, void* g_rows, void* g_down,
                             void* g_up, void* workspace, hipStream_t stream) {
  return GS_BY_TYPE(backward_of)(P, grad, rows, down, up, hidden, g_rows, g_down, g_up,
                                 workspace, stream);
}
#undef GS_BY_TYPE

}  // namespace gs
