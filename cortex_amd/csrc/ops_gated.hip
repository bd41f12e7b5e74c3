// ops_gated.hip -- the first products of a gated feed-forward block with what follows them (ct_gated_gemm), and the product that its
// backward pass begins with (ct_gated_gemm_gradient), dense or by group.
//
//   [gate up] = x [G; U]^T,   inner = f(gate) * up                                         (G above U in one matrix)
//   d = dy W,   d_gate = d * up * f'(gate),   d_up = d * f(gate)
//
// Forward, a tile takes as many rows of G as of U, the same ones, so that a block has the gate and the up of its results: neither is stored
// unless the backward pass wants them, and no launch reads them again.  Backward, the product's results are no tensor: each is
// taken with its gate and up as its sum is done.  What the gradients of x, G and U are formed of lies in one matrix, [d_gate d_up], so
// that they are plain products of it.
//
// The sums are those of ct_grouped_gemm's kernels (split_tile.h, grouped.h, double_tile.h), and so is what bounds them: the matrix
// cores at many rows, the reading of the weights at a few.
#include <cmath>

#include "common.h"
#include "double_tile.h"
#include "grouped.h"
#include "pair_tile.h"
#include "rows.h"
#include "split_tile.h"

using namespace cthip;

namespace {

struct GatedArgs {
  GroupedArgs g;         // its n: columns of the results; its c: of parts of k, or null
  void* inner;           // may be absent from a gradient
  void* pre;             // may be absent forward
  const void* pre_read;  // of a gradient
  int64_t ld_inner, ld_pre, ld_pre_read;
  int activation;
};

// f and its derivative.  Evaluated once to a result, in the tensor's type, whose functions are off by a few units in the last place.
template <class T>
__device__ __forceinline__ void activate(int kind, T x, T* value, T* slope) {
  constexpr T kRootHalf = (T)0.70710678118654752440, kDensity = (T)0.39894228040143267794;
  switch (kind) {
    case CT_GATE_LOGISTIC:
    case CT_GATE_SWISH: {
      const T p = T(1) / (T(1) + exp(-x)), rest = T(1) / (T(1) + exp(x));   // rest: 1 - p, to its last place
      *value = kind == CT_GATE_SWISH ? x * p : p;
      *slope = kind == CT_GATE_SWISH ? p + x * p * rest : p * rest;
      break;
    }
    case CT_GATE_TANH: {
      const T t = tanh(x);
      *value = t;
      *slope = (T(1) - t) * (T(1) + t);
      break;
    }
    case CT_GATE_GELU: {
      const T share = T(0.5) * erfc(-x * kRootHalf);
      *value = x * share;
      *slope = share + x * kDensity * exp(T(-0.5) * x * x);
      break;
    }
    default: {
      *value = x > T(0) ? x : (x != x ? x : T(0));
      *slope = x > T(0) ? T(1) : T(0);
    }
  }
}

template <class T>
__device__ __forceinline__ void finish(const GatedArgs& a, int64_t row, uint32_t column, T gate, T up) {
  T value, slope;
  activate(a.activation, gate, &value, &slope);
  static_cast<T*>(a.inner)[row * a.ld_inner + column] = value * up;
  if (!a.pre) return;
  T* pre = static_cast<T*>(a.pre) + row * a.ld_pre + column;
  pre[0] = gate;
  pre[a.g.n] = up;
}

template <class T>
__device__ __forceinline__ void finish_gradient(const GatedArgs& a, int64_t row, uint32_t column, T d) {
  const T* read = static_cast<const T*>(a.pre_read) + row * a.ld_pre_read + column;
  const T gate = read[0], up = read[a.g.n];
  T value, slope;
  activate(a.activation, gate, &value, &slope);
  T* pre = static_cast<T*>(a.pre) + row * a.ld_pre + column;
  pre[0] = d * up * slope;
  pre[a.g.n] = d * value;
  if (a.inner) static_cast<T*>(a.inner)[row * a.ld_inner + column] = value * up;
}

// The row of a lane's r-th cell in a tile of 32 x 32, behind its first one's.
__device__ __forceinline__ constexpr uint32_t row_at(int r) { return 8 * (r / 4) + r % 4; }

// A lane's cells of a column, `rows` rows of them there but for those of the bits of `skip`.  Addresses are the first cell's and uniform multiples of the stride; all that is
// read is on its way before the first result is stored, for that may be where it was read.
__device__ __forceinline__ void finish_column(const GatedArgs& a, int64_t row, uint32_t column, uint32_t rows, const float (&gate)[16], const float (&up)[16],
                                              uint32_t skip = 0) {
  float* const inner = static_cast<float*>(a.inner) + row * a.ld_inner + column;
  float* const pre = static_cast<float*>(a.pre) + row * a.ld_pre + column;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    if (row_at(r) >= rows || skip >> r & 1) continue;
    float value, slope;
    activate(a.activation, gate[r], &value, &slope);
    inner[row_at(r) * a.ld_inner] = value * up[r];
    if (a.pre) {
      pre[row_at(r) * a.ld_pre] = gate[r];
      pre[row_at(r) * a.ld_pre + a.g.n] = up[r];
    }
  }
}

__device__ __forceinline__ void finish_gradient_column(const GatedArgs& a, int64_t row, uint32_t column, uint32_t rows, const float (&d)[16],
                                                       uint32_t skip = 0) {
  const float* const read = static_cast<const float*>(a.pre_read) + row * a.ld_pre_read + column;
  float* const pre = static_cast<float*>(a.pre) + row * a.ld_pre + column;
  float* const inner = static_cast<float*>(a.inner) + row * a.ld_inner + column;
  float gate[16], up[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int64_t at = min(row_at(r), rows - 1) * a.ld_pre_read;
    gate[r] = read[at];
    up[r] = read[at + a.g.n];
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    if (row_at(r) >= rows || skip >> r & 1) continue;
    float value, slope;
    activate(a.activation, gate[r], &value, &slope);
    pre[row_at(r) * a.ld_pre] = d[r] * up[r] * slope;
    pre[row_at(r) * a.ld_pre + a.g.n] = d[r] * value;
    if (a.inner) inner[row_at(r) * a.ld_inner] = value * up[r];
  }
}

// Sums of a part of k, [part][row][gate up], or [part][row][column] of a gradient.
template <class T>
__device__ __forceinline__ void keep_pair(const GatedArgs& a, uint32_t part, int64_t row, uint32_t column, T gate, T up) {
  T* to = static_cast<T*>(a.g.c) + part * a.g.c_split + row * a.g.ldc + column;
  to[0] = gate;
  to[a.g.n] = up;
}

// ------------------------------------------------------------------ float: the matrix cores, three pieces to a float

// Of BN rows of the weights in a tile each 64 are 32 of G and the same 32 of U.
template <int BM, int BN, int T>
struct GatedSource : TileShare<BM, BN, T, true, true> {
  using Share = TileShare<BM, BN, T, true, true>;
  using Share::BK;
  using Share::U;
  using Share::UA;
  const float* row[U];
  bool absent[UA], any_absent;   // an index outside a: zeros in the place of its row
  uint32_t k, begin;
  __device__ __forceinline__ GatedSource(const GroupedArgs& a, const Group& g, uint32_t row0, uint32_t col0, uint32_t begin, uint32_t tid)
      : Share{tid}, any_absent(false), k(a.k), begin(begin) {
#pragma unroll
    for (int i = 0; i < UA; ++i) {
      const uint32_t at = g.first + min(row0 + this->row_of(i), g.rows - 1), from = a.index_a ? (uint32_t)a.index_a[at] : at;
      absent[i] = from >= a.a_rows;
      any_absent |= absent[i];
      row[i] = static_cast<const float*>(a.a) + (int64_t)(absent[i] ? 0 : from) * a.lda + this->chunk_of(i) * 8;
    }
    any_absent = __ballot(any_absent) != 0;
    const float* b = static_cast<const float*>(a.b) + (int64_t)g.index * a.b_stride;
#pragma unroll
    for (int i = UA; i < U; ++i) {
      const uint32_t r = this->row_of(i), column = min(col0 + r / 64 * 32 + r % 32, a.n - 1);
      row[i] = b + (int64_t)(r / 32 % 2 ? a.n + column : column) * a.ldb + this->chunk_of(i) * 8;
    }
  }
  __device__ __forceinline__ void rewind() {}
  __device__ __forceinline__ void load(int i, uint32_t tile, f32x4 (&to)[2]) const {
    const int64_t k0 = min(begin + tile * BK, k - BK);
    __builtin_memcpy(&to[0], row[i] + k0, 16);
    __builtin_memcpy(&to[1], row[i] + k0 + 4, 16);
  }
  __device__ __forceinline__ void drop(int i, uint32_t tile, f32x4 (&r)[2]) const {
    if (i < UA && any_absent) {
      asm volatile("");   // stays a branch
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e / 4][e % 4] = absent[i] ? 0.f : r[e / 4][e % 4];
    }
    const uint32_t k0 = begin + tile * BK;
    if (k0 + BK <= k) return;
    asm volatile("");
    const uint32_t repeated = k0 - (k - BK);
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e / 4][e % 4] = this->chunk_of(i) * 8 + e < repeated ? 0.f : r[e / 4][e % 4];
  }
};

// Waves of 64 columns have a gate and its up in one lane; of 32 a wave of gates and one of ups, which gives its sums to the other.
template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) gated_split_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr int T = 64 * WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
  static_assert(NT % 2 == 0 || (NT == 1 && WN == 2), "gates beside their ups");
  __shared__ __attribute__((aligned(16))) uint16_t lds[split_tile_lds(BM, BN)];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, BM, &g)) return;
  const uint32_t row0 = g.tile * BM, col0 = at.n_tile * (BN / 2), tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t begin = at.part * a.g.part, count = min(a.g.part, a.g.k - begin), lane = tid & 63, half = lane >> 5;
  GatedSource<BM, BN, T> source(a.g, g, row0, col0, begin, tid);
  float result[MT][NT][16];
  split_tile<BM, BN, WM, WN>(source, (count + 2 * kTileDepth - 1) / (2 * kTileDepth) * 2, lds, tid, result);
  if constexpr (NT == 1) {
    static_assert(WM * MT * 64 * 16 * 4 <= split_tile_lds(BM, BN) * 2, "the ups fit LDS");
    float* ups = reinterpret_cast<float*>(lds) + wave / WN * (MT * 64 * 16) + lane;
    __syncthreads();
    if (wave % WN == 1) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) ups[(t * 16 + r) * 64] = result[t][0][r];
    }
    __syncthreads();
    if (wave % WN == 1) return;
  }
  const float* ups = reinterpret_cast<const float*>(lds) + wave / WN * (MT * 64 * 16) + lane;
#pragma unroll
  for (int u = 0; u < NT; u += 2) {
    const uint32_t column = col0 + (wave % WN * (NT / 2) + u / 2) * 32 + (lane & 31);
    if (column >= a.g.n) continue;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint32_t m = row0 + (wave / WN * MT + t) * 32 + 4 * half;
      if (m >= g.rows) continue;
      float up[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) up[r] = NT == 1 ? ups[(t * 16 + r) * 64] : result[t][NT == 1 ? 0 : u + 1][r];
      if (!a.g.c) {
        finish_column(a, (int64_t)g.first + m, column, g.rows - m, result[t][u], up);
        continue;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (m + row_at(r) < g.rows) keep_pair(a, at.part, (int64_t)g.first + m + row_at(r), column, result[t][u][r], up[r]);
    }
  }
}

template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, 2) gated_gradient_split_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr int T = 64 * WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
  __shared__ __attribute__((aligned(16))) uint16_t lds[split_tile_lds(BM, BN)];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, BM, &g)) return;
  const uint32_t row0 = g.tile * BM, col0 = at.n_tile * BN, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t begin = at.part * a.g.part, count = min(a.g.part, a.g.k - begin), lane = tid & 63;
  GroupedSource<BM, BN, T, false> source(a.g, g, row0, col0, begin, tid);
  float result[MT][NT][16];
  split_tile<BM, BN, WM, WN>(source, (count + 2 * kTileDepth - 1) / (2 * kTileDepth) * 2, lds, tid, result);
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const uint32_t column = col0 + wave % WN * (NT * 32) + u * 32 + (lane & 31);
    if (column >= a.g.n) continue;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint32_t m = row0 + (wave / WN * MT + t) * 32 + 4 * (lane >> 5);
      if (m >= g.rows) continue;
      const int64_t row = (int64_t)g.first + m;
      if (!a.g.c) {
        finish_gradient_column(a, row, column, g.rows - m, result[t][u]);
        continue;
      }
      float* const to = static_cast<float*>(a.g.c) + at.part * a.g.c_split + row * a.g.ldc + column;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (m + row_at(r) < g.rows) to[row_at(r) * a.g.ldc] = result[t][u][r];
    }
  }
}

// ------------------------------------------------------------------ float, many rows: two halves to a float

// Three products of halves in place of six of bfloat16 pieces (pair_tile.h), of operands that are split once ahead of them: rows of
// the left one and columns of the right one have a power of two each, so that an element is held to 2^-23 of itself, or to 2^-51 of the
// largest of its row (or column) if that is more.  The chip's power bounds both kinds: 8192 rows, 1024 k, 5632 gates and ups 340 us
// with the splitting, with three pieces 600.  What is not finite has no power of two: rows of a NaN are NaN, and results of a row or column of infinities are
// formed once more from the floats.  So are sums that are small beside what a row or column with elements below 2^-28 of its largest may be off by
// (the large elements meet small ones, or none): no element of a float is held to less in them than in a product of floats.
//
// In the place of a row's exponent: twice the exponent, one more if it has such elements.
constexpr int kRowOfZeros = -2000, kAbsentRow = 2000, kRowOfNan = 2002, kRowOfInfinity = 2004;

// For a row whose largest magnitude has these bits, and the least one that is not 0.
__device__ __forceinline__ int exponent_for(uint32_t most, uint32_t least) {
  if (most > 0x7f800000u) return kRowOfNan;
  if (most == 0x7f800000u) return kRowOfInfinity;
  if (most == 0) return kRowOfZeros;
  const int log2 = most >> 23 ? (int)(most >> 23) - 127 : 31 - __clz(most) - 149, exponent = kPairTop - log2;
  return 2 * exponent + (ldexpf(__builtin_bit_cast(float, least), exponent) < 0x1p-13f);
}
__device__ __forceinline__ int power_of(int exponent) { return exponent >> 1; }
// In the scale of the pieces elements below 2^-13 are off by 2^-36 at most, and what they are multiplied by is below 2^15: a sum of k products is off by
// 2 k 2^-21 for both operands, 2^-24 of the sums from here on.
__device__ __forceinline__ float least_sum(uint32_t k) { return 16.f * (float)k; }

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

struct PiecesArgs {
  const float* x;      // matrices of `rows` rows (or, of a right operand by columns, k of them)
  char* pieces;
  int* exponents;
  uint32_t* partial;   // [matrix][part][largest least][row], by columns
  int64_t ld, stride;
  uint32_t rows, k, parts;
};

// Rows of k floats as pieces, a row to a wave: read once where 64 lanes hold it.
constexpr uint32_t kRowHeld = 8;   // times eight floats to a lane
__global__ void __launch_bounds__(256) pieces_of_rows_kernel(const PiecesArgs a) {
  const uint32_t row = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (row >= a.rows) return;
  const float* x = a.x + (int64_t)blockIdx.y * a.stride + (int64_t)row * a.ld;
  const uint32_t runs = (a.k + kPairRun - 1) / kPairRun;
  auto load = [&](uint32_t k, f32x4 (&v)[2]) {
    if (k + 8 <= a.k) {
      __builtin_memcpy(&v[0], x + k, 16);
      __builtin_memcpy(&v[1], x + k + 4, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e / 4][e % 4] = k + e < a.k ? x[k + e] : 0.f;
    }
  };
  f32x4 held[kRowHeld][2];
  uint32_t most = 0, least = ~0u;
  auto look_at = [&](const f32x4 (&v)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t x = magnitude(v[e / 4][e % 4]);
      most = max(most, x);
      least = min(least, x - 1);   // of 0 the largest word
    }
  };
#pragma unroll
  for (uint32_t i = 0; i < kRowHeld; ++i)
    if (i * 512 < a.k) {
      load(i * 512 + lane * 8, held[i]);
      look_at(held[i]);
    }
  for (uint32_t k = kRowHeld * 512; k < a.k; k += 512) {
    f32x4 v[2];
    load(k + lane * 8, v);
    look_at(v);
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    most = max(most, (uint32_t)__shfl_xor((int)most, d));
    least = min(least, (uint32_t)__shfl_xor((int)least, d));
  }
  const int exponent = exponent_for(most, least + 1), power = power_of(exponent);
  const int64_t at = (int64_t)blockIdx.y * a.rows + row;
  if (lane == 0) a.exponents[at] = exponent;
  char* to = a.pieces + at * runs * kPairRunBytes;
  auto store = [&](uint32_t k, const f32x4 (&v)[2]) {
    if (k >= runs * kPairRun) return;
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      _Float16 h, l;
      split_pair_apart(exponent < kAbsentRow ? ldexpf(v[e / 4][e % 4], power) : 0.f, &h, &l);
      hi[e] = h;
      lo[e] = l;
    }
    char* p = to + k / kPairRun * kPairRunBytes + k % kPairRun * 2;
    *reinterpret_cast<f16x8*>(p) = hi;
    *reinterpret_cast<f16x8*>(p + 64) = lo;
  };
#pragma unroll
  for (uint32_t i = 0; i < kRowHeld; ++i)
    if (i * 512 < a.k) store(i * 512 + lane * 8, held[i]);
  for (uint32_t k = kRowHeld * 512; k < a.k; k += 512) {
    f32x4 v[2];
    load(k + lane * 8, v);
    store(k + lane * 8, v);
  }
}

// The largest magnitudes of columns, and the least ones that are not 0, of a part of the k rows each.
__global__ void __launch_bounds__(256) most_of_columns_kernel(const PiecesArgs a) {
  __shared__ uint32_t found[4][2][64];
  const uint32_t c = threadIdx.x % 64, column = blockIdx.x * 64 + c, each = (a.k + a.parts - 1) / a.parts, first = blockIdx.y * each;
  const float* x = a.x + (int64_t)blockIdx.z * a.stride + min(column, a.rows - 1);
  uint32_t most = 0, least = ~0u;
  for (uint32_t k0 = first + threadIdx.x / 64; k0 < min(first + each, a.k); k0 += 16) {
    float v[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) v[e] = x[(int64_t)min(k0 + e * 4, a.k - 1) * a.ld];   // once more is no harm
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      most = max(most, magnitude(v[e]));
      least = min(least, magnitude(v[e]) - 1);   // of 0 the largest word
    }
  }
  found[threadIdx.x / 64][0][c] = most;
  found[threadIdx.x / 64][1][c] = least;
  __syncthreads();
  if (threadIdx.x < 64 && column < a.rows) {
    uint32_t* const to = a.partial + ((int64_t)blockIdx.z * a.parts + blockIdx.y) * 2 * a.rows + column;
    to[0] = max(max(found[0][0][c], found[1][0][c]), max(found[2][0][c], found[3][0][c]));
    to[a.rows] = min(min(found[0][1][c], found[1][1][c]), min(found[2][1][c], found[3][1][c]));
  }
}

// 64 columns of 64 rows as pieces, k down the columns.
__global__ void __launch_bounds__(256) pieces_of_columns_kernel(const PiecesArgs a) {
  __shared__ uint32_t cells[64][65];
  __shared__ int exponents[64];
  const uint32_t c = threadIdx.x % 64, column0 = blockIdx.x * 64, k0 = blockIdx.y * 64, column = min(column0 + c, a.rows - 1);
  const float* x = a.x + (int64_t)blockIdx.z * a.stride + column;
  float values[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) values[i] = x[(int64_t)min(k0 + i * 4 + threadIdx.x / 64, a.k - 1) * a.ld];
  if (threadIdx.x < 64) {
    uint32_t most = 0, least = ~0u;
    for (uint32_t part = 0; part < a.parts; ++part) {
      const uint32_t* const from = a.partial + ((int64_t)blockIdx.z * a.parts + part) * 2 * a.rows + column;
      most = max(most, from[0]);
      least = min(least, from[a.rows]);
    }
    exponents[c] = exponent_for(most, least + 1);
    if (blockIdx.y == 0 && column0 + c < a.rows) a.exponents[(int64_t)blockIdx.z * a.rows + column] = exponents[c];
  }
  __syncthreads();
  const int exponent = exponents[c];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t k = i * 4 + threadIdx.x / 64;
    _Float16 hi, lo;
    split_pair_apart(k0 + k < a.k && exponent < kAbsentRow ? ldexpf(values[i], power_of(exponent)) : 0.f, &hi, &lo);
    cells[c][k] = (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
  }
  __syncthreads();
  const uint32_t runs = (a.k + kPairRun - 1) / kPairRun;
#pragma unroll
  for (int i = 0; i < 2; ++i) {   // eight k of a column to a lane
    const uint32_t at = i * 256 + threadIdx.x, r = at / 8, k = at % 8 * 8, run = k0 / kPairRun + k / kPairRun;
    if (column0 + r >= a.rows || run >= runs) continue;
    pair_u32x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t v = cells[r][k + 2 * e], w = cells[r][k + 2 * e + 1];
      hi[e] = (v & 0xffff) | w << 16;
      lo[e] = v >> 16 | (w & 0xffff0000u);
    }
    char* p = a.pieces + (((int64_t)blockIdx.z * a.rows + column0 + r) * runs + run) * kPairRunBytes + k % kPairRun * 2;
    *reinterpret_cast<pair_u32x4*>(p) = hi;
    *reinterpret_cast<pair_u32x4*>(p + 64) = lo;
  }
}

struct GatedPieces {
  const char *left, *right;   // [row of a], [group][row of the weights, or column]
  const int *left_exponents, *right_exponents;
  uint32_t runs;
};

// A product in floats by a wave; stride: of the right operand's k.
__device__ __forceinline__ float plain_product(const float* left, const float* right, int64_t stride, uint32_t k) {
  float sum = 0.f;
#pragma unroll 4
  for (uint32_t i = threadIdx.x % 64; i < k; i += 64) sum += left[i] * right[i * stride];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
  return sum;
}

template <int BM, int BN, int WM, int WN, bool kGradient>
__global__ void __launch_bounds__(64 * WM * WN, 2) gated_pair_kernel(const GatedArgs a, const GatedPieces pieces, const GroupedPlan p) {
  constexpr int T = 64 * WM * WN, MT = BM / WM / 32, NT = BN / WN / 32, kColumns = kGradient ? BN : BN / 2;
  static_assert(kGradient || NT % 2 == 0, "gates beside their ups");
  __shared__ __attribute__((aligned(16))) char lds[pair_tile_lds(BM, BN)];
  __shared__ int exponents[BM + BN];
  __shared__ uint32_t again[BM][kColumns / 32];   // cells whose sums are formed from the floats
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, BM, &g)) return;
  const uint32_t row0 = g.tile * BM, col0 = at.n_tile * kColumns, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row_bytes = (int64_t)pieces.runs * kPairRunBytes, right0 = (int64_t)g.index * (kGradient ? a.g.n : 2 * (int64_t)a.g.n);
  auto left_row = [&](uint32_t r) {   // of a; one outside it is absent
    const uint32_t row = g.first + min(row0 + r, g.rows - 1);
    return a.g.index_a ? (uint32_t)a.g.index_a[row] : row;
  };
  auto right_row = [&](uint32_t r) {
    const uint32_t column = min(col0 + (kGradient ? r : r / 64 * 32 + r % 32), a.g.n - 1);
    return kGradient || r / 32 % 2 == 0 ? column : a.g.n + column;
  };
  bool found = false;
  for (uint32_t i = tid; i < BM + BN; i += T) {
    if (i < BM) {
      const uint32_t row = left_row(i);
      exponents[i] = row < a.g.a_rows ? pieces.left_exponents[row] : kAbsentRow;
    } else {
      exponents[i] = pieces.right_exponents[right0 + right_row(i - BM)];
    }
    found |= exponents[i] >= kAbsentRow || exponents[i] & 1;
  }
  for (uint32_t i = tid; i < BM * (kColumns / 32); i += T) (&again[0][0])[i] = 0;
  found = __syncthreads_or(found);
  const PairRows<BM, BN, T> source(
      [&](uint32_t r) {
        const uint32_t row = left_row(r);
        return pieces.left + (row < a.g.a_rows ? row : 0) * row_bytes;
      },
      [&](uint32_t r) { return pieces.right + (right0 + right_row(r)) * row_bytes; }, tid);
  pair_f32x16 sum[2][MT][NT];
  pair_tile<BM, BN, WM, WN, 1, true>(source, pieces.runs, lds, tid, sum);
  // what has exponents
  const float least = least_sum(a.g.k);
#pragma unroll
  for (int at_u = 0; at_u < (kGradient ? NT : NT / 2); ++at_u) {
    const int u = kGradient ? at_u : 2 * at_u;
    const uint32_t n = (wave % WN * NT + u) * 32 + (lane & 31), column = col0 + (wave % WN * (kGradient ? NT : NT / 2) + at_u) * 32 + (lane & 31);
    if (column >= a.g.n) continue;
    const int right = exponents[BM + n], right_up = kGradient ? 0 : exponents[BM + n + 32];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const uint32_t m = (wave / WN * MT + t) * 32 + 4 * (lane >> 5);
      if (row0 + m >= g.rows) continue;
      float first[16], second[16];
      uint32_t skip = 0;
      auto sum_of = [&](int of, int r) { return sum[0][t][of][r] + sum[1][t][of][r] * (1.f / (1 << kPairApart)); };
      if (!found) {   // as mostly: nothing to look for
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int left = power_of(exponents[m + row_at(r)]);
          first[r] = ldexpf(sum_of(u, r), -(left + power_of(right)));
          if constexpr (!kGradient) second[r] = ldexpf(sum_of(u + 1, r), -(left + power_of(right_up)));
        }
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int left = exponents[m + row_at(r)];
          bool skipped = false;
          auto cell = [&](int of, int right) {
            const float x = sum_of(of, r);
            if (left == kRowOfNan || right == kRowOfNan || (left == kAbsentRow && right >= kAbsentRow)) return __builtin_nanf("");   // zeros by infinities, too
            if (left == kAbsentRow) return 0.f;
            skipped |= max(left, right) >= kAbsentRow || (((left | right) & 1) && min(left, right) != kRowOfZeros && fabsf(x) < least);
            return ldexpf(x, -(power_of(left) + power_of(right)));
          };
          first[r] = cell(u, right);
          if constexpr (!kGradient) second[r] = cell(u + 1, right_up);
          if (!skipped) continue;
          skip |= 1u << r;
          atomicOr(&again[m + row_at(r)][(column - col0) / 32], 1u << (column - col0) % 32);
        }
      }
      if constexpr (kGradient) finish_gradient_column(a, (int64_t)g.first + row0 + m, column, g.rows - row0 - m, first, skip);
      else finish_column(a, (int64_t)g.first + row0 + m, column, g.rows - row0 - m, first, second, skip);
    }
  }
  if (!found) return;
  // rows and columns of infinities, and what is small beside what it may be off by: a cell to a wave
  __syncthreads();
  auto product = [&](uint32_t r, uint32_t n) -> float {
    if (exponents[r] == kRowOfNan || exponents[BM + n] == kRowOfNan) return __builtin_nanf("");
    const float* b = static_cast<const float*>(a.g.b) + (int64_t)g.index * a.g.b_stride + (int64_t)right_row(n) * (kGradient ? 1 : a.g.ldb);
    return plain_product(static_cast<const float*>(a.g.a) + (int64_t)left_row(r) * a.g.lda, b, kGradient ? a.g.ldb : 1, a.g.k);
  };
  for (uint32_t i = wave; i < BM * (kColumns / 32); i += WM * WN) {
    const uint32_t r = i / (kColumns / 32), c0 = i % (kColumns / 32) * 32;
    if (row0 + r >= g.rows) break;
    for (uint32_t cells = __builtin_amdgcn_readfirstlane(again[r][c0 / 32]); cells; cells &= cells - 1) {
      const uint32_t c = c0 + __builtin_ctz(cells), n = kGradient ? c : c / 32 * 64 + c % 32;
      const int64_t row = (int64_t)g.first + row0 + r;
      const float x = product(r, n), y = kGradient ? 0.f : product(r, n + (kGradient ? 0 : 32));
      if (lane != 0) continue;
      if constexpr (kGradient) finish_gradient(a, row, col0 + c, x);
      else finish(a, row, col0 + c, x, y);
    }
  }
}

// ------------------------------------------------------------------ float, a few rows to a group

// Of 16 NT rows of the weights half are of G and the other half the same ones of U.
template <int W, int NT>
__global__ void __launch_bounds__(64 * W, 4) gated_thin_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr uint32_t BM = 16, BN = 16 * NT, kColumns = BN / 2;
  __shared__ float partial[W][BM * BN];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, BM, &g)) return;
  const uint32_t row0 = g.tile * BM, col0 = at.n_tile * kColumns, at16 = threadIdx.x % 16;
  const uint32_t row = g.first + min(row0 + at16, g.rows - 1), from = a.g.index_a ? (uint32_t)a.g.index_a[row] : row;
  const bool absent = from >= a.g.a_rows;   // an index outside a: zeros in the place of its row
  const float* left = static_cast<const float*>(a.g.a) + (int64_t)(absent ? 0 : from) * a.g.lda;
  const float* b = static_cast<const float*>(a.g.b) + (int64_t)g.index * a.g.b_stride;
  const float* right[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const uint32_t r = u * 16 + at16, column = min(col0 + r % kColumns, a.g.n - 1);
    right[u] = b + (int64_t)(r / kColumns ? a.g.n + column : column) * a.g.ldb;
  }
  thin_sums<W, NT, true>(left, absent, right, a.g.ldb, BN, a.g.k, partial);
  for (uint32_t i = threadIdx.x; i < BM * kColumns; i += 64 * W) {
    const uint32_t m = row0 + i / kColumns, column = col0 + i % kColumns, cell = i / kColumns * BN + i % kColumns;
    float gate = partial[0][cell], up = partial[0][cell + kColumns];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      gate += partial[w][cell];
      up += partial[w][cell + kColumns];
    }
    if (m < g.rows && column < a.g.n) finish(a, (int64_t)g.first + m, column, gate, up);
  }
}

template <int W, int NT>
__global__ void __launch_bounds__(64 * W, 4) gated_gradient_thin_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr uint32_t BM = 16, BN = 16 * NT;
  __shared__ float partial[W][BM * BN];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, BM, &g)) return;
  const uint32_t row0 = g.tile * BM, col0 = at.n_tile * BN, row = g.first + min(row0 + threadIdx.x % 16, g.rows - 1);
  const float* right[1] = {static_cast<const float*>(a.g.b) + (int64_t)g.index * a.g.b_stride + col0};
  thin_sums<W, NT, false>(static_cast<const float*>(a.g.a) + (int64_t)row * a.g.lda, false, right, a.g.ldb, a.g.n - col0, a.g.k, partial);
  for (uint32_t i = threadIdx.x; i < BM * BN; i += 64 * W) {
    float sum = partial[0][i];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += partial[w][i];
    if (row0 + i / BN < g.rows && col0 + i % BN < a.g.n) finish_gradient(a, (int64_t)g.first + row0 + i / BN, col0 + i % BN, sum);
  }
}

// ------------------------------------------------------------------ double

// Half of a tile's S columns are gates, the other half their ups; they meet in LDS.
constexpr uint32_t kDoubleSide = 64;

__global__ void __launch_bounds__(256, 2) gated_double_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr uint32_t S = kDoubleSide;
  using Row = DoubleRow<S>;
  __shared__ double cells[S][S + 1];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, S, &g)) return;
  const uint32_t row0 = g.tile * S, col0 = at.n_tile * (S / 2), begin = at.part * a.g.part, count = min(a.g.part, a.g.k - begin);
  const uint32_t row = g.first + min(row0 + Row::row(), g.rows - 1), from = a.g.index_a ? (uint32_t)a.g.index_a[row] : row;
  const bool present = from < a.g.a_rows;
  const uint32_t column = min(col0 + Row::row() % (S / 2), a.g.n - 1);
  const double* b = static_cast<const double*>(a.g.b) + (int64_t)g.index * a.g.b_stride;
  double_tile<S>(count, Row{static_cast<const double*>(a.g.a) + (int64_t)(present ? from : 0) * a.g.lda + begin, count, present},
                 Row{b + (int64_t)(Row::row() / (S / 2) ? a.g.n + column : column) * a.g.ldb + begin, count, true},
                 [&](uint32_t r, uint32_t n, double sum) { cells[r][n] = sum; });
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < S * S / 2; i += 256) {
    const uint32_t m = i / (S / 2), n = i % (S / 2);
    if (row0 + m >= g.rows || col0 + n >= a.g.n) continue;
    const double gate = cells[m][n], up = cells[m][n + S / 2];
    if (a.g.c) keep_pair(a, at.part, (int64_t)g.first + row0 + m, col0 + n, gate, up);
    else finish(a, (int64_t)g.first + row0 + m, col0 + n, gate, up);
  }
}

__global__ void __launch_bounds__(256, 2) gated_gradient_double_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr uint32_t S = kDoubleSide;
  using Row = DoubleRow<S>;
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, S, &g)) return;
  const uint32_t row0 = g.tile * S, col0 = at.n_tile * S, begin = at.part * a.g.part, count = min(a.g.part, a.g.k - begin);
  const double* b = static_cast<const double*>(a.g.b) + (int64_t)g.index * a.g.b_stride;
  const uint32_t row = g.first + min(row0 + Row::row(), g.rows - 1);
  double_tile<S>(count, Row{static_cast<const double*>(a.g.a) + (int64_t)row * a.g.lda + begin, count, true},
                 DoubleColumns<S>(b + (int64_t)begin * a.g.ldb + col0, a.g.ldb, nullptr, 0, count, count, a.g.n - col0),
                 [&](uint32_t r, uint32_t n, double sum) {
                   if (row0 + r >= g.rows || col0 + n >= a.g.n) return;
                   const int64_t to = (int64_t)g.first + row0 + r;
                   if (a.g.c) static_cast<double*>(a.g.c)[at.part * a.g.c_split + to * a.g.ldc + col0 + n] = sum;
                   else finish_gradient(a, to, col0 + n, sum);
                 });
}

// Smaller products: 32 x 32 sums to a block, straight from memory (double_tile.h).
constexpr int kDirectWaves = 4;

__global__ void __launch_bounds__(64 * kDirectWaves, 2) gated_direct_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr uint32_t S = kDirectSide, kColumns = S / 2;
  using Rows = DoubleDirect<true>;
  __shared__ double partial[kDirectWaves][S * kDirectPitch];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, S, &g)) return;
  const uint32_t row0 = g.tile * S, col0 = at.n_tile * kColumns, begin = at.part * a.g.part, count = min(a.g.part, a.g.k - begin);
  const double* b = static_cast<const double*>(a.g.b) + (int64_t)g.index * a.g.b_stride;
  const Rows left = Rows::rows(static_cast<const double*>(a.g.a) + begin, a.g.lda, [&](uint32_t r) -> int64_t {
    const uint32_t row = g.first + min(row0 + r, g.rows - 1), from = a.g.index_a ? (uint32_t)a.g.index_a[row] : row;
    return from < a.g.a_rows ? (int64_t)from : -1;
  });
  const Rows right = Rows::rows(b + begin, a.g.ldb, [&](uint32_t r) -> int64_t {
    const uint32_t column = min(col0 + r % kColumns, a.g.n - 1);
    return r / kColumns ? (int64_t)a.g.n + column : column;
  });
  double_direct(count, left, right, partial);
#pragma unroll
  for (uint32_t i = threadIdx.x; i < S * kColumns; i += 64 * kDirectWaves) {
    const uint32_t m = i / kColumns, n = i % kColumns;
    if (row0 + m >= g.rows || col0 + n >= a.g.n) continue;
    const double gate = direct_sum(partial, m, n), up = direct_sum(partial, m, n + kColumns);
    if (a.g.c) keep_pair(a, at.part, (int64_t)g.first + row0 + m, col0 + n, gate, up);
    else finish(a, (int64_t)g.first + row0 + m, col0 + n, gate, up);
  }
}

__global__ void __launch_bounds__(64 * kDirectWaves, 2) gated_gradient_direct_kernel(const GatedArgs a, const GroupedPlan p) {
  constexpr uint32_t S = kDirectSide;
  using Rows = DoubleDirect<true>;
  __shared__ double partial[kDirectWaves][S * kDirectPitch];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a.g, at.m_tile, S, &g)) return;
  const uint32_t row0 = g.tile * S, col0 = at.n_tile * S, begin = at.part * a.g.part, count = min(a.g.part, a.g.k - begin);
  const double* b = static_cast<const double*>(a.g.b) + (int64_t)g.index * a.g.b_stride;
  const Rows left = Rows::rows(static_cast<const double*>(a.g.a) + begin, a.g.lda, [&](uint32_t r) { return (int64_t)g.first + min(row0 + r, g.rows - 1); });
  double_direct(count, left, DoubleDirect<false>::columns(b + (int64_t)begin * a.g.ldb + col0, a.g.ldb, a.g.n - col0), partial);
#pragma unroll
  for (uint32_t i = threadIdx.x; i < S * S; i += 64 * kDirectWaves) {
    const uint32_t r = i / S, n = i % S;
    if (row0 + r >= g.rows || col0 + n >= a.g.n) continue;
    const int64_t to = (int64_t)g.first + row0 + r;
    const double sum = direct_sum(partial, r, n);
    if (a.g.c) static_cast<double*>(a.g.c)[at.part * a.g.c_split + to * a.g.ldc + col0 + n] = sum;
    else finish_gradient(a, to, col0 + n, sum);
  }
}

// ------------------------------------------------------------------ the parts of k brought together

template <class T>
__device__ __forceinline__ T sum_of_parts(const T* partial, uint32_t parts, int64_t split) {
  double sum = 0.0;
  for (uint32_t s0 = 0; s0 < parts; s0 += 8) {   // loads of eight parts on their way
    T x[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = partial[min(s0 + s, parts - 1) * split];
#pragma unroll
    for (int s = 0; s < 8; ++s) sum += s0 + s < parts ? x[s] : T(0);
  }
  return (T)sum;
}

template <class T, bool kGradient>
__global__ void __launch_bounds__(256) gated_sum_kernel(const GatedArgs a, uint32_t parts, uint32_t cells, FastDiv n_fd) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= cells) return;
  uint32_t row, column;
  n_fd.divmod(i, row, column);
  const uint2 last = group_rows(a.g, a.g.groups - 1);
  if (row < group_rows(a.g, 0).x || row >= last.x + last.y) return;
  const T* partial = static_cast<const T*>(a.g.c) + (int64_t)row * a.g.ldc + column;
  const T sum = sum_of_parts(partial, parts, a.g.c_split);
  if constexpr (kGradient) finish_gradient(a, (int64_t)row, column, sum);
  else finish(a, (int64_t)row, column, sum, sum_of_parts(partial + a.g.n, parts, a.g.c_split));
}

// ------------------------------------------------------------------ the host's side

// The tiles that there are if the groups are even; `pairs`: a tile's columns are gates and ups.
struct Shape {
  int64_t rows, columns, groups, k, stored;   // stored: sums of a row
  int64_t row_tiles(int64_t height) const { return groups * ceil_div(rows / groups, height); }
  int64_t blocks(int64_t height, int64_t width) const { return row_tiles(height) * ceil_div(stored, width); }
};

// Microseconds of the kernels for a few rows, 64 or 16 sums of a row to a block: the weights at 5.6 TB/s if 200 units read them, half of
// that again for each further tile of rows; the float instructions at 110 TFLOP/s, mostly meanwhile; the rows, which each block reads,
// at 16 TB/s.  Us of 16 and of 64: one row, 4096 by 8192 gates and ups, 48 and 53; sixteen 68 and 54; 16 rows, 1024 by 4096, 10.5 and 12;
// 32, 2048 by 4096, 32 and 22; one, 1024 by 2816, 8 and 12.
double time_of_few(const Shape& s, int64_t width) {
  const double blocks = (double)s.blocks(16, width), tiles = (double)s.row_tiles(16) / (double)s.groups, units = std::min(1.0, blocks / (width == 64 ? 200 : 256));
  const double read = (double)(4 * s.groups * s.k * s.stored) * (0.5 + 0.5 * tiles) / (5.6e6 * (width == 64 ? units : 1.0));
  const double products = (double)(32 * s.row_tiles(16) * s.k * s.stored) / (110e6 * units);
  return (width == 64 ? 4.5 : 3.5) + std::max(read, products) + 0.3 * std::min(read, products) + blocks * (double)(64 * s.k) / 16e6 +
         1.5 * (double)((s.blocks(16, width) - 1) / (4 * kUnits));
}
// From these many k on a block has sixteen waves, of eight: 51 and 57 us at 4096 k; below 1024 the launch of sixteen takes longer.
constexpr uint32_t kFewK16 = 1024, kFewK64 = 2049;
constexpr bool few_waves(int64_t width, uint32_t k) { return k < (width == 64 ? kFewK64 : kFewK16); }

// Microseconds of tiles of doubles, of 32 a side straight from memory and of 64 by way of LDS, whose cells are finished four at a time and
// sixteen at a time.  Us of both, forward and gradient: 509 rows, 301 by 517, 16 and 15, 23 and 31; 1000 rows, 700 by 900, 80 and 43, 74 and 57;
// 4096, 512 by 512, 105 and 66, 95 and 63; 4096, 301 by 517, 81 and 50, 83 and 64; 200, 4096 by 64 in parts 18 and 11.  (Tiles of 32 by way of
// LDS: 509 rows 18 and 16; 512 rows, 512 by 512, 21 and 16, here 22 and 12.)
double time_of_direct(int64_t tiles, double k, bool gradient) { return 5.0 + (double)ceil_div(tiles, kUnits) * (0.0117 * k + (gradient ? 1.2 : 0.9)); }
double time_of_double(int64_t tiles, double k, bool gradient) {
  const double rounds = (double)ceil_div(tiles, kUnits);
  return 5.0 + k * (0.015 + 0.037 * rounds) + rounds * (gradient ? 8.0 : 3.5);
}

int64_t aligned(int64_t bytes) { return ceil_div(bytes, 256) * 256; }

// Two blocks of four waves to a unit: one's results go to memory beside the other's products (a gradient's product of 8192 rows, 2816 by
// 1024, 255 us, in tiles of 256 by 128 of eight waves 270).
constexpr int kPairM = 128, kPairN = 128, kPairWavesM = 2, kPairWavesN = 2;

// Microseconds beyond the products' for a round of blocks, whose results' bytes bound it: with three pieces, and with two halves.
constexpr double end_of_round(bool pairs, bool gradient) { return pairs ? (gradient ? 36.0 : 10.0) : (gradient ? 25.0 : 12.0); }

// Microseconds with two halves to a float: the splitting, of all groups' weights, at 3.5 TB/s; rounds of blocks, two to a unit or in the last one by themselves.
double time_of_pairs(const Shape& s, int64_t left_rows, int64_t all_groups, bool gradient) {
  const int64_t right = all_groups * s.stored, blocks = s.blocks(kPairM, kPairN), full = blocks / (2 * kUnits), rest = blocks % (2 * kUnits);
  const double split = (double)s.k * (8.0 * (double)left_rows + (gradient ? 12.0 : 8.0) * (double)right) / 3.5e6;
  const double end = end_of_round(true, gradient), runs = (double)ceil_div(s.k, kPairRun);
  return 10.0 + split + (double)full * (end + 1.38 * runs) + (rest == 0 ? 0.0 : rest <= kUnits ? 0.6 * end + 0.8 * runs : end + 1.38 * runs);
}

// Whether scratch was there, and the launches have been made.
template <bool kGradient>
bool run_pairs(hipStream_t s, const GatedArgs& a, const Shape& shape, int64_t left_rows, int64_t all_groups) {
  const int64_t runs = ceil_div(shape.k, kPairRun), right_rows = all_groups * shape.stored, parts = std::min<int64_t>(32, ceil_div(shape.k, 64));
  const int64_t left_bytes = aligned(left_rows * runs * kPairRunBytes), right_bytes = aligned(right_rows * runs * kPairRunBytes);
  const int64_t partial_bytes = kGradient ? aligned(right_rows * parts * 8) : 0;
  const ProductScratch scratch(s, (size_t)(left_bytes + right_bytes + aligned(left_rows * 4) + aligned(right_rows * 4) + partial_bytes));
  char* const base = static_cast<char*>(scratch.get());
  if (!base) return false;
  char* const right = base + left_bytes;
  int* const left_exponents = reinterpret_cast<int*>(right + right_bytes);
  int* const right_exponents = left_exponents + aligned(left_rows * 4) / 4;
  PiecesArgs of_left{static_cast<const float*>(a.g.a), base, left_exponents, nullptr, a.g.lda, 0, (uint32_t)left_rows, (uint32_t)shape.k, 0};
  hipLaunchKernelGGL(pieces_of_rows_kernel, dim3((uint32_t)ceil_div(left_rows, 4)), dim3(256), 0, s, of_left);
  PiecesArgs of_right{static_cast<const float*>(a.g.b), right, right_exponents, reinterpret_cast<uint32_t*>(right_exponents + aligned(right_rows * 4) / 4),
                      a.g.ldb, a.g.b_stride, (uint32_t)shape.stored, (uint32_t)shape.k, (uint32_t)parts};
  const uint32_t groups = (uint32_t)all_groups;
  if constexpr (kGradient) {
    const uint32_t columns = (uint32_t)ceil_div(shape.stored, 64);
    hipLaunchKernelGGL(most_of_columns_kernel, dim3(columns, (uint32_t)parts, groups), dim3(256), 0, s, of_right);
    hipLaunchKernelGGL(pieces_of_columns_kernel, dim3(columns, (uint32_t)ceil_div(shape.k, 64), groups), dim3(256), 0, s, of_right);
  } else {
    hipLaunchKernelGGL(pieces_of_rows_kernel, dim3((uint32_t)ceil_div(shape.stored, 4), groups), dim3(256), 0, s, of_right);
  }
  const GatedPieces pieces{base, right, left_exponents, right_exponents, (uint32_t)runs};
  const int64_t m_tiles = a.g.offsets ? shape.rows / kPairM + shape.groups : ceil_div(shape.rows, kPairM), n_tiles = ceil_div(shape.stored, kPairN);
  for_launches(m_tiles, n_tiles, 1, [&](dim3 grid, const GroupedPlan& plan) {
    hipLaunchKernelGGL((gated_pair_kernel<kPairM, kPairN, kPairWavesM, kPairWavesN, kGradient>), grid, dim3(64 * kPairWavesM * kPairWavesN), 0, s, a, pieces, plan);
  });
  return true;
}

template <class T, bool kGradient, class Launch>
int run(const char* name, hipStream_t s, GatedArgs a, const Shape& shape, bool split, Launch launch) {
  const int64_t cells = shape.rows * shape.stored, pair = kGradient ? 1 : 2;
  const int64_t k_tiles = ceil_div(shape.k, kTileDepth), results = shape.rows * shape.columns;
  auto add_up = [&](int64_t parts) {
    hipLaunchKernelGGL((gated_sum_kernel<T, kGradient>), dim3((uint32_t)ceil_div(results, 256)), dim3(256), 0, s, a, (uint32_t)parts, (uint32_t)results,
                       FastDiv((uint32_t)shape.columns));
  };
  if (shape.k == 0) {   // sums of no terms
    CT_REQUIRE(results <= kMostExtent, "%s: %lld rows of %lld columns", name, (long long)shape.rows, (long long)shape.columns);
    add_up(0);
    note_kernel(kGradient ? "gated_gradient_sum" : "gated_sum");
    return after_launch(s);
  }
  auto choose = [&](int64_t most_parts) {
    if constexpr (std::is_same<T, double>::value) {
      Choice best{32, 32, 1, 1e12};
      for (int64_t parts = 1; parts <= most_parts && (parts == 1 || shape.k >= parts * 64); parts *= 2) {
        const int64_t small = shape.blocks(kDirectSide, kDirectSide) * parts, large = shape.blocks(kDoubleSide, kDoubleSide) * parts;
        const double k = (double)shape.k / (double)parts, sum = time_of_sum(parts, cells, sizeof(double));
        if (time_of_direct(small, k, kGradient) + sum < best.us) best = {32, 32, parts, time_of_direct(small, k, kGradient) + sum};
        if (time_of_double(large, k, kGradient) + sum < best.us) best = {64, 64, parts, time_of_double(large, k, kGradient) + sum};
      }
      return best;
    } else {
      const double thin64 = time_of_few(shape, 64), thin16 = time_of_few(shape, 16);
      Choice best{16, thin16 < thin64 ? 16 : 64, 1, std::min(thin64, thin16)};
      if (split) consider_parts(&best, shape.blocks(64, 64), shape.blocks(128, 128), k_tiles, cells, most_parts);
      return best;
    }
  };
  Choice best = choose(kMostParts);
  if constexpr (std::is_same<T, float>::value) {
    const int64_t left_rows = a.g.a_rows;
    double us = best.us;
    if (best.height == 128) us += end_of_round(false, kGradient) * (double)ceil_div(shape.blocks(128, 128) * best.parts, kUnits);
    if (shape.k >= kPairRun && time_of_pairs(shape, left_rows, a.g.groups, kGradient) < us && run_pairs<kGradient>(s, a, shape, left_rows, a.g.groups)) {
      note_kernel(kGradient ? "gated_gradient_pairs" : "gated_pairs");
      return after_launch(s);
    }
  }
  const Parts<T> parts(s, best.parts, cells);
  if (parts.count() < best.parts) best = choose(1);
  const int64_t m_tiles = a.g.offsets ? shape.rows / best.height + shape.groups : ceil_div(shape.rows, best.height), n_tiles = ceil_div(shape.columns, best.width / pair);
  CT_REQUIRE(m_tiles <= kMostTiles / parts.count() / n_tiles, "%s: %lld rows of %lld columns", name, (long long)shape.rows, (long long)shape.columns);
  a.g.c = const_cast<T*>(parts.partial());
  a.g.ldc = shape.stored;
  a.g.c_split = cells;
  a.g.part = (uint32_t)(std::is_same<T, double>::value ? ceil_div(shape.k, parts.count()) : tiles_of_part(k_tiles, parts.count()) * kTileDepth);
  const uint32_t band = best.height == 16 && shape.rows <= 16 * shape.groups ? 1 : kBand;
  launch(a, best, m_tiles, n_tiles, parts.count(), band);
  if (parts.partial()) add_up(parts.count());
  static const char* const kNames[] = {"gated_thin", "gated_thin_long", "gated_thin_wide", "gated_thin_wide_long", "gated_medium", "gated_medium+gated_sum",
                                       "gated_large", "gated_large+gated_sum", "gated_double", "gated_double+gated_sum", "gated_double_tiles",
                                       "gated_double_tiles+gated_sum"};
  static const char* const kGradientNames[] = {"gated_gradient_thin", "gated_gradient_thin_long", "gated_gradient_thin_wide", "gated_gradient_thin_wide_long",
                                               "gated_gradient_medium", "gated_gradient_medium+gated_sum", "gated_gradient_large",
                                               "gated_gradient_large+gated_sum", "gated_gradient_double", "gated_gradient_double+gated_sum",
                                               "gated_gradient_double_tiles", "gated_gradient_double_tiles+gated_sum"};
  const int several = parts.count() > 1;
  const int kernel = std::is_same<T, double>::value ? (best.height == 64 ? 10 : 8) + several
                     : best.height == 16            ? (best.width == 64 ? 2 : 0) + !few_waves(best.width, a.g.k)
                                                    : (best.height == 128 ? 6 : 4) + several;
  note_kernel(kGradient ? kGradientNames[kernel] : kNames[kernel]);
  return after_launch(s);
}

constexpr int64_t kMostStride = int64_t(1) << 40;
bool known(int activation) { return activation >= CT_GATE_LOGISTIC && activation <= CT_GATE_GELU; }

}  // namespace

#define CT_GATED_FLOATING(name) CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, name ": datatype must be float or double")

extern "C" {

int ct_gated_gemm(void* stream, void* inner, int64_t inner_colstride, void* pre, int64_t pre_colstride, int activation, const void* a,
                  int64_t a_row_count, int64_t a_col_count, int64_t a_colstride, const int32_t* index, const void* b, int64_t hidden,
                  int64_t b_colstride, int64_t b_stride, const int32_t* offsets, int64_t n_groups, int64_t row_count, int dtype) {
  CT_GATED_FLOATING("ct_gated_gemm");
  CT_REQUIRE(known(activation), "ct_gated_gemm: unknown activation %d", activation);
  CT_REQUIRE(extent(a_row_count) && extent(a_col_count) && extent(hidden) && extent(2 * hidden) && extent(row_count), "ct_gated_gemm: bad extent");
  CT_REQUIRE(n_groups >= 0 && n_groups <= kMostGroups, "ct_gated_gemm: %lld groups, at most %lld are taken", (long long)n_groups, (long long)kMostGroups);
  CT_REQUIRE(offsets || n_groups <= 1, "ct_gated_gemm: %lld groups without offsets", (long long)n_groups);
  if (n_groups == 0 || row_count == 0 || hidden == 0) return CT_OK;
  CT_REQUIRE(inner && (a_col_count == 0 || (b && (a || a_row_count == 0))), "ct_gated_gemm: null buffer");
  CT_REQUIRE(index || a_row_count >= row_count, "ct_gated_gemm: a has %lld rows of %lld", (long long)a_row_count, (long long)row_count);
  CT_REQUIRE(inner_colstride >= hidden && (!pre || pre_colstride >= 2 * hidden) && a_colstride >= a_col_count && b_colstride >= a_col_count,
             "ct_gated_gemm: a column stride below the row's length");
  CT_REQUIRE(b_stride >= 0, "ct_gated_gemm: negative stride of matrices");
  CT_REQUIRE(std::max({inner_colstride, pre_colstride, a_colstride, b_colstride, b_stride}) <= kMostStride, "ct_gated_gemm: a stride beyond 2^40");
  if (!index) a_row_count = row_count;   // rows beyond these are not looked at
  const int64_t size = dtype_size(dtype);
  const RowRange results[] = {{inner, row_count, hidden, inner_colstride}, {pre, row_count, 2 * hidden, pre_colstride}};
  CT_REQUIRE(!rows_meet(results[0], results[1], size), "ct_gated_gemm: the results overlap");
  for (const RowRange& result : results) {
    CT_REQUIRE(!rows_meet(result, {a_col_count ? a : nullptr, a_row_count, a_col_count, a_colstride}, size) &&
                   !run_meets({a_col_count ? b : nullptr, ((n_groups - 1) * b_stride + (2 * hidden - 1) * b_colstride + a_col_count) * size}, result, size),
               "ct_gated_gemm: a result overlaps an operand");
    CT_REQUIRE(!run_meets({offsets, (n_groups + 1) * 4}, result, size) && !run_meets({index, row_count * 4}, result, size),
               "ct_gated_gemm: a result overlaps the offsets or the index");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  GatedArgs args{};
  args.g.a = a; args.g.b = b; args.g.index_a = index; args.g.offsets = offsets;
  args.g.lda = a_colstride; args.g.ldb = b_colstride; args.g.b_stride = b_stride;
  args.g.groups = (uint32_t)n_groups; args.g.rows = (uint32_t)row_count; args.g.a_rows = (uint32_t)a_row_count;
  args.g.n = (uint32_t)hidden; args.g.k = a_row_count > 0 ? (uint32_t)a_col_count : 0;   // no row of a is there: sums of no terms
  args.inner = inner; args.pre = pre;
  args.ld_inner = inner_colstride; args.ld_pre = pre_colstride;
  args.activation = activation;
  const Shape shape{row_count, hidden, std::min(n_groups, row_count), (int64_t)args.g.k, 2 * hidden};
  if (dtype == CT_F64) {
    return run<double, false>("ct_gated_gemm", s, args, shape, true, [&](const GatedArgs& a, const Choice& best, int64_t m_tiles, int64_t n_tiles, int64_t parts, uint32_t band) {
      for_launches(m_tiles, n_tiles, parts, [&](dim3 grid, const GroupedPlan& plan) {
        if (best.height == 64) hipLaunchKernelGGL(gated_double_kernel, grid, dim3(256), 0, s, a, plan);
        else hipLaunchKernelGGL(gated_direct_kernel, grid, dim3(64 * kDirectWaves), 0, s, a, plan);
      }, band);
    });
  }
  return run<float, false>("ct_gated_gemm", s, args, shape, shape.k >= kTileDepth, [&](const GatedArgs& a, const Choice& best, int64_t m_tiles, int64_t n_tiles, int64_t parts, uint32_t band) {
    for_launches(m_tiles, n_tiles, parts, [&](dim3 grid, const GroupedPlan& plan) {
      const bool few = few_waves(best.width, a.g.k);
      if (best.height == 128) hipLaunchKernelGGL((gated_split_kernel<128, 128, 4, 2>), grid, dim3(512), 0, s, a, plan);
      else if (best.height == 64) hipLaunchKernelGGL((gated_split_kernel<64, 64, 2, 2>), grid, dim3(256), 0, s, a, plan);
      else if (best.width == 64 && few) hipLaunchKernelGGL((gated_thin_kernel<8, 4>), grid, dim3(512), 0, s, a, plan);
      else if (best.width == 64) hipLaunchKernelGGL((gated_thin_kernel<16, 4>), grid, dim3(1024), 0, s, a, plan);
      else if (few) hipLaunchKernelGGL((gated_thin_kernel<8, 1>), grid, dim3(512), 0, s, a, plan);
      else hipLaunchKernelGGL((gated_thin_kernel<16, 1>), grid, dim3(1024), 0, s, a, plan);
    }, band);
  });
}

int ct_gated_gemm_gradient(void* stream, void* pre_gradient, int64_t pre_gradient_colstride, void* inner, int64_t inner_colstride, int activation,
                           const void* a, int64_t a_col_count, int64_t a_colstride, const void* b, int64_t hidden, int64_t b_colstride,
                           int64_t b_stride, const void* pre, int64_t pre_colstride, const int32_t* offsets, int64_t n_groups, int64_t row_count,
                           int dtype) {
  CT_GATED_FLOATING("ct_gated_gemm_gradient");
  CT_REQUIRE(known(activation), "ct_gated_gemm_gradient: unknown activation %d", activation);
  CT_REQUIRE(extent(a_col_count) && extent(hidden) && extent(2 * hidden) && extent(row_count), "ct_gated_gemm_gradient: bad extent");
  CT_REQUIRE(n_groups >= 0 && n_groups <= kMostGroups, "ct_gated_gemm_gradient: %lld groups, at most %lld are taken", (long long)n_groups, (long long)kMostGroups);
  CT_REQUIRE(offsets || n_groups <= 1, "ct_gated_gemm_gradient: %lld groups without offsets", (long long)n_groups);
  if (n_groups == 0 || row_count == 0 || hidden == 0) return CT_OK;
  CT_REQUIRE(pre_gradient && pre && (a_col_count == 0 || (a && b)), "ct_gated_gemm_gradient: null buffer");
  CT_REQUIRE(pre_gradient_colstride >= 2 * hidden && pre_colstride >= 2 * hidden && (!inner || inner_colstride >= hidden) && a_colstride >= a_col_count &&
                 b_colstride >= hidden,
             "ct_gated_gemm_gradient: a column stride below the row's length");
  CT_REQUIRE(b_stride >= 0, "ct_gated_gemm_gradient: negative stride of matrices");
  CT_REQUIRE(std::max({pre_gradient_colstride, inner_colstride, pre_colstride, a_colstride, b_colstride, b_stride}) <= kMostStride,
             "ct_gated_gemm_gradient: a stride beyond 2^40");
  const int64_t size = dtype_size(dtype);
  const RowRange results[] = {{pre_gradient, row_count, 2 * hidden, pre_gradient_colstride}, {inner, row_count, hidden, inner_colstride}};
  const RowRange read{pre, row_count, 2 * hidden, pre_colstride};
  CT_REQUIRE(!rows_meet(results[0], results[1], size), "ct_gated_gemm_gradient: the results overlap");
  const bool in_place = pre_gradient == pre && pre_gradient_colstride == pre_colstride;
  CT_REQUIRE((in_place || !rows_meet(results[0], read, size)) && !rows_meet(results[1], read, size), "ct_gated_gemm_gradient: a result overlaps pre");
  for (const RowRange& result : results) {
    CT_REQUIRE(!rows_meet(result, {a_col_count ? a : nullptr, row_count, a_col_count, a_colstride}, size) &&
                   !run_meets({a_col_count ? b : nullptr, ((n_groups - 1) * b_stride + (a_col_count - 1) * b_colstride + hidden) * size}, result, size),
               "ct_gated_gemm_gradient: a result overlaps an operand");
    CT_REQUIRE(!run_meets({offsets, (n_groups + 1) * 4}, result, size), "ct_gated_gemm_gradient: a result overlaps the offsets");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  GatedArgs args{};
  args.g.a = a; args.g.b = b; args.g.offsets = offsets;
  args.g.lda = a_colstride; args.g.ldb = b_colstride; args.g.b_stride = b_stride;
  args.g.groups = (uint32_t)n_groups; args.g.rows = args.g.a_rows = (uint32_t)row_count;
  args.g.n = (uint32_t)hidden; args.g.k = (uint32_t)a_col_count;
  args.inner = inner; args.pre = pre_gradient; args.pre_read = pre;
  args.ld_inner = inner_colstride; args.ld_pre = pre_gradient_colstride; args.ld_pre_read = pre_colstride;
  args.activation = activation;
  const Shape shape{row_count, hidden, std::min(n_groups, row_count), a_col_count, hidden};
  if (dtype == CT_F64) {
    return run<double, true>("ct_gated_gemm_gradient", s, args, shape, true, [&](const GatedArgs& a, const Choice& best, int64_t m_tiles, int64_t n_tiles, int64_t parts, uint32_t band) {
      for_launches(m_tiles, n_tiles, parts, [&](dim3 grid, const GroupedPlan& plan) {
        if (best.height == 64) hipLaunchKernelGGL(gated_gradient_double_kernel, grid, dim3(256), 0, s, a, plan);
        else hipLaunchKernelGGL(gated_gradient_direct_kernel, grid, dim3(64 * kDirectWaves), 0, s, a, plan);
      }, band);
    });
  }
  const bool split = a_col_count >= kTileDepth && b_colstride <= kMostSplitLd;
  return run<float, true>("ct_gated_gemm_gradient", s, args, shape, split, [&](const GatedArgs& a, const Choice& best, int64_t m_tiles, int64_t n_tiles, int64_t parts, uint32_t band) {
    for_launches(m_tiles, n_tiles, parts, [&](dim3 grid, const GroupedPlan& plan) {
      const bool few = few_waves(best.width, a.g.k);
      if (best.height == 128) hipLaunchKernelGGL((gated_gradient_split_kernel<128, 128, 2, 4>), grid, dim3(512), 0, s, a, plan);
      else if (best.height == 64) hipLaunchKernelGGL((gated_gradient_split_kernel<64, 64, 2, 2>), grid, dim3(256), 0, s, a, plan);
      else if (best.width == 64 && few) hipLaunchKernelGGL((gated_gradient_thin_kernel<8, 4>), grid, dim3(512), 0, s, a, plan);
      else if (best.width == 64) hipLaunchKernelGGL((gated_gradient_thin_kernel<16, 4>), grid, dim3(1024), 0, s, a, plan);
      else if (few) hipLaunchKernelGGL((gated_gradient_thin_kernel<8, 1>), grid, dim3(512), 0, s, a, plan);
      else hipLaunchKernelGGL((gated_gradient_thin_kernel<16, 1>), grid, dim3(1024), 0, s, a, plan);
    }, band);
  });
}

}  // extern "C"
