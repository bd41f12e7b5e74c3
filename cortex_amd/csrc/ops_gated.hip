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

// A lane's cells of a column, `rows` rows of them there.  Addresses are the first cell's and uniform multiples of the stride; all that is
// read is on its way before the first result is stored, for that may be where it was read.
__device__ __forceinline__ void finish_column(const GatedArgs& a, int64_t row, uint32_t column, uint32_t rows, const float (&gate)[16], const float (&up)[16]) {
  float* const inner = static_cast<float*>(a.inner) + row * a.ld_inner + column;
  float* const pre = static_cast<float*>(a.pre) + row * a.ld_pre + column;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    if (row_at(r) >= rows) continue;
    float value, slope;
    activate(a.activation, gate[r], &value, &slope);
    inner[row_at(r) * a.ld_inner] = value * up[r];
    if (a.pre) {
      pre[row_at(r) * a.ld_pre] = gate[r];
      pre[row_at(r) * a.ld_pre + a.g.n] = up[r];
    }
  }
}

__device__ __forceinline__ void finish_gradient_column(const GatedArgs& a, int64_t row, uint32_t column, uint32_t rows, const float (&d)[16]) {
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
    if (row_at(r) >= rows) continue;
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
template <int S>
__global__ void __launch_bounds__(256, 2) gated_double_kernel(const GatedArgs a, const GroupedPlan p) {
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

template <int S>
__global__ void __launch_bounds__(256, 2) gated_gradient_double_kernel(const GatedArgs a, const GroupedPlan p) {
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
      consider_double_parts(&best, shape.blocks(32, 32), shape.blocks(64, 64), shape.k, shape.k, cells, most_parts);
      return best;
    } else {
      const double thin64 = time_of_few(shape, 64), thin16 = time_of_few(shape, 16);
      Choice best{16, thin16 < thin64 ? 16 : 64, 1, std::min(thin64, thin16)};
      if (split) consider_parts(&best, shape.blocks(64, 64), shape.blocks(128, 128), k_tiles, cells, most_parts);
      return best;
    }
  };
  Choice best = choose(kMostParts);
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
  static const char* const kNames[] = {"gated_thin", "gated_medium", "gated_large", "gated_medium+gated_sum", "gated_large+gated_sum", "gated_double",
                                       "gated_double+gated_sum"};
  static const char* const kGradientNames[] = {"gated_gradient_thin", "gated_gradient_medium", "gated_gradient_large", "gated_gradient_medium+gated_sum",
                                               "gated_gradient_large+gated_sum", "gated_gradient_double", "gated_gradient_double+gated_sum"};
  const int kernel = std::is_same<T, double>::value ? 5 + (parts.count() > 1) : best.height == 16 ? 0 : 1 + (best.height == 128) + 2 * (parts.count() > 1);
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
        if (best.height == 64) hipLaunchKernelGGL((gated_double_kernel<64>), grid, dim3(256), 0, s, a, plan);
        else hipLaunchKernelGGL((gated_double_kernel<32>), grid, dim3(256), 0, s, a, plan);
      }, band);
    });
  }
  return run<float, false>("ct_gated_gemm", s, args, shape, shape.k >= kTileDepth, [&](const GatedArgs& a, const Choice& best, int64_t m_tiles, int64_t n_tiles, int64_t parts, uint32_t band) {
    for_launches(m_tiles, n_tiles, parts, [&](dim3 grid, const GroupedPlan& plan) {
      const bool few = a.g.k < (best.width == 64 ? kFewK64 : kFewK16);   // k
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
        if (best.height == 64) hipLaunchKernelGGL((gated_gradient_double_kernel<64>), grid, dim3(256), 0, s, a, plan);
        else hipLaunchKernelGGL((gated_gradient_double_kernel<32>), grid, dim3(256), 0, s, a, plan);
      }, band);
    });
  }
  const bool split = a_col_count >= kTileDepth && b_colstride <= kMostSplitLd;
  return run<float, true>("ct_gated_gemm_gradient", s, args, shape, split, [&](const GatedArgs& a, const Choice& best, int64_t m_tiles, int64_t n_tiles, int64_t parts, uint32_t band) {
    for_launches(m_tiles, n_tiles, parts, [&](dim3 grid, const GroupedPlan& plan) {
      const bool few = a.g.k < (best.width == 64 ? kFewK64 : kFewK16);   // k
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
