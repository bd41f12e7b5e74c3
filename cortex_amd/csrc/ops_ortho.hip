// ops_ortho.hip -- matrices made orthogonal by Newton-Schulz products (ct_orthogonalize) and the optimizer step that is made of
// it (ct_muon_step).
//
// With X = G / (|G| + epsilon), |G| the root of the sum of all squares, each step takes
//   A = X X^T,   B = a I + b A + c A A,   X = B X
// on the side of the matrix that is shorter (X^T X, and X B, of a tall one).  A step maps every singular value s of X to
// s (a + b s^2 + c s^4) and leaves the singular vectors, so after a few of them all that are not tiny are near one.
//
// What bounds it: the products.  A and A A are symmetric: tiles below the diagonal are computed and stored twice.  Nothing is
// done between the products: a I + b A + c A A is formed from the sums as they are stored, and a product stores its results as
// the next one reads them.
//
// Float.  The products are those of pair_tile.h, two halves to a float, which hold an element to 2^-39 of a bound.  So that rows, or columns, far
// below the others keep a float's bits all the same, what is multiplied has powers of two taken out.  With X = D Y, D the
// diagonal of a power of two to each row that its norm does not exceed, and so no element of Y one,
//   G = Y Y^T,   M = a I + (b G + c (G D) (G D)^T) D^2,   X after the step = D M Y
// and M is what a I + b A + c A A is between rows of D Y: of an element of it what matters to its row of Y is held.  For the product
// with M, whose sums run down the columns of Y, each column of Y has a power of two of its own too.
//   Where these come from: a row's norm after a step is at most its norm before, which G has on its diagonal, times the largest
// |a + b s^2 + c s^4|, and the coefficients bound the singular values, 1 at first and the largest s (a + b s^2 + c s^4) below the last bound then.
// A column's largest element is recorded as it is stored and has a bound after the next step (StepBounds).  All of them are powers of two, so
// they round nothing.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "common.h"
#include "double_tile.h"
#include "ortho.h"
#include "pair_tile.h"
#include "rows.h"

using namespace cthip;

namespace {

// Consecutive units of work on one die: neighbouring tiles share operands in its L2.
__device__ __forceinline__ uint32_t unit_of_block(uint32_t b, uint32_t units) {
  const uint32_t per_die = (units + kXcds - 1) / kXcds;
  return (b % kXcds) * per_die + b / kXcds;
}

// Tiles of one product in bands of some rows, column after column, so that those that run at once on a die need few rows and columns; of a
// symmetric one those at and below the diagonal.
constexpr uint32_t kBand = 8;

struct TileOrder {
  uint32_t units, tiles, m_tiles, n_tiles;   // tiles of a matrix; units: of all of them
  uint32_t band;                             // rows of a band, of a symmetric product of square tiles
  FastDiv tiles_fd, band_fd;
};

struct TilePlace {
  uint32_t matrix, m_tile, n_tile;
};

// kTall: tiles of a symmetric product are 4 high by 3 wide, not square.
template <bool kSymmetric, bool kTall = false>
__device__ __forceinline__ bool place_of_unit(const TileOrder& o, uint32_t unit, TilePlace* p) {
  if (unit >= o.units) return false;
  uint32_t tile, band, rest;
  o.tiles_fd.divmod(unit, p->matrix, tile);
  if constexpr (kSymmetric) {
    // band b has `rows` rows of `whole` columns and what is below the diagonal beyond them; the bands before it
    const uint32_t rows = kTall ? 3 : o.band;
    auto before = [&](uint32_t b) { return kTall ? 6 * b * b + 3 * b : rows * b * (rows * b + 1) / 2; };
    band = (uint32_t)(kTall ? (sqrtf(24.f * (float)tile + 9.f) - 3.f) * (1.f / 12.f) : (sqrtf(8.f * (float)tile + 1.f) - 1.f) * 0.5f / (float)rows);   // may be one off
    if (before(band) > tile) --band;
    if (before(band + 1) <= tile) ++band;
    rest = tile - before(band);
    const uint32_t there = min(rows, o.m_tiles - band * rows), whole = kTall ? 4 * band + 2 : band * rows + 1;
    uint32_t row = 0, column = 0;
    if (rest < there * whole) {
      column = rest / there;
      row = rest - column * there;
    } else {   // a column has a row less than the one before it
      rest -= there * whole;
      column = whole;
      for (uint32_t left = there - 1; rest >= left; --left, ++column) rest -= left;
      row = rest + column - whole + 1;
    }
    p->m_tile = band * rows + row;
    p->n_tile = column;
  } else {
    o.band_fd.divmod(tile, band, rest);
    const uint32_t rows = min(kBand, o.m_tiles - band * kBand);
    p->n_tile = rest / rows;
    p->m_tile = band * kBand + rest - p->n_tile * rows;
  }
  return true;
}

template <bool kSymmetric, bool kTall = false>
__device__ __forceinline__ bool place_of(const TileOrder& o, TilePlace* p) {
  return place_of_unit<kSymmetric, kTall>(o, unit_of_block(blockIdx.x, o.units), p);
}

enum Product { kGram, kSquare, kUpdate, kLast };
constexpr bool is_symmetric(Product p) { return p == kGram || p == kSquare; }

// ------------------------------------------------------------------ the norm, and the matrix divided by it

constexpr uint32_t kParts = 1024;

__device__ __forceinline__ double sum_of_block(double x, double* lds) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) x += __shfl_down(x, d);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = x;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// The sums of squares of parts of a matrix of doubles; of a step, the momentum before them.  One read of what there is, a write of the
// momentum: bound by memory.  Squares of doubles may be no doubles: those of what is beyond 2^480, and below 2^-480, are summed apart, of
// 2^-600 and of 2^600 as much, [matrix][these three][part].
constexpr double kLargeDouble = 0x1p480, kSmallDouble = 0x1p-480;
constexpr int kDoubleShift = 600;

__global__ void __launch_bounds__(256) start_norm_kernel(const StartArgs a, uint32_t parts, uint64_t each, bool dense) {
  using T = double;
  __shared__ double lds[4];
  const int64_t base = (int64_t)blockIdx.y * a.stride;
  const uint64_t cells = (uint64_t)a.rows * a.columns, first = blockIdx.x * each, end = min(first + each, cells);
  double sum = 0.0, large = 0.0, small = 0.0;
  for (uint64_t i0 = first + threadIdx.x; i0 < end; i0 += 4 * 256) {
    T x[4], g[4];
    int64_t at[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t i = min(i0 + e * 256, end - 1);
      at[e] = base + (dense ? (int64_t)i : (int64_t)(i / a.columns) * a.ld + (int64_t)(i % a.columns));
      x[e] = static_cast<const T*>(a.x)[at[e]];
      if (a.gradient) g[e] = static_cast<const T*>(a.gradient)[at[e]];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (i0 + e * 256 >= end) continue;
      if (a.gradient) {
        const T step = (T)a.gradient_alpha * g[e];
        x[e] = (T)a.decay * x[e] + step;
        static_cast<T*>(a.momentum)[at[e]] = x[e];
        if (a.nesterov) x[e] = step + (T)a.decay * x[e];
      }
      const double size = fabs(x[e]);
      if (size >= kLargeDouble) {
        const double y = ldexp(x[e], -kDoubleShift);
        large += y * y;
      } else if (size < kSmallDouble) {
        const double y = ldexp(x[e], kDoubleShift);
        small += y * y;
      } else {
        sum += x[e] * x[e];
      }
    }
  }
  double* const to = a.partial + (int64_t)blockIdx.y * 3 * kParts + blockIdx.x;
  const double total = sum_of_block(sum, lds);
  if (threadIdx.x == 0) to[0] = total;
  __syncthreads();
  const double total_large = sum_of_block(large, lds);
  if (threadIdx.x == 0) to[kParts] = total_large;
  __syncthreads();
  const double total_small = sum_of_block(small, lds);
  if (threadIdx.x == 0) to[2 * kParts] = total_small;
}

// 1 / (|X| + epsilon) is factor * 2^power.
struct InverseNorm {
  double factor;
  int power;
};
__device__ __forceinline__ InverseNorm inverse_norm_of_doubles(const StartArgs& a, uint32_t matrix, uint32_t parts, double* lds) {
  double x[3] = {};
#pragma unroll
  for (uint32_t b = 0; b < 3; ++b)
#pragma unroll
    for (uint32_t i = 0; i < kParts / 256; ++i) {
      const uint32_t at = i * 256 + threadIdx.x;
      const double y = a.partial[((int64_t)matrix * 3 + b) * kParts + min(at, parts - 1)];
      x[b] += at < parts ? y : 0.0;
    }
  const bool any_large = __syncthreads_or(x[1] != 0.0), any_small = __syncthreads_or(x[2] != 0.0);
  double sum = sum_of_block(x[0], lds);
  if (any_large) {
    __syncthreads();
    sum = sum_of_block(x[1], lds) + ldexp(sum, -2 * kDoubleShift);
    return {1.0 / (sqrt(sum) + ldexp(a.epsilon, -kDoubleShift)), -kDoubleShift};
  }
  if (any_small) {
    __syncthreads();
    const double small = sum_of_block(x[2], lds);
    if (sum == 0.0) return {1.0 / (sqrt(small) + ldexp(a.epsilon, kDoubleShift)), kDoubleShift};
    sum += ldexp(small, -2 * kDoubleShift);
  }
  return {1.0 / (sqrt(sum) + a.epsilon), 0};
}

__device__ __forceinline__ double inverse_norm(const StartArgs& a, uint32_t matrix, uint32_t parts, double* lds) {
  double x = 0.0;
#pragma unroll
  for (uint32_t i = 0; i < kParts / 256; ++i) {
    const uint32_t at = i * 256 + threadIdx.x;
    const double y = a.partial[(int64_t)matrix * kParts + min(at, parts - 1)];
    x += at < parts ? y : 0.0;
  }
  return 1.0 / (sqrt(sum_of_block(x, lds)) + a.epsilon);
}

// Powers of two of the rows and columns of X on its shorter side, in the workspace: [matrix][..] each.
struct Exponents {
  int *rows, *columns;            // X = 2^(rows) Y, no element of a column of Y above 2^(columns)
  int* rows_of_input;             // rows' without that of 1 / (|input| + epsilon)
  double* squares;                // sums over strips of the input's rows, [matrix][strip][row]
  uint32_t* most_columns;         // bits of the largest magnitudes in columns of Y, times 2^kPairTop
  int64_t stride_squares;
  uint32_t stride_rows, stride_columns, strips;
};

// k with x <= 2^k; of 0, and of a NaN, any that no power here reaches.
template <class T>
__device__ __forceinline__ int exponent_above(T x) {
  int k = -2000;
  if (x > T(0)) (void)frexp(x, &k);
  return k;
}

constexpr uint32_t kMostStrips = 16;
constexpr int kLeastColumn = -100;   // of columns further below the rows' largest

// k with root(squares) <= 2^k.  A row of X has the exponent of its norm in the input and that of 1 / (|input| + epsilon): 2^1 at most, or 2^2 of a
// row of norm 1, which is a quarter of that then.
__device__ __forceinline__ int exponent_of_root(double squares) { return (exponent_above(squares * 1.0001) + 1) >> 1; }

// Of a column's largest magnitude, times 2^kPairTop.
__device__ __forceinline__ int column_of_most(uint32_t most, int growth) {
  return min(max(exponent_above(__builtin_bit_cast(float, most)) - kPairTop + growth, kLeastColumn), 0);
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu; }

// Rows and columns of the input that a block reads, 64 of the shorter side and 64 of the longer one: a lane's i-th element.  What is outside
// repeats the last ones.
template <bool kTall>
struct Square64 {
  uint32_t shorter, longer;       // where it is
  bool inside;
  int64_t at;                     // in the input
  __device__ __forceinline__ Square64(const StartArgs& a, uint32_t m, uint32_t n, uint32_t m0, uint32_t n0, uint32_t i) {
    const uint32_t lane = threadIdx.x % 64, other = i * 4 + threadIdx.x / 64;   // lanes along the input's rows
    shorter = m0 + (kTall ? lane : other);
    longer = n0 + (kTall ? other : lane);
    inside = shorter < m && longer < n;
    shorter = min(shorter, m - 1);
    longer = min(longer, n - 1);
    at = blockIdx.z * a.stride + (int64_t)(kTall ? longer : shorter) * a.ld + (kTall ? shorter : longer);
  }
};

// As start_norm_kernel, and the sums of squares of the input's rows on its shorter side: blocks of 64 of them by strips of 64 `tiles` of the longer
// side.  Clears the words for the columns' largest.
template <bool kTall>
__global__ void __launch_bounds__(256) start_scan_kernel(const StartArgs a, uint32_t tiles, const Exponents e) {
  __shared__ double lds[4], squares[4][64];
  const uint32_t m = kTall ? a.columns : a.rows, n = kTall ? a.rows : a.columns, part = blockIdx.y * gridDim.x + blockIdx.x;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (uint32_t i = part * 256 + threadIdx.x; i < e.stride_columns; i += gridDim.x * gridDim.y * 256) e.most_columns[blockIdx.z * (int64_t)e.stride_columns + i] = 0;
  const uint32_t m0 = blockIdx.y * 64, first = blockIdx.x * tiles * 64, end = min(first + tiles * 64, n);
  double sums[kTall ? 1 : 16] = {};   // of a lane's row; of 16 rows of a wave
  for (uint32_t n0 = first; n0 < end; n0 += 64) {
    float x[16], g[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const Square64<kTall> at(a, m, n, m0, n0, i);
      x[i] = static_cast<const float*>(a.x)[at.at];
      if (a.gradient) g[i] = static_cast<const float*>(a.gradient)[at.at];
    }
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const Square64<kTall> at(a, m, n, m0, n0, i);
      if (!at.inside) continue;
      if (a.gradient) {
        const float step = (float)a.gradient_alpha * g[i];
        x[i] = (float)a.decay * x[i] + step;
        static_cast<float*>(a.momentum)[at.at] = x[i];
        if (a.nesterov) x[i] = step + (float)a.decay * x[i];
      }
      sums[kTall ? 0 : i] += (double)x[i] * (double)x[i];
    }
  }
  double mine = sums[0];
  if constexpr (kTall) {
    squares[wave][lane] = mine;
    __syncthreads();
    if (wave == 0) mine = squares[0][lane] + squares[1][lane] + squares[2][lane] + squares[3][lane];
  } else {
    // half of the sums to the other half of the lanes at a time: row i of a wave's is lane 4 i's in the end
#pragma unroll
    for (int d = 32; d >= 4; d >>= 1)
#pragma unroll
      for (int i = 0; i < d / 4; ++i) {
        const bool high = lane & d;
        const double given = high ? sums[i] : sums[i + d / 4];
        sums[i] = (high ? sums[i + d / 4] : sums[i]) + __shfl_xor(given, d);
      }
    mine = sums[0];
    mine += __shfl_xor(mine, 2);
    mine += __shfl_xor(mine, 1);
    if (lane % 4 == 0) squares[0][lane + wave] = mine;   // row i * 4 + wave
    __syncthreads();
    if (wave == 0) mine = squares[0][lane];
  }
  if (wave == 0 && m0 + lane < m) e.squares[blockIdx.z * e.stride_squares + (int64_t)blockIdx.x * m + m0 + lane] = mine;
  const double total = sum_of_block(wave == 0 ? mine : 0.0, lds);
  if (threadIdx.x == 0) a.partial[(int64_t)blockIdx.z * kParts + part] = total;
}

// The exponents of `count` rows of the input from m0 on, in LDS, and for the next launch.
__device__ __forceinline__ void rows_of_input(const Exponents& e, uint32_t m, uint32_t m0, uint32_t count, int* rows, bool keep) {
  for (uint32_t i = threadIdx.x; i < count; i += 256) {
    const double* from = e.squares + blockIdx.z * e.stride_squares + min(m0 + i, m - 1);
    double x[kMostStrips], sum = 0.0;
#pragma unroll
    for (uint32_t strip = 0; strip < kMostStrips; ++strip) x[strip] = from[(int64_t)min(strip, e.strips - 1) * m];
#pragma unroll
    for (uint32_t strip = 0; strip < kMostStrips; ++strip) sum += strip < e.strips ? x[strip] : 0.0;
    rows[i] = exponent_of_root(sum);
    if (keep && m0 + i < m) e.rows_of_input[blockIdx.z * (int64_t)e.stride_rows + m0 + i] = rows[i];
  }
}

// The largest magnitudes of the columns of Y, or up to twice those, over strips of the shorter side, kMostAcross squares of 64 at most.
constexpr uint32_t kMostAcross = 8;
template <bool kTall>
__global__ void __launch_bounds__(256) start_columns_kernel(const StartArgs a, uint32_t tiles, const Exponents e) {
  __shared__ uint32_t most[64];
  __shared__ int rows[kMostAcross * 64];
  const uint32_t m = kTall ? a.columns : a.rows, n = kTall ? a.rows : a.columns, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t n0 = blockIdx.y * 64, first = blockIdx.x * tiles * 64, end = min(first + tiles * 64, m);
  if (threadIdx.x < 64) most[lane] = 0;
  rows_of_input(e, m, first, tiles * 64, rows, blockIdx.y == 0);
  uint32_t found[16] = {};
  bool ready = false;
  for (uint32_t m0 = first; m0 < end; m0 += 64) {
    float x[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) x[i] = start_value<float>(a, Square64<kTall>(a, m, n, m0, n0, i).at);
    if (!ready) __syncthreads();
    ready = true;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      found[i] = max(found[i], magnitude(ldexpf(x[i], kPairTop - rows[Square64<kTall>(a, m, n, m0, n0, i).shorter - first])));
  }
  if constexpr (kTall) {
#pragma unroll
    for (int d = 32; d >= 4; d >>= 1)   // as start_scan_kernel's sums
#pragma unroll
      for (int i = 0; i < d / 4; ++i) {
        const bool high = lane & d;
        const uint32_t given = high ? found[i] : found[i + d / 4];
        found[i] = max(high ? found[i + d / 4] : found[i], (uint32_t)__shfl_xor((int)given, d));
      }
    found[0] = max(found[0], (uint32_t)__shfl_xor((int)found[0], 2));
    found[0] = max(found[0], (uint32_t)__shfl_xor((int)found[0], 1));
    if (lane % 4 == 0) most[lane + wave] = found[0];
  } else {
#pragma unroll
    for (uint32_t i = 1; i < 16; ++i) found[0] = max(found[0], found[i]);
    atomicMax(&most[lane], found[0]);
  }
  __syncthreads();
  if (threadIdx.x < 64 && n0 + threadIdx.x < n) atomicMax(&e.most_columns[blockIdx.z * (int64_t)e.stride_columns + n0 + threadIdx.x], most[threadIdx.x]);
}

// 64 x 64 elements as pieces, by rows of the input and by its columns, and the exponents.
template <bool kTall>
__global__ void __launch_bounds__(256) start_pieces_kernel(const StartArgs a, uint32_t parts, const Exponents e, char* by_rows, char* by_columns,
                                                           int64_t stride_rows, int64_t stride_columns) {
  __shared__ double lds[4];
  __shared__ uint32_t cells[64][65];
  __shared__ int of_short[64], of_long[64];
  const uint32_t matrix = blockIdx.z, row0 = blockIdx.y * 64, column0 = blockIdx.x * 64, m = kTall ? a.columns : a.rows, n = kTall ? a.rows : a.columns;
  const uint32_t m0 = kTall ? column0 : row0, n0 = kTall ? row0 : column0;
  float values[16];   // on their way while the norm is added up: no branch that lanes take apart
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i) values[i] = start_value<float>(a, Square64<kTall>(a, m, n, m0, n0, i).at);
  const double factor = inverse_norm(a, matrix, parts, lds);
  const int of_factor = exponent_above(factor);
  if (threadIdx.x < 64) of_short[threadIdx.x] = e.rows_of_input[(int64_t)matrix * e.stride_rows + min(m0 + threadIdx.x, m - 1)];
  if (threadIdx.x >= 64 && threadIdx.x < 128) {
    const uint32_t at = n0 + threadIdx.x % 64;
    const int64_t to = (int64_t)matrix * e.stride_columns + min(at, n - 1);
    const int k = column_of_most(e.most_columns[to], 0);
    of_long[threadIdx.x % 64] = k;
    if (m0 == 0 && at < n) e.columns[to] = k;
  }
  __syncthreads();
  if (n0 == 0 && threadIdx.x < 64 && m0 + threadIdx.x < m) e.rows[(int64_t)matrix * e.stride_rows + m0 + threadIdx.x] = of_short[threadIdx.x] + of_factor;
  const uint32_t c = threadIdx.x % 64;
#pragma unroll
  for (uint32_t i = 0; i < 16; ++i) {
    const Square64<kTall> at(a, m, n, m0, n0, i);
    values[i] = at.inside ? (float)ldexp((double)values[i] * factor, kPairTop - of_factor - of_short[at.shorter - m0]) : 0.f;
  }
  // eight k of a row to a lane, both pieces: 64 rows of two runs
  auto put = [&](char* to, uint32_t row0, uint32_t rows, uint32_t k0, uint32_t columns, bool turned) {
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t at = i * 256 + threadIdx.x, r = at / 8, k = at % 8 * 8, run = (k0 + k) / kPairRun, runs = (columns + kPairRun - 1) / kPairRun;
      if (row0 + r >= rows || run >= runs) continue;
      pair_u32x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = turned ? cells[k + 2 * e][r] : cells[r][k + 2 * e], y = turned ? cells[k + 2 * e + 1][r] : cells[r][k + 2 * e + 1];
        hi[e] = (x & 0xffff) | y << 16;
        lo[e] = x >> 16 | (y & 0xffff0000u);
      }
      char* p = to + ((int64_t)(row0 + r) * runs + run) * kPairRunBytes + k % 32 * 2;
      *reinterpret_cast<pair_u32x4*>(p) = hi;
      *reinterpret_cast<pair_u32x4*>(p + 64) = lo;
    }
  };
#pragma unroll
  for (int with_columns = 0; with_columns < 2; ++with_columns) {   // Y, and what its columns' powers of two leave of it
    if (with_columns) __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      const uint32_t r = i * 4 + threadIdx.x / 64;
      _Float16 hi, lo;
      split_pair(with_columns ? ldexpf(values[i], -of_long[kTall ? r : c]) : values[i], &hi, &lo);
      cells[r][c] = (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
    }
    __syncthreads();
    if ((with_columns != 0) == kTall) put(by_rows + matrix * stride_rows, row0, a.rows, column0, a.columns, false);
    else put(by_columns + matrix * stride_columns, column0, a.columns, row0, a.rows, true);
  }
}

__global__ void __launch_bounds__(256) start_double_kernel(const StartArgs a, uint32_t parts, double* to, int64_t stride, uint32_t ld,
                                                           FastDiv columns_fd, uint32_t cells) {
  __shared__ double lds[4];
  const InverseNorm inverse = inverse_norm_of_doubles(a, blockIdx.y, parts, lds);
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < cells; i += gridDim.x * 256) {
    uint32_t row, column;
    columns_fd.divmod(i, row, column);
    to[blockIdx.y * stride + (int64_t)row * ld + column] = ldexp(start_value<double>(a, (int64_t)blockIdx.y * a.stride + (int64_t)row * a.ld + column), inverse.power) * inverse.factor;
  }
}

// ------------------------------------------------------------------ float

struct PairArgs {
  const char *left, *right;           // pieces, k along the rows
  int64_t left_stride, right_stride;  // between matrices, bytes
  TileOrder order;
  uint32_t m, n, runs;
  int shift;                          // powers of two in the sums
  // results as pieces, [m][n] and [n][m]; of a symmetric product only the first
  char *by_rows, *by_columns;
  int64_t rows_stride, columns_stride;
  int store;                          // powers of two of those
  const int *row_exponents, *column_exponents;   // of the results' rows and columns, [matrix][..]
  uint32_t row_exponents_stride, column_exponents_stride;
  // of kGram and kSquare: G itself, below the diagonal and in the squares of 32 on it, [matrix][m][m]
  float* gram;
  int64_t gram_stride;
  float a, b, c;                      // of kSquare
  // G's diagonal, as of kGram, and the exponents of the rows that follow from it (next_row); of kUpdate the columns' next ones and largest elements
  uint32_t* squares;
  int *next_rows, *next_columns;
  const uint32_t* most;
  uint32_t* next_most;
  uint32_t clear;                     // of kSquare: words of next_most
  float most_factor;
  int most_next, least_change, growth;
  // of kLast: out = alpha * (sums) + beta * out
  float* out;
  int64_t ldo, out_stride;
  float alpha, beta;
};

// The exponent of a row after a step, from its own and its square in G.  |x'| <= |x| most_factor, and below the bound of all singular values.  It
// falls no faster than by least_change: smaller rows are then just smaller in Y, and a column's growth has a bound.
__device__ __forceinline__ int next_row(const PairArgs& a, uint32_t square, int exponent) {
  const int norm = exponent_above(sqrtf(fmaxf(__builtin_bit_cast(float, square), 0.f)) * a.most_factor);
  return max(min(exponent + norm, a.most_next), exponent + a.least_change);
}

// What a block's tile needs of exponents, a lane's row and column: read ahead of the products, and put in LDS behind them.
struct Staged {
  int row, column;
  uint32_t square, most;
};
template <Product kProduct>
__device__ __forceinline__ Staged staged_exponents(const PairArgs& a, const TilePlace& at, uint32_t row0, uint32_t column0) {
  const int64_t row = (int64_t)at.matrix * a.row_exponents_stride + min(row0 + threadIdx.x, a.m - 1);
  const int64_t column = (int64_t)at.matrix * a.column_exponents_stride + min(column0 + threadIdx.x, a.n - 1);
  Staged s{a.row_exponents[row], a.column_exponents[column], 0, 0};
  if constexpr (kProduct == kUpdate) {
    s.square = a.squares[row];
    s.most = a.most[column];
  }
  return s;
}

// Of kUpdate's rows by how much they change.  The first tiles of rows and columns record what follows.
template <Product kProduct>
__device__ __forceinline__ void put_exponents(const PairArgs& a, const TilePlace& at, uint32_t row0, uint32_t rows, uint32_t column0, uint32_t columns,
                                              Staged s, int* of_rows, int* of_columns, int* of_next) {
  if (threadIdx.x < rows) {
    if constexpr (kProduct == kUpdate) {
      const int next = next_row(a, s.square, s.row);
      if (at.n_tile == 0 && row0 + threadIdx.x < a.m) a.next_rows[(int64_t)at.matrix * a.row_exponents_stride + row0 + threadIdx.x] = next;
      s.row -= next;
    }
    of_rows[threadIdx.x] = s.row;
  }
  if (threadIdx.x < columns) {
    of_columns[threadIdx.x] = s.column;
    if constexpr (kProduct == kUpdate) {
      const int next = column_of_most(s.most, a.growth);
      if (at.m_tile == 0 && column0 + threadIdx.x < a.n) a.next_columns[(int64_t)at.matrix * a.column_exponents_stride + column0 + threadIdx.x] = next;
      of_next[threadIdx.x] = next;
    }
  }
}

// Words that kUpdate records to, before it.
template <Product kProduct, uint32_t kThreads>
__device__ __forceinline__ void clear_most(const PairArgs& a) {
  if constexpr (kProduct == kSquare) {
    for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < a.clear; i += gridDim.x * kThreads) a.next_most[i] = 0;
  }
}

// Two results that are stored of a cell's sum: at (row, column), and at (column, row) of what lies by columns.
struct Stored {
  float by_rows, by_columns;
};
// `gram`: G's cell.
template <Product kProduct>
__device__ __forceinline__ Stored results_of(const PairArgs& a, float sum, float gram, bool diagonal, int row, int column, int next) {
  if constexpr (kProduct == kGram) {
    return {ldexpf(sum, column + a.store), ldexpf(sum, row + a.store)};
  } else if constexpr (kProduct == kSquare) {
    const float x = a.c * sum + a.b * gram, i = diagonal ? a.a : 0.f;
    return {ldexpf(ldexpf(x, 2 * column) + i, a.store), ldexpf(ldexpf(x, 2 * row) + i, a.store)};
  } else {
    const float x = ldexpf(sum, row + column);
    return {x, ldexpf(x, -next)};
  }
}

// Tiles of SM x SN by WM x WN waves, loads kAhead runs ahead.
template <int SM_, int SN_, int WM_, int WN_, int kAhead_>
struct PairTile {
  static constexpr int SM = SM_, SN = SN_, WM = WM_, WN = WN_, kAhead = kAhead_, T = 64 * WM * WN, MT = SM / WM / 32, NT = SN / WN / 32;
  static constexpr bool kTall = SM != SN;
  static_assert(!kTall || SM * 3 == SN * 4, "what place_of_unit counts");
};
using Tile256 = PairTile<256, 256, 2, 4, 1>;
using TileTall = PairTile<256, 192, 4, 2, 1>;
using Tile128 = PairTile<128, 128, 2, 2, 1>;
using Tile64 = PairTile<64, 64, 2, 2, 2>;

// Results of a wave's 32 x 32 cells go to memory in whole lines: by way of an image in LDS, rows of 32 with both pieces in a word,
// from which eight lanes take a run of a row, or of a column.  (Stored from the registers a line of 128 bytes took 16 instructions of a few
// bytes each: 16 us to a block of 256 x 256.)
// Orders what the lanes of a wave write to LDS and read there.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr uint32_t kImagePitch = 36, kImageWords = 32 * kImagePitch;

__device__ __forceinline__ void store_lines(const uint32_t* image, uint32_t lane, bool turned, char* to, uint32_t row0, uint32_t rows, uint32_t runs,
                                            uint32_t run) {
  if (run >= runs) return;
  const uint32_t pieces = lane >> 2 & 1 ? 0x07060302u : 0x05040100u, k = lane % 4 * 8;   // both words' upper halves, or lower ones
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t r = i * 8 + lane / 8;
    uint32_t w[8];
    if (turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = image[(k + e) * kImagePitch + r];
    } else {
      const pair_u32x4 x = *reinterpret_cast<const pair_u32x4*>(image + r * kImagePitch + k), y = *reinterpret_cast<const pair_u32x4*>(image + r * kImagePitch + k + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = x[e];
        w[e + 4] = y[e];
      }
    }
    pair_u32x4 line;
#pragma unroll
    for (int e = 0; e < 4; ++e) line[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], pieces);
    if (row0 + r < rows) *reinterpret_cast<pair_u32x4*>(to + ((int64_t)(row0 + r) * runs + run) * kPairRunBytes + lane % 8 * 16) = line;
  }
}

template <class Tile, Product kProduct>
__global__ void __launch_bounds__(Tile::T, 2) pair_kernel(const PairArgs a) {
  constexpr int SM = Tile::SM, SN = Tile::SN, WM = Tile::WM, WN = Tile::WN, MT = Tile::MT, NT = Tile::NT;
  __shared__ __attribute__((aligned(16))) char lds[pair_tile_lds(SM, SN)];
  static_assert(WM * WN * kImageWords * 4 + (SM + 2 * SN) * 4 <= pair_tile_lds(SM, SN), "an image to a wave, and exponents");
  clear_most<kProduct, Tile::T>(a);
  TilePlace at;
  if (!place_of<is_symmetric(kProduct), Tile::kTall>(a.order, &at)) return;
  const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const uint32_t row0 = at.m_tile * SM, column0 = at.n_tile * SN, row_bytes = a.runs * kPairRunBytes;
  if (Tile::kTall && column0 >= a.n) return;   // a last row of tiles may be counted longer than it is
  static_assert(SM <= Tile::T && SN <= Tile::T, "a row and a column to a lane");
  const Staged staged = staged_exponents<kProduct>(a, at, row0, column0);
  const char* left = a.left + at.matrix * a.left_stride;
  pair_f32x16 sums[1][MT][NT];
  const PairMatrices<SM, SN, Tile::T> source(left + (int64_t)row0 * row_bytes, a.m - 1 - row0, a.right + at.matrix * a.right_stride + (int64_t)column0 * row_bytes,
                                           a.n - 1 - column0, row_bytes, tid);
  pair_tile<SM, SN, WM, WN, Tile::kAhead, false>(source, a.runs, lds, tid, sums);
  pair_f32x16 (&sum)[MT][NT] = sums[0];
  const uint32_t wave_m = row0 + wave / WN * (MT * 32), wave_n = column0 + wave % WN * (NT * 32), c = lane & 31, half = lane >> 5;
  int* const of_rows = reinterpret_cast<int*>(lds) + WM * WN * kImageWords;
  int *const of_columns = of_rows + SM, *const of_next = of_columns + SN;
  __syncthreads();
  put_exponents<kProduct>(a, at, row0, SM, column0, SN, staged, of_rows, of_columns, of_next);
  __syncthreads();
  if constexpr (kProduct == kLast) {
    float* out = a.out + at.matrix * a.out_stride;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const uint32_t n = wave_n + u * 32 + c;
      if (n >= a.n) continue;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float* const cells = out + (int64_t)(wave_m + t * 32 + 4 * half) * a.ldo + n;
        const uint32_t rows = a.m - min(wave_m + t * 32 + 4 * half, a.m);
        float before[16];   // all on their way before the first is stored
        if (a.beta != 0.f) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8u * (r / 4) + r % 4 < rows) before[r] = cells[(int64_t)(8 * (r / 4) + r % 4) * a.ldo];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float value = a.alpha * ldexpf(sum[t][u][r], a.shift + of_rows[wave_m - row0 + t * 32 + 4 * half + 8 * (r / 4) + r % 4] + of_columns[n - column0]);
          if (8u * (r / 4) + r % 4 < rows) cells[(int64_t)(8 * (r / 4) + r % 4) * a.ldo] = a.beta == 0.f ? value : value + a.beta * before[r];
        }
      }
    }
  } else {
    // k along the columns of these results, and along the rows
    const uint32_t runs_n = (a.n + kPairRun - 1) / kPairRun, runs_m = (a.m + kPairRun - 1) / kPairRun;
    char* by_rows = a.by_rows + at.matrix * a.rows_stride;
    char* by_columns = is_symmetric(kProduct) ? by_rows : a.by_columns + at.matrix * a.columns_stride;
    uint32_t* image = reinterpret_cast<uint32_t*>(lds) + wave * kImageWords;
    float* gram = a.gram + at.matrix * a.gram_stride;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const uint32_t n0 = wave_n + u * 32;
      const int column = of_columns[n0 - column0 + c], next = kProduct == kUpdate ? of_next[n0 - column0 + c] : 0;
      uint32_t most = 0;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const uint32_t m0 = wave_m + t * 32;
        if (m0 >= a.m || n0 >= a.n || (is_symmetric(kProduct) && m0 < n0)) continue;
        float before[16];   // G's cells, all on their way before the first is used
        if constexpr (kProduct == kSquare) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            before[r] = gram[(int64_t)min(m0 + 8 * (r / 4) + 4 * half + r % 4, a.m - 1) * a.m + min(n0 + c, a.n - 1)];
        }
        float x[16];
        int of_row[16];   // read ahead: behind a condition each read would be waited for by itself
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          of_row[r] = of_rows[m0 - row0 + 8 * (r / 4) + 4 * half + r % 4];
          x[r] = ldexpf(sum[t][u][r], a.shift);
        }
        auto results = [&](int r) {
          return results_of<kProduct>(a, x[r], kProduct == kSquare ? before[r] : 0.f, m0 + 8 * (r / 4) + 4 * half + r % 4 == n0 + c, of_row[r], column, next);
        };
        const bool whole = m0 + 32 <= a.m && n0 + 32 <= a.n;
        auto put = [&](int r, float value) {
          const uint32_t row = 8 * (r / 4) + 4 * half + r % 4;
          if (!whole) value = m0 + row < a.m && n0 + c < a.n ? value : 0.f;
          _Float16 hi, lo;
          split_pair(value, &hi, &lo);
          image[row * kImagePitch + c] = (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
        };
        if constexpr (kProduct == kGram) {
          float* const cells = gram + (int64_t)(m0 + 4 * half) * a.m + n0 + c;
          const uint32_t rows = n0 + c < a.n ? a.m - min(m0 + 4 * half, a.m) : 0;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8u * (r / 4) + r % 4 < rows) cells[(int64_t)(8 * (r / 4) + r % 4) * a.m] = x[r];
          if (m0 == n0 && c < a.n - n0) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (8u * (r / 4) + 4 * half + r % 4 == c) a.squares[(int64_t)at.matrix * a.row_exponents_stride + n0 + c] = __builtin_bit_cast(uint32_t, x[r]);
          }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float value = results(r).by_rows;
          if constexpr (kProduct == kUpdate) most = max(most, magnitude(value));   // rows beyond the last repeat it
          put(r, value);
        }
        wave_fence();
        store_lines(image, lane, false, by_rows, m0, a.m, runs_n, n0 / 32);
        if (is_symmetric(kProduct) && m0 == n0) {
          wave_fence();
          continue;
        }
        // one image for both where they are the same, as they mostly are
        const bool same = is_symmetric(kProduct) ? __all(of_rows[m0 - row0 + c] == column && column == __builtin_amdgcn_readfirstlane(column)) : __all(next == 0);
        if (!same) {
          wave_fence();
#pragma unroll
          for (int r = 0; r < 16; ++r) put(r, results(r).by_columns);
          wave_fence();
        }
        store_lines(image, lane, true, by_columns, n0, a.n, runs_m, m0 / 32);
        wave_fence();
      }
      if constexpr (kProduct == kUpdate) {
        most = max(most, (uint32_t)__shfl_xor((int)most, 32));
        if (half == 0 && n0 + c < a.n) atomicMax(&a.next_most[(int64_t)at.matrix * a.column_exponents_stride + n0 + c], most);
      }
    }
  }
}

// Products too small to fill the chip with such tiles: a block owns 32 x 32, its W waves take every W-th of the runs first .. end - 1 each,
// straight from memory into the operands of v_mfma_f32_16x16x32_f16, whose 16 rows of a piece of a run are 16 times 64 bytes.  Nothing is
// left out of the products.  The sums of all waves, added in their order: cell i of a lane's, of cells_at(i).
typedef float pair_f32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kSmallSide = 32, kSmallCells = kSmallSide * kSmallSide;

template <int W>
__device__ __forceinline__ void small_sums(const char* left, uint32_t last_left, const char* right, uint32_t last_right, int64_t row_bytes, uint32_t first,
                                           uint32_t end, float (&partial)[W][kSmallCells]) {
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Every other row's pieces change places, so that a load's 64 bytes of each of sixteen lines fall on all banks of a cache (512 x 512 in five steps
  // 131 -> 108 us): all four products are formed whichever comes first.
  const int32_t first_piece = lane % 2 * 64, other_piece = 64 - first_piece;
  const char *l[2], *r[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    l[t] = left + min(t * 16 + lane % 16, last_left) * row_bytes + lane / 16 * 16;
    r[t] = right + min(t * 16 + lane % 16, last_right) * row_bytes + lane / 16 * 16;
  }
  f16x8 x[2][2][2], y[2][2][2];   // of two runs; [][rows][piece]
  auto load = [&](uint32_t run, int slot) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        x[slot][t][p] = *reinterpret_cast<const f16x8*>(l[t] + (int64_t)run * kPairRunBytes + (p == 0 ? first_piece : other_piece));
        y[slot][t][p] = *reinterpret_cast<const f16x8*>(r[t] + (int64_t)run * kPairRunBytes + (p == 0 ? first_piece : other_piece));
      }
  };
  pair_f32x4 sum[2][2] = {};
  auto multiply = [&](int slot) {
#pragma unroll
    for (int i = 3; i >= 0; --i)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) sum[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[slot][t][i / 2], y[slot][u][i % 2], sum[t][u], 0, 0, 0);
  };
  uint32_t run = first + wave;
  if (run < end) {
    load(run, 0);
    for (; run + 2 * W < end; run += 2 * W) {   // no load behind a branch, which would be waited for at once
      load(run + W, 1);
      multiply(0);
      load(run + 2 * W, 0);
      multiply(1);
    }
    if (run + W < end) {
      load(run + W, 1);
      multiply(0);
      multiply(1);
    } else {
      multiply(0);
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) partial[wave][(t * 16 + lane / 16 * 4 + e) * kSmallSide + u * 16 + lane % 16] = sum[t][u][e];
  __syncthreads();
}

// What a block of 32 x 32 keeps: images of the results by rows and by columns, and the columns' largest elements.
struct SmallImage {
  uint32_t by_rows[kImageWords], by_columns[kImageWords];
  uint32_t most[kSmallSide];
};

// What a lane's cells (cell i * kThreads + threadIdx.x, all of one column) need besides their sums: read ahead of those.
template <Product kProduct, uint32_t kThreads>
struct SmallCells {
  static constexpr uint32_t kCells = kSmallCells / kThreads;
  int rows[kCells], column, next = 0;
  uint32_t squares[kCells], most;
  float gram[kCells];
  __device__ __forceinline__ SmallCells(const PairArgs& a, const TilePlace& at, SmallImage& image) {
    const uint32_t n = min(at.n_tile * kSmallSide + threadIdx.x % kSmallSide, a.n - 1);
    const int64_t of_row = (int64_t)at.matrix * a.row_exponents_stride, of_column = (int64_t)at.matrix * a.column_exponents_stride;
    column = a.column_exponents[of_column + n];
    if constexpr (kProduct == kUpdate) most = a.most[of_column + n];
#pragma unroll
    for (uint32_t i = 0; i < kCells; ++i) {
      const uint32_t m = min(at.m_tile * kSmallSide + (i * kThreads + threadIdx.x) / kSmallSide, a.m - 1);
      rows[i] = a.row_exponents[of_row + m];
      if constexpr (kProduct == kUpdate) squares[i] = a.squares[of_row + m];
      gram[i] = kProduct == kSquare ? a.gram[at.matrix * a.gram_stride + (int64_t)m * a.m + n] : 0.f;
    }
    if (threadIdx.x < kSmallSide) image.most[threadIdx.x] = 0;
  }
  // Behind the sums: the exponents after the step, which the first tiles of rows and columns record.
  __device__ __forceinline__ void step(const PairArgs& a, const TilePlace& at) {
    if constexpr (kProduct == kUpdate) {
      next = column_of_most(most, a.growth);
      const uint32_t n = at.n_tile * kSmallSide + threadIdx.x;
      if (at.m_tile == 0 && threadIdx.x < kSmallSide && n < a.n) a.next_columns[(int64_t)at.matrix * a.column_exponents_stride + n] = next;
#pragma unroll
      for (uint32_t i = 0; i < kCells; ++i) {
        const uint32_t m = at.m_tile * kSmallSide + (i * kThreads + threadIdx.x) / kSmallSide;
        const int next_one = next_row(a, squares[i], rows[i]);
        if (at.n_tile == 0 && threadIdx.x % kSmallSide == 0 && m < a.m) a.next_rows[(int64_t)at.matrix * a.row_exponents_stride + m] = next_one;
        rows[i] -= next_one;
      }
    }
  }
  // The i-th cell's result: to the images, or where it is for.
  __device__ __forceinline__ void finish(const PairArgs& a, const TilePlace& at, uint32_t i, float x, SmallImage& image) {
    const uint32_t cell = i * kThreads + threadIdx.x, row = cell / kSmallSide, c = cell % kSmallSide, m = at.m_tile * kSmallSide + row, n = at.n_tile * kSmallSide + c;
    const bool inside = m < a.m && n < a.n;
    if constexpr (kProduct == kLast) {
      if (!inside) return;
      x = ldexpf(x, a.shift + rows[i] + column);
      float& to = a.out[at.matrix * a.out_stride + (int64_t)m * a.ldo + n];
      to = a.beta == 0.f ? a.alpha * x : a.alpha * x + a.beta * to;
    } else {
      x = ldexpf(x, a.shift);
      if (kProduct == kGram && inside) {
        a.gram[at.matrix * a.gram_stride + (int64_t)m * a.m + n] = x;
        if (m == n) a.squares[(int64_t)at.matrix * a.row_exponents_stride + m] = __builtin_bit_cast(uint32_t, x);
      }
      const Stored to = results_of<kProduct>(a, x, gram[i], m == n, rows[i], column, next);
      if (kProduct == kUpdate && inside) atomicMax(&image.most[c], magnitude(to.by_rows));
      auto put = [&](uint32_t* words, float value) {
        _Float16 hi, lo;
        split_pair(inside ? value : 0.f, &hi, &lo);
        words[row * kImagePitch + c] = (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
      };
      put(image.by_rows, to.by_rows);
      put(image.by_columns, to.by_columns);
    }
  }
};

// Two waves store the images.
template <Product kProduct>
__device__ __forceinline__ void store_small(const PairArgs& a, const TilePlace& at, const SmallImage& image) {
  const uint32_t runs_n = (a.n + kPairRun - 1) / kPairRun, runs_m = (a.m + kPairRun - 1) / kPairRun, wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  __syncthreads();
  if (wave == 0) store_lines(image.by_rows, lane, false, a.by_rows + at.matrix * a.rows_stride, at.m_tile * kSmallSide, a.m, runs_n, at.n_tile);
  if (wave == 1 && (!is_symmetric(kProduct) || at.m_tile != at.n_tile))
    store_lines(image.by_columns, lane, true, is_symmetric(kProduct) ? a.by_rows + at.matrix * a.rows_stride : a.by_columns + at.matrix * a.columns_stride,
                at.n_tile * kSmallSide, a.n, runs_m, at.m_tile);
  if (kProduct == kUpdate && wave == 2 && lane < kSmallSide && at.n_tile * kSmallSide + lane < a.n)
    atomicMax(&a.next_most[(int64_t)at.matrix * a.column_exponents_stride + at.n_tile * kSmallSide + lane], image.most[lane]);
}

template <int W, Product kProduct>
__global__ void __launch_bounds__(64 * W, 4) pair_small_kernel(const PairArgs a) {
  __shared__ float partial[W][kSmallCells];
  __shared__ __attribute__((aligned(16))) SmallImage image;
  clear_most<kProduct, 64 * W>(a);
  TilePlace at;
  if (!place_of<is_symmetric(kProduct)>(a.order, &at)) return;
  const int64_t row_bytes = (int64_t)a.runs * kPairRunBytes;
  const uint32_t row0 = at.m_tile * kSmallSide, column0 = at.n_tile * kSmallSide;
  SmallCells<kProduct, 64 * W> cells(a, at, image);
  small_sums<W>(a.left + at.matrix * a.left_stride + row0 * row_bytes, a.m - 1 - row0, a.right + at.matrix * a.right_stride + column0 * row_bytes,
                a.n - 1 - column0, row_bytes, 0, a.runs, partial);
  cells.step(a, at);
#pragma unroll
  for (uint32_t i = 0; i < cells.kCells; ++i) {
    const uint32_t cell = i * 64 * W + threadIdx.x;
    float x = partial[0][cell];
#pragma unroll
    for (int w = 1; w < W; ++w) x += partial[w][cell];
    cells.finish(a, at, i, x, image);
  }
  if constexpr (kProduct != kLast) store_small<kProduct>(a, at, image);
}

// X X^T of few rows that are long: parts of k to a block each, [matrix][tile][part], and a second launch that adds them up, in their order
// (200 x 8000 41 us in one launch, 13 in two).
constexpr int kPartWaves = 8;
__global__ void __launch_bounds__(64 * kPartWaves, 4) gram_part_kernel(const PairArgs a, uint32_t part_runs, FastDiv parts_fd, float* sums, int64_t sums_stride) {
  __shared__ float partial[kPartWaves][kSmallCells];
  uint32_t unit, part;
  parts_fd.divmod(blockIdx.x, unit, part);
  TilePlace at;
  if (!place_of_unit<true>(a.order, unit, &at)) return;
  const int64_t row_bytes = (int64_t)a.runs * kPairRunBytes;
  const uint32_t row0 = at.m_tile * kSmallSide, column0 = at.n_tile * kSmallSide;
  const char* x = a.left + at.matrix * a.left_stride;
  small_sums<kPartWaves>(x + row0 * row_bytes, a.m - 1 - row0, x + column0 * row_bytes, a.n - 1 - column0, row_bytes, part * part_runs,
                         min((part + 1) * part_runs, a.runs), partial);
  float* to = sums + at.matrix * sums_stride + ((int64_t)(unit - at.matrix * a.order.tiles) * parts_fd.d + part) * kSmallCells;
#pragma unroll
  for (uint32_t i = threadIdx.x; i < kSmallCells; i += 64 * kPartWaves) {
    float sum = partial[0][i];
#pragma unroll
    for (int w = 1; w < kPartWaves; ++w) sum += partial[w][i];
    to[i] = sum;
  }
}

__global__ void __launch_bounds__(256) gram_join_kernel(const PairArgs a, uint32_t parts, const float* sums, int64_t sums_stride) {
  __shared__ __attribute__((aligned(16))) SmallImage image;
  TilePlace at;
  if (!place_of_unit<true>(a.order, blockIdx.x, &at)) return;
  SmallCells<kGram, 256> cells(a, at, image);
  const float* from = sums + at.matrix * sums_stride + (int64_t)(blockIdx.x - at.matrix * a.order.tiles) * parts * kSmallCells + threadIdx.x;
  float x[kSmallCells / 256] = {};
  for (uint32_t part0 = 0; part0 < parts; part0 += 8) {   // loads of eight parts on their way
    float y[8][kSmallCells / 256];
#pragma unroll
    for (uint32_t p = 0; p < 8; ++p)
#pragma unroll
      for (uint32_t i = 0; i < kSmallCells / 256; ++i) y[p][i] = from[(int64_t)min(part0 + p, parts - 1) * kSmallCells + i * 256];
#pragma unroll
    for (uint32_t p = 0; p < 8; ++p)
#pragma unroll
      for (uint32_t i = 0; i < kSmallCells / 256; ++i) x[i] += part0 + p < parts ? y[p][i] : 0.f;
  }
#pragma unroll
  for (uint32_t i = 0; i < kSmallCells / 256; ++i) cells.finish(a, at, i, x[i], image);
  store_small<kGram>(a, at, image);
}

// ------------------------------------------------------------------ double

// Matrices lie as they are given, wide ([m][n], m <= n) or tall ([n][m]), with rows 16 bytes beyond a whole number of lines of 128 bytes apart,
// so that 64 bytes of each of sixteen rows fall on all banks of a cache alike (X X^T of 1024 x 1024 37 us; with 1024, or an odd number of
// lines, from row to row 48).
struct DoubleArgs {
  const double* x;
  const double* square;   // A, or B
  double* out;
  int64_t x_stride, square_stride, out_stride, ldo;
  TileOrder order;
  uint32_t m, n;          // rows and columns of the results
  uint32_t depth, ldx, ld_square;
  double a, b, c, alpha, beta;
};

// Large products: tiles of 64 staged in LDS.
constexpr uint32_t kDoubleSide = 64;

template <Product kProduct, bool kTall>
__global__ void __launch_bounds__(256, 2) ortho_double_kernel(const DoubleArgs a) {
  constexpr uint32_t S = kDoubleSide;
  using Row = DoubleRow<S>;
  using Columns = DoubleColumns<S>;
  TilePlace at;
  if (!place_of<is_symmetric(kProduct)>(a.order, &at)) return;
  const uint32_t row0 = at.m_tile * S, column0 = at.n_tile * S;
  const double* x = a.x + at.matrix * a.x_stride;
  const double* square = a.square + at.matrix * a.square_stride;
  double* out = a.out + at.matrix * a.out_stride;
  auto row_of = [&](const double* p, uint32_t ld, uint32_t first, uint32_t rows) {
    return Row{p + (int64_t)min(first + Row::row(), rows - 1) * ld, a.depth, true};
  };
  auto columns_of = [&](const double* p, uint32_t ld, uint32_t first, uint32_t columns) {
    return Columns(p + first, ld, nullptr, 0, a.depth, a.depth, columns - first);
  };
  if constexpr (is_symmetric(kProduct)) {
    auto store = [&](uint32_t r, uint32_t n, double sum) {
      r += row0;
      n += column0;
      if (r >= a.m || n >= a.n || r < n) return;
      if constexpr (kProduct == kSquare) sum = a.c * sum + a.b * square[(int64_t)r * a.ld_square + n] + (r == n ? a.a : 0.0);
      out[(int64_t)r * a.ldo + n] = sum;
      out[(int64_t)n * a.ldo + r] = sum;
    };
    if constexpr (kProduct == kSquare) double_tile<S>(a.depth, row_of(square, a.ld_square, row0, a.m), row_of(square, a.ld_square, column0, a.n), store);
    else if constexpr (kTall) double_tile<S>(a.depth, columns_of(x, a.ldx, row0, a.m), columns_of(x, a.ldx, column0, a.n), store);
    else double_tile<S>(a.depth, row_of(x, a.ldx, row0, a.m), row_of(x, a.ldx, column0, a.n), store);
  } else {
    auto store = [&](uint32_t r, uint32_t n, double sum) {
      if (row0 + r >= a.m || column0 + n >= a.n) return;
      double& cell = out[(int64_t)(row0 + r) * a.ldo + column0 + n];
      if constexpr (kProduct == kUpdate) cell = sum;
      else cell = a.beta == 0.0 ? a.alpha * sum : a.alpha * sum + a.beta * cell;
    };
    if constexpr (kTall) double_tile<S>(a.depth, row_of(x, a.ldx, row0, a.m), row_of(square, a.ld_square, column0, a.n), store);
    else double_tile<S>(a.depth, row_of(square, a.ld_square, row0, a.m), columns_of(x, a.ldx, column0, a.n), store);
  }
}

// Smaller ones: 32 x 32 by four waves, straight from memory.  X X^T of few rows that are long: parts of k to a block each, whose sums a second
// launch adds up, in their order (64 x 8000 110 us in one launch, 13 in two).
constexpr int kDirectWaves = 4;
using DirectSums = double[kDirectWaves][kDirectSide * kDirectPitch];

template <Product kProduct, bool kTall>
__device__ __forceinline__ void direct_sums(const DoubleArgs& a, const TilePlace& at, uint32_t first, uint32_t depth, DirectSums& partial) {
  using Rows = DoubleDirect<true>;
  using Columns = DoubleDirect<false>;
  const uint32_t row0 = at.m_tile * kDirectSide, column0 = at.n_tile * kDirectSide;
  const double* x = a.x + at.matrix * a.x_stride;
  const double* square = a.square + at.matrix * a.square_stride;
  auto rows_of = [&](const double* p, uint32_t ld, uint32_t row, uint32_t rows) {
    return Rows::rows(p + first, ld, [&](uint32_t r) { return (int64_t)min(row + r, rows - 1); });
  };
  auto columns_of = [&](const double* p, uint32_t ld, uint32_t column, uint32_t columns) {
    return Columns::columns(p + (int64_t)first * ld + column, ld, columns - column);
  };
  if constexpr (kProduct == kSquare) double_direct(depth, rows_of(square, a.ld_square, row0, a.m), rows_of(square, a.ld_square, column0, a.n), partial);
  else if constexpr (kProduct == kGram && kTall) double_direct(depth, columns_of(x, a.ldx, row0, a.m), columns_of(x, a.ldx, column0, a.n), partial);
  else if constexpr (kProduct == kGram) double_direct(depth, rows_of(x, a.ldx, row0, a.m), rows_of(x, a.ldx, column0, a.n), partial);
  else if constexpr (kTall) double_direct(depth, rows_of(x, a.ldx, row0, a.m), rows_of(square, a.ld_square, column0, a.n), partial);
  else double_direct(depth, rows_of(square, a.ld_square, row0, a.m), columns_of(x, a.ldx, column0, a.n), partial);
}

// A block's 32 x 32 cells, four of them a lane's.
constexpr uint32_t kDirectCells = kDirectSide * kDirectSide / (64 * kDirectWaves);

// Cells at and below the diagonal, and what is above it from those.
__device__ __forceinline__ void store_symmetric(const DoubleArgs& a, const TilePlace& at, const double (&sums)[kDirectCells], double* image) {
  double* out = a.out + at.matrix * a.out_stride;
  const uint32_t row0 = at.m_tile * kDirectSide, column0 = at.n_tile * kDirectSide;
#pragma unroll
  for (uint32_t i = 0; i < kDirectCells; ++i) {
    const uint32_t cell = i * 64 * kDirectWaves + threadIdx.x, r = cell / kDirectSide, n = cell % kDirectSide, m = row0 + r, c = column0 + n;
    image[r * kDirectPitch + n] = sums[i];
    if (m < a.m && m >= c) out[(int64_t)m * a.ldo + c] = sums[i];
  }
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kDirectCells; ++i) {
    const uint32_t cell = i * 64 * kDirectWaves + threadIdx.x, r = cell % kDirectSide, n = cell / kDirectSide, m = row0 + r, c = column0 + n;
    if (m < a.m && m > c) out[(int64_t)c * a.ldo + m] = image[r * kDirectPitch + n];
  }
}

template <Product kProduct, bool kTall>
__global__ void __launch_bounds__(64 * kDirectWaves, 2) ortho_direct_kernel(const DoubleArgs a) {
  __shared__ DirectSums partial;
  TilePlace at;
  if (!place_of<is_symmetric(kProduct)>(a.order, &at)) return;
  const uint32_t row0 = at.m_tile * kDirectSide, column0 = at.n_tile * kDirectSide;
  double* out = a.out + at.matrix * a.out_stride;
  // what the results are added to, on its way meanwhile
  double before[kDirectCells], sums[kDirectCells];
#pragma unroll
  for (uint32_t i = 0; i < kDirectCells; ++i) {
    const uint32_t cell = i * 64 * kDirectWaves + threadIdx.x, r = min(row0 + cell / kDirectSide, a.m - 1), n = min(column0 + cell % kDirectSide, a.n - 1);
    if constexpr (kProduct == kSquare) before[i] = a.square[at.matrix * a.square_stride + (int64_t)r * a.ld_square + n];
    if constexpr (kProduct == kLast) before[i] = a.beta == 0.0 ? 0.0 : out[(int64_t)r * a.ldo + n];
  }
  direct_sums<kProduct, kTall>(a, at, 0, a.depth, partial);
#pragma unroll
  for (uint32_t i = 0; i < kDirectCells; ++i) {
    const uint32_t cell = i * 64 * kDirectWaves + threadIdx.x, r = cell / kDirectSide, n = cell % kDirectSide;
    sums[i] = direct_sum(partial, r, n);
    if constexpr (kProduct == kSquare) sums[i] = a.c * sums[i] + a.b * before[i] + (row0 + r == column0 + n ? a.a : 0.0);
    if constexpr (kProduct == kLast) sums[i] = a.beta == 0.0 ? a.alpha * sums[i] : a.alpha * sums[i] + a.beta * before[i];
    if (!is_symmetric(kProduct) && row0 + r < a.m && column0 + n < a.n) out[(int64_t)(row0 + r) * a.ldo + column0 + n] = sums[i];
  }
  if constexpr (is_symmetric(kProduct)) store_symmetric(a, at, sums, partial[0]);   // lanes have read their own cells
}

// [matrix][tile][part][cell]
template <bool kTall>
__global__ void __launch_bounds__(64 * kDirectWaves, 2) direct_part_kernel(const DoubleArgs a, uint32_t part_depth, FastDiv parts_fd, double* room, int64_t room_stride) {
  __shared__ DirectSums partial;
  uint32_t unit, part;
  parts_fd.divmod(blockIdx.x, unit, part);
  TilePlace at;
  if (!place_of_unit<true>(a.order, unit, &at)) return;
  direct_sums<kGram, kTall>(a, at, part * part_depth, min(part_depth, a.depth - part * part_depth), partial);
  double* to = room + at.matrix * room_stride + ((int64_t)(unit - at.matrix * a.order.tiles) * parts_fd.d + part) * (kDirectSide * kDirectSide);
#pragma unroll
  for (uint32_t i = 0; i < kDirectCells; ++i) {
    const uint32_t cell = i * 64 * kDirectWaves + threadIdx.x;
    to[cell] = direct_sum(partial, cell / kDirectSide, cell % kDirectSide);
  }
}

__global__ void __launch_bounds__(64 * kDirectWaves) direct_join_kernel(const DoubleArgs a, uint32_t parts, const double* room, int64_t room_stride) {
  __shared__ double image[kDirectSide * kDirectPitch];
  TilePlace at;
  if (!place_of_unit<true>(a.order, blockIdx.x, &at)) return;
  const double* from = room + at.matrix * room_stride + (int64_t)(blockIdx.x - at.matrix * a.order.tiles) * parts * (kDirectSide * kDirectSide) + threadIdx.x;
  double sums[kDirectCells] = {};
  for (uint32_t part0 = 0; part0 < parts; part0 += 8) {   // loads of eight parts on their way
    double y[8][kDirectCells];
#pragma unroll
    for (uint32_t p = 0; p < 8; ++p)
#pragma unroll
      for (uint32_t i = 0; i < kDirectCells; ++i) y[p][i] = from[(int64_t)min(part0 + p, parts - 1) * (kDirectSide * kDirectSide) + i * 64 * kDirectWaves];
#pragma unroll
    for (uint32_t p = 0; p < 8; ++p)
#pragma unroll
      for (uint32_t i = 0; i < kDirectCells; ++i) sums[i] += part0 + p < parts ? y[p][i] : 0.0;
  }
  store_symmetric(a, at, sums, image);
}

// ------------------------------------------------------------------ the host's side

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t aligned(int64_t bytes) { return ceil_div(bytes, 256) * 256; }

constexpr int64_t kMostSide = int64_t(1) << 21, kMostCount = 65535, kMostStride = int64_t(1) << 40;
constexpr int kMostSteps = 64;

int64_t spread_rows(int64_t doubles) { return ceil_div(std::max<int64_t>(doubles - 2, 0), 16) * 16 + 2; }

// Where the matrices between the products lie in the workspace: bytes of a matrix each.
struct Layout {
  int64_t m, n;                                  // the shorter side and the longer one
  int64_t x, turned, square, partial, matrix;   // matrix: of all that belongs to one
  int64_t row_words, column_words;               // of floats: words of an array with one to each row (three of these), or column (four), of the shorter side
  int64_t ldx, ld_square;                        // of doubles
  Layout(int64_t rows, int64_t columns, int dtype) : m(std::min(rows, columns)), n(std::max(rows, columns)) {
    if (dtype == CT_F32) {
      x = aligned(m * ceil_div(n, kPairRun) * kPairRunBytes);
      turned = aligned(n * ceil_div(m, kPairRun) * kPairRunBytes);
      square = aligned(m * ceil_div(m, kPairRun) * kPairRunBytes);
    } else {
      ldx = spread_rows(columns);
      ld_square = spread_rows(m);
      x = turned = aligned(rows * ldx * 8);
      square = aligned(m * ld_square * 8);
    }
    partial = (dtype == CT_F32 ? 1 : 3) * kParts * 8;
    row_words = ceil_div(m, 64) * 64;
    column_words = ceil_div(n, 64) * 64;
    matrix = (dtype == CT_F32 ? x + 3 * row_words * 4 + 4 * column_words * 4 : 0) + 2 * turned + 2 * square + partial;
    if (dtype == CT_F32 && m <= kMostFew) matrix = std::max(matrix, aligned(few_bytes(m, n)));
  }
};

// Matrices beyond this many cells take turns: by then each launch fills the chip.
constexpr int64_t kCellsAtOnce = int64_t(1) << 26;

// Of a symmetric product the tiles at and below the diagonal.
int64_t tiles_of(int64_t count, int64_t m, int64_t n, int64_t height, int64_t width, bool symmetric) {
  const int64_t mt = ceil_div(m, height), nt = ceil_div(n, width);
  if (!symmetric) return count * mt * nt;
  if (height == width) return count * (mt * (mt + 1) / 2);
  const int64_t q = mt / 3, r = mt % 3;   // as place_of_unit counts them
  return count * (6 * q * q + 3 * q + (r == 0 ? 0 : r == 1 ? 4 * q + 2 : 8 * q + 5));
}
int64_t tiles_of(int64_t count, int64_t m, int64_t n, int64_t side, bool symmetric) { return tiles_of(count, m, n, side, side, symmetric); }

TileOrder order_of(int64_t count, int64_t m, int64_t n, int64_t height, int64_t width, bool symmetric) {
  TileOrder o;
  const int64_t tiles = tiles_of(1, m, n, height, width, symmetric), nt = ceil_div(n, width);
  o.m_tiles = (uint32_t)ceil_div(m, height);
  o.n_tiles = (uint32_t)nt;
  o.tiles = (uint32_t)tiles;
  o.units = (uint32_t)(count * tiles);
  o.tiles_fd = FastDiv(o.tiles);
  o.band_fd = FastDiv((uint32_t)(kBand * nt));
  o.band = o.units <= 24 * kXcds ? kBand / 2 : kBand;
  return o;
}
TileOrder order_of(int64_t count, int64_t m, int64_t n, int64_t side, bool symmetric) { return order_of(count, m, n, side, side, symmetric); }

dim3 grid_of(const TileOrder& o) { return dim3((uint32_t)(ceil_div(o.units, kXcds) * kXcds)); }

constexpr int64_t kUnits = 256;

// Microseconds of `tiles` tiles over `runs` runs of 32 k.  Small tiles are bound by what the L2 caches give, or one to a unit by latency; of
// 128 a side two blocks share a unit; large ones are bound by the matrix cores, whose clock is higher while some of them rest.  Us of 32,
// 64, 128 and 256 a side: X X^T of 128 x 784 7.6, 10, 26, 46; 512 x 512 5.8, 9.0; 1024 x 1024 16, 12, 32, 76; 2048 x 2048 73, 48, 58, 126;
// sixteen of 1024 x 2816 500, 229, 207, 199; 4096 x 8192 1090, 559, 546, 471; B X of 1024 x 1024 21, 14, 33, 77; of the others from 2048 on 129,
// 71, 64, 130; 814, 436, 331, 296; 2139, 1018, 780, 651.  Within 15 % of most of the 150 times of which these are a part.
double time_of_32(int64_t tiles, int64_t runs, bool symmetric) {
  return 3.0 + ((symmetric ? 0.5 : 1.2) + 0.144 * (double)runs) * (double)ceil_div(tiles, kUnits);
}
double time_of_64(int64_t tiles, int64_t runs) {
  return 5.0 + (double)runs * (tiles <= kUnits ? 0.23 : std::max(0.44, 0.285 * (double)tiles / kUnits));
}
double time_of_128(int64_t tiles, int64_t runs) {
  const int64_t full = tiles / (2 * kUnits), rest = tiles % (2 * kUnits);
  return 7.0 * (double)(full + (rest > 0)) + (double)runs * (1.5 * (double)full + (rest == 0 ? 0.0 : rest <= kUnits ? 0.8 : 1.45));
}
double time_of_256(int64_t tiles, int64_t runs) {
  const int64_t full = tiles / kUnits, rest = tiles % kUnits;
  return 14.0 * (double)(full + (rest > 0)) + (double)runs * (2.5 * (double)full + (rest > 0 ? 1.75 + 0.75 * (double)rest / kUnits : 0.0));
}
// 256 by 192, of symmetric products: in whole calls X X^T of 4096 x 8192, 187 tiles, takes 480 us (136 of 256 a side 527), of sixteen 1024 x 2816,
// 240 tiles, 200 (160, 223); a call of 4096 x 4096 4086 (of 128 and 256 a side 4612, 4475).
double time_of_tall(int64_t tiles, int64_t runs) {
  const int64_t full = tiles / kUnits, rest = tiles % kUnits;
  return 12.0 * (double)(full + (rest > 0)) + (double)runs * (1.95 * (double)full + (rest > 0 ? 1.05 + 0.95 * (double)rest / kUnits : 0.0));
}

double time_of_gram(int64_t count, int64_t m, int64_t runs) {
  auto tiles = [&](int64_t side) { return tiles_of(count, m, m, side, true); };
  return std::min({time_of_32(tiles(kSmallSide), runs, true), time_of_64(tiles(64), runs), time_of_128(tiles(128), runs),
                   time_of_tall(tiles_of(count, m, m, 256, 192, true), runs), time_of_256(tiles(256), runs)});
}
// With parts of k and the launch that joins them.
double time_of_parts(int64_t count, int64_t m, int64_t runs, int64_t parts) {
  return time_of_32(tiles_of(count, m, m, kSmallSide, true) * parts, ceil_div(runs, parts), true) + 5.0;
}

template <class Tile, Product kProduct>
void launch_tile(hipStream_t s, PairArgs a, int64_t count) {
  a.order = order_of(count, a.m, a.n, Tile::SM, Tile::SN, is_symmetric(kProduct));
  hipLaunchKernelGGL((pair_kernel<Tile, kProduct>), grid_of(a.order), dim3(Tile::T), 0, s, a);
}

template <Product kProduct>
void launch_small(hipStream_t s, PairArgs a, int64_t count) {
  a.order = order_of(count, a.m, a.n, kSmallSide, is_symmetric(kProduct));
  if (a.runs <= 4) hipLaunchKernelGGL((pair_small_kernel<4, kProduct>), grid_of(a.order), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((pair_small_kernel<8, kProduct>), grid_of(a.order), dim3(512), 0, s, a);
}

// How many parts the k of X X^T is divided into, in the room of a matrix's `bytes`: blocks for half the chip, a run to a wave at least.
int64_t gram_parts(int64_t count, int64_t m, int64_t runs, int64_t bytes) {
  const int64_t tiles = tiles_of(1, m, m, kSmallSide, true);
  return std::min({2 * kUnits / (count * tiles), ceil_div(runs, kPartWaves), bytes / (tiles * (int64_t)kSmallCells * 4)});
}

// `room`: of a matrix, the others' are room_bytes apart.
void launch_gram_parts(hipStream_t s, PairArgs a, int64_t count, int64_t parts, void* room, int64_t room_bytes) {
  a.order = order_of(count, a.m, a.n, kSmallSide, true);
  const uint32_t part_runs = (uint32_t)ceil_div(a.runs, parts);
  parts = ceil_div(a.runs, part_runs);
  float* const sums = static_cast<float*>(room);
  hipLaunchKernelGGL(gram_part_kernel, dim3((uint32_t)(a.order.units * parts)), dim3(64 * kPartWaves), 0, s, a, part_runs, FastDiv((uint32_t)parts), sums, room_bytes / 4);
  hipLaunchKernelGGL(gram_join_kernel, dim3(a.order.units), dim3(256), 0, s, a, (uint32_t)parts, sums, room_bytes / 4);
}

// The side of the tiles taken.
template <Product kProduct>
const char* launch_pair(hipStream_t s, const PairArgs& a, int64_t count) {
  auto tiles = [&](int64_t side) { return tiles_of(count, a.m, a.n, side, is_symmetric(kProduct)); };
  const double small = time_of_64(tiles(64), a.runs), medium = time_of_128(tiles(128), a.runs), large = time_of_256(tiles(256), a.runs);
  if constexpr (is_symmetric(kProduct)) {
    const double tall = time_of_tall(tiles_of(count, a.m, a.n, 256, 192, true), a.runs);
    if (tall < std::min({time_of_32(tiles(kSmallSide), a.runs, true), small, medium, large})) return launch_tile<TileTall, kProduct>(s, a, count), "256x192";
  }
  if (time_of_32(tiles(kSmallSide), a.runs, is_symmetric(kProduct)) <= std::min({small, medium, large})) return launch_small<kProduct>(s, a, count), "32";
  if (small <= medium && small <= large) return launch_tile<Tile64, kProduct>(s, a, count), "64";
  if (medium <= large) return launch_tile<Tile128, kProduct>(s, a, count), "128";
  return launch_tile<Tile256, kProduct>(s, a, count), "256";
}

// Microseconds of `tiles` tiles over `depth` k, of 64 a side by way of LDS and of 32 straight from memory.  Us of both: X X^T of 301 x 517 29
// and 12, of five of them 30 and 16, of 1024 x 1024 53 and 37, 2000 x 2000 234 and 197, four of 1024 x 2048 239 and 202; B X of the same
// 20 and 8, 22 and 19, 58 and 52, 312 and 359, 321 and 351.  (Tiles of 32 by way of LDS: X X^T of five 301 x 517 19, B X 22.)
double time_of_double(int64_t tiles, int64_t depth) { return 5.0 + (double)depth * (0.012 + 0.036 * (double)ceil_div(tiles, kUnits)); }
double time_of_direct(int64_t tiles, int64_t depth) { return 5.0 + (double)depth * 0.0117 * (double)ceil_div(tiles, kUnits); }

template <Product kProduct>
void launch_double(hipStream_t s, DoubleArgs a, int64_t count, bool tall) {
  constexpr bool kSymmetric = is_symmetric(kProduct);
  const int64_t large = tiles_of(count, a.m, a.n, kDoubleSide, kSymmetric), small = tiles_of(count, a.m, a.n, kDirectSide, kSymmetric);
  if (time_of_direct(small, a.depth) <= time_of_double(large, a.depth)) {
    a.order = order_of(count, a.m, a.n, kDirectSide, kSymmetric);
    const dim3 grid = grid_of(a.order), block(64 * kDirectWaves);
    if (tall) hipLaunchKernelGGL((ortho_direct_kernel<kProduct, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((ortho_direct_kernel<kProduct, false>), grid, block, 0, s, a);
  } else {
    a.order = order_of(count, a.m, a.n, kDoubleSide, kSymmetric);
    const dim3 grid = grid_of(a.order);
    if (tall) hipLaunchKernelGGL((ortho_double_kernel<kProduct, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((ortho_double_kernel<kProduct, false>), grid, dim3(256), 0, s, a);
  }
}

// X X^T, in parts of k where there are few tiles: a block for each unit, 32 parts at most (the launch that joins them waits for each eight),
// 64 k at least, in the room of a matrix's `bytes`.
void launch_double_gram(hipStream_t s, DoubleArgs a, int64_t count, bool tall, void* room, int64_t bytes) {
  const int64_t tiles = tiles_of(1, a.m, a.n, kDirectSide, true);
  const int64_t most = std::min({kUnits / (count * tiles), ceil_div(a.depth, 64), bytes / (tiles * kDirectSide * kDirectSide * 8), (int64_t)32});
  const int64_t part_depth = most > 1 ? ceil_div(ceil_div(a.depth, most), kDirectRun) * kDirectRun : a.depth, parts = ceil_div(a.depth, part_depth);
  if (parts == 1 || time_of_direct(count * tiles * parts, part_depth) + 5.0 + 0.1 * (double)parts >= time_of_direct(count * tiles, a.depth))
    return launch_double<kGram>(s, a, count, tall);
  a.order = order_of(count, a.m, a.n, kDirectSide, true);
  const dim3 grid((uint32_t)(a.order.units * parts)), block(64 * kDirectWaves);
  double* const sums = static_cast<double*>(room);
  if (tall) hipLaunchKernelGGL((direct_part_kernel<true>), grid, block, 0, s, a, (uint32_t)part_depth, FastDiv((uint32_t)parts), sums, bytes / 8);
  else hipLaunchKernelGGL((direct_part_kernel<false>), grid, block, 0, s, a, (uint32_t)part_depth, FastDiv((uint32_t)parts), sums, bytes / 8);
  hipLaunchKernelGGL(direct_join_kernel, dim3(a.order.units), block, 0, s, a, (uint32_t)parts, sums, bytes / 8);
}

// The largest |a + b s + c s^2| for s of 0 to `most`, and the largest |v (a + b v^2 + c v^4)| for v of 0 to the root of it.
double most_of_factor(double a, double b, double c, double most) {
  double found = std::max(std::abs(a), std::abs(a + (b + c * most) * most));
  const double turn = c != 0 ? -b / (2 * c) : -1.0;
  if (turn > 0 && turn < most) found = std::max(found, std::abs(a + (b + c * turn) * turn));
  return found;
}
double most_of_step(double a, double b, double c, double most) {
  auto value = [&](double s) { return std::abs(std::sqrt(s) * (a + (b + c * s) * s)); };
  double found = value(most);
  // a + 3 b s + 5 c s^2 = 0
  const double root = 9 * b * b - 20 * a * c;
  if (c == 0) {
    const double s = b != 0 ? -a / (3 * b) : -1.0;
    if (s > 0 && s < most) found = std::max(found, value(s));
  } else if (root >= 0) {
    for (double sign : {-1.0, 1.0}) {
      const double s = (-3 * b + sign * std::sqrt(root)) / (10 * c);
      if (s > 0 && s < most) found = std::max(found, value(s));
    }
  }
  return found;
}

// k with 1.02 bound, for what rounding adds, at most 2^k.
int exponent_of(double bound) {
  int exponent;
  std::frexp(std::max(1.02 * bound, 0x1p-900), &exponent);
  return exponent;
}

// A row's exponent falls by that of the largest |a + b s^2 + c s^4| less this in a step at most.
constexpr int kMostFall = 6;

// What a step of floats needs to know of its coefficients, for singular values up to `most`.
struct StepBounds {
  double next, factor;   // of the singular values after it, and the largest |a + b s^2 + c s^4|
  int factor_exponent, m_exponent, growth;
  StepBounds(double a, double b, double c, double most, int64_t m) {
    const double squares = most * most;
    factor = most_of_factor(a, b, c, squares);
    next = most_of_step(a, b, c, squares);
    factor_exponent = exponent_of(factor);
    // b G + c G D D G is Y (b I + c X^T X) Y^T, and D is at most `largest`
    const double inner = std::max(std::abs(b), std::abs(b + c * squares)), largest = std::ldexp(1.0, exponent_of(most));
    m_exponent = exponent_of(std::abs(a) + largest * largest * inner);
    // A row of M times a column of Y, against the column's largest, as the row's exponent falls: |a|; and the root of the sum of the squares of D, at most
    // root(m) * largest, times that of (the rest of M's row) / D, which is a row of Y times (b I + c X^T X) X^T
    const double fall = std::ldexp(1.0, kMostFall - factor_exponent);
    const double of_norm = factor > 0 ? std::max(1.0 / factor, next > 0 ? most / next : 0.0) : 0.0;   // |y| as it falls: |x| / |x'|'s bound
    growth = std::max(0, exponent_of(std::abs(a) * fall + std::sqrt((double)m) * largest * most * inner * std::min(fall, of_norm)));
  }
};

struct Request {
  StartArgs start;
  void* out;
  int64_t ldo, out_stride;
  double alpha, beta;
  const double* coefficients;
  int steps;
  int64_t count, rows, columns;
  void* workspace;
  int64_t workspace_bytes;
  int dtype;
};

constexpr double kMostValue = 0x1p40;
// Of floats before the last step: M has the squares of these values, times what b and c are to a, and is made of floats.
constexpr double kMostFloat = 0x1p30;

// The norm, the exponents of rows and columns, and Y in pieces.  Strips over the longer side are as many as fill the chip, kMostStrips at most; those over the
// shorter one as long as leaves four blocks to a unit, for each block adds up its rows' squares first (sixteen of 2816 x 1024: 112 us, with eight blocks
// 132, with 32 153).
void launch_start(hipStream_t s, const StartArgs& a, Exponents e, uint32_t count, bool tall, char* by_rows, char* by_columns, int64_t stride_rows,
                  int64_t stride_columns) {
  const int64_t of_rows = ceil_div(a.rows, 64), of_columns = ceil_div(a.columns, 64), shorter = tall ? of_columns : of_rows, longer = tall ? of_rows : of_columns;
  const int64_t most = std::min<int64_t>({kMostStrips, kParts / shorter, std::max<int64_t>(1, 8 * kUnits / (count * shorter))}), tiles = ceil_div(longer, std::min(most, longer));
  e.strips = (uint32_t)ceil_div(longer, tiles);
  const uint32_t parts = (uint32_t)(e.strips * shorter);
  const int64_t across = std::min<int64_t>({std::max<int64_t>(1, count * shorter * longer / (4 * kUnits)), shorter, kMostAcross});
  const dim3 over_longer(e.strips, (uint32_t)shorter, count), over_shorter((uint32_t)ceil_div(shorter, across), (uint32_t)longer, count);
  const dim3 all((uint32_t)of_columns, (uint32_t)of_rows, count);
  auto launch = [&](auto is_tall) {
    constexpr bool kTall = decltype(is_tall)::value;
    hipLaunchKernelGGL((start_scan_kernel<kTall>), over_longer, dim3(256), 0, s, a, (uint32_t)tiles, e);
    hipLaunchKernelGGL((start_columns_kernel<kTall>), over_shorter, dim3(256), 0, s, a, (uint32_t)across, e);
    hipLaunchKernelGGL((start_pieces_kernel<kTall>), all, dim3(256), 0, s, a, parts, e, by_rows, by_columns, stride_rows, stride_columns);
  };
  if (tall) launch(std::true_type{});
  else launch(std::false_type{});
}

int run_float(hipStream_t s, const Request& r, const Layout& l, int64_t at_once) {
  const bool tall = r.rows > r.columns;
  char* const base = static_cast<char*>(r.workspace);
  char* const x = base;
  char* turned[2] = {x + at_once * l.x, x + at_once * (l.x + l.turned)};
  char* const square = turned[1] + at_once * l.turned;
  char* const factor = square + at_once * l.square;
  double* const partial = reinterpret_cast<double*>(factor + at_once * l.square);
  int* const words = reinterpret_cast<int*>(partial + at_once * kParts);
  int* of_rows[2] = {words, words + at_once * l.row_words};
  int* of_columns[2] = {words + at_once * 2 * l.row_words, words + at_once * (2 * l.row_words + l.column_words)};
  uint32_t* const recorded = reinterpret_cast<uint32_t*>(of_columns[1] + at_once * l.column_words);
  const int64_t gram_bytes = aligned(l.m * l.m * 4);
  const char *of_gram = "", *of_square = "", *of_update = "", *of_last = "";
  for (int64_t first = 0; first < r.count; first += at_once) {
    const int64_t count = std::min(at_once, r.count - first);
    uint32_t *const of_squares = recorded, *most_of[2] = {recorded + at_once * l.row_words, recorded + at_once * (l.row_words + l.column_words)};
    StartArgs start = r.start;
    start.move(first * start.stride * 4);
    start.partial = partial;
    // the sums of the input's rows are where Y by columns is next
    const Exponents exponents{of_rows[0], of_columns[0], of_rows[1], reinterpret_cast<double*>(turned[1]), most_of[0], l.turned / 8, (uint32_t)l.row_words,
                              (uint32_t)l.column_words, 0};
    launch_start(s, start, exponents, (uint32_t)count, tall, tall ? turned[0] : x, tall ? x : turned[0], tall ? l.turned : l.x, tall ? l.x : l.turned);
    double most = 1.0;
    for (int step = 0; step < r.steps; ++step) {
      const double* k = r.coefficients + 3 * step;
      const StepBounds bounds(k[0], k[1], k[2], most, l.m);
      const int now = step & 1, next = now ^ 1, most_exponent = exponent_of(most);
      const bool last = step + 1 == r.steps;
      PairArgs g{};
      g.left = g.right = x;
      g.left_stride = g.right_stride = l.x;
      g.m = g.n = (uint32_t)l.m;
      g.runs = (uint32_t)ceil_div(l.n, kPairRun);
      g.shift = -2 * kPairTop;
      g.by_rows = square;
      g.rows_stride = l.square;
      g.store = kPairTop - most_exponent;
      g.row_exponents = g.column_exponents = of_rows[now];
      g.row_exponents_stride = g.column_exponents_stride = (uint32_t)l.row_words;
      // Y by columns lies in one of two places; the other has room for G, and behind it for sums of parts of k
      g.gram = reinterpret_cast<float*>(turned[next]);
      g.gram_stride = l.turned / 4;
      g.squares = of_squares;
      const int64_t parts = gram_parts(count, l.m, g.runs, l.turned - gram_bytes);
      if (parts > 1 && time_of_parts(count, l.m, g.runs, parts) < time_of_gram(count, l.m, g.runs)) {
        launch_gram_parts(s, g, count, parts, turned[next] + gram_bytes, l.turned);
        of_gram = "parts";
      } else {
        of_gram = launch_pair<kGram>(s, g, count);
      }
      g.left = g.right = square;
      g.left_stride = g.right_stride = l.square;
      g.runs = (uint32_t)ceil_div(l.m, kPairRun);
      g.shift = 2 * (most_exponent - kPairTop);
      g.by_rows = factor;
      g.store = kPairTop - bounds.m_exponent;
      g.a = (float)k[0];
      g.b = (float)k[1];
      g.c = (float)k[2];
      g.next_most = most_of[next];
      g.clear = last ? 0 : (uint32_t)(count * l.column_words);
      of_square = launch_pair<kSquare>(s, g, count);
      PairArgs u{};
      u.left = factor;
      u.left_stride = l.square;
      u.right = turned[now];
      u.right_stride = l.turned;
      u.m = (uint32_t)l.m;
      u.n = (uint32_t)l.n;
      u.runs = (uint32_t)ceil_div(l.m, kPairRun);
      u.row_exponents = of_rows[now];
      u.row_exponents_stride = (uint32_t)l.row_words;
      u.column_exponents = of_columns[now];
      u.column_exponents_stride = (uint32_t)l.column_words;
      if (!last) {
        u.shift = bounds.m_exponent - kPairTop;
        u.by_rows = x;
        u.rows_stride = l.x;
        u.by_columns = turned[next];
        u.columns_stride = l.turned;
        u.squares = of_squares;
        u.next_rows = of_rows[next];
        u.next_columns = of_columns[next];
        u.most = most_of[now];
        u.next_most = most_of[next];
        u.most_factor = (float)(1.02 * bounds.factor);
        u.most_next = exponent_of(bounds.next);
        u.least_change = bounds.factor_exponent - kMostFall;
        u.growth = bounds.growth;
        of_update = launch_pair<kUpdate>(s, u, count);
      } else {
        u.shift = bounds.m_exponent - 2 * kPairTop;
        if (tall) {   // the rows of the result are those of X^T
          std::swap(u.left, u.right);
          std::swap(u.left_stride, u.right_stride);
          std::swap(u.row_exponents, u.column_exponents);
          std::swap(u.row_exponents_stride, u.column_exponents_stride);
          std::swap(u.m, u.n);
        }
        u.out = static_cast<float*>(r.out) + first * r.out_stride;
        u.ldo = r.ldo;
        u.out_stride = r.out_stride;
        u.alpha = (float)r.alpha;
        u.beta = (float)r.beta;
        of_last = launch_pair<kLast>(s, u, count);
      }
      most = bounds.next;
    }
  }
  thread_local char name[96];   // the tiles of each product, of the last matrices
  std::snprintf(name, sizeof name, "orthogonalize_pair gram %s square %s update %s result %s", of_gram, of_square, of_update, of_last);
  note_kernel(name);
  return after_launch(s);
}

int run_double(hipStream_t s, const Request& r, const Layout& l, int64_t at_once) {
  const bool tall = r.rows > r.columns;
  char* const base = static_cast<char*>(r.workspace);
  double* x[2] = {reinterpret_cast<double*>(base), reinterpret_cast<double*>(base + at_once * l.x)};
  double* const gram = reinterpret_cast<double*>(base + 2 * at_once * l.x);
  double* const factor = reinterpret_cast<double*>(base + 2 * at_once * l.x + at_once * l.square);
  double* const partial = reinterpret_cast<double*>(base + 2 * at_once * (l.x + l.square));
  const int64_t cells = r.rows * r.columns, parts = std::min<int64_t>(kParts, ceil_div(cells, 4096));
  const uint64_t each = (uint64_t)ceil_div(cells, parts);
  for (int64_t first = 0; first < r.count; first += at_once) {
    const int64_t count = std::min(at_once, r.count - first);
    StartArgs start = r.start;
    start.move(first * start.stride * 8);
    start.partial = partial;
    hipLaunchKernelGGL(start_norm_kernel, dim3((uint32_t)parts, (uint32_t)count), dim3(256), 0, s, start, (uint32_t)parts, each,
                       start.ld == r.columns);
    hipLaunchKernelGGL(start_double_kernel, dim3((uint32_t)std::min<int64_t>(ceil_div(cells, 256), 4096), (uint32_t)count), dim3(256), 0, s, start,
                       (uint32_t)parts, x[0], l.x / 8, (uint32_t)l.ldx, FastDiv((uint32_t)r.columns), (uint32_t)cells);
    for (int step = 0; step < r.steps; ++step) {
      const double* k = r.coefficients + 3 * step;
      DoubleArgs g{};
      g.x = x[step & 1];
      g.x_stride = l.x / 8;
      g.ldx = (uint32_t)l.ldx;
      g.ld_square = (uint32_t)l.ld_square;
      g.ldo = l.ld_square;
      g.square_stride = g.out_stride = l.square / 8;
      g.m = g.n = (uint32_t)l.m;
      g.out = gram;
      g.square = gram;
      g.depth = (uint32_t)l.n;
      launch_double_gram(s, g, count, tall, x[(step + 1) & 1], l.x);
      g.out = factor;
      g.depth = (uint32_t)l.m;
      g.a = k[0];
      g.b = k[1];
      g.c = k[2];
      launch_double<kSquare>(s, g, count, false);
      g.square = factor;
      g.m = (uint32_t)r.rows;
      g.n = (uint32_t)r.columns;
      if (step + 1 < r.steps) {
        g.out = x[(step + 1) & 1];
        g.out_stride = l.x / 8;
        g.ldo = l.ldx;
        launch_double<kUpdate>(s, g, count, tall);
      } else {
        g.out = static_cast<double*>(r.out) + first * r.out_stride;
        g.out_stride = r.out_stride;
        g.ldo = r.ldo;
        g.alpha = r.alpha;
        g.beta = r.beta;
        launch_double<kLast>(s, g, count, tall);
      }
    }
  }
  note_kernel("orthogonalize_double");
  return after_launch(s);
}

int check_extents(const char* name, int64_t count, int64_t rows, int64_t columns) {
  CT_REQUIRE(count >= 0 && rows >= 0 && columns >= 0, "%s: negative extent", name);
  CT_REQUIRE(rows <= kMostSide && columns <= kMostSide && count <= kMostCount, "%s: %lld matrices of %lld by %lld, at most %lld of %lld a side are taken",
             name, (long long)count, (long long)rows, (long long)columns, (long long)kMostCount, (long long)kMostSide);
  CT_REQUIRE(rows * columns < int64_t(1) << 31, "%s: a matrix of %lld by %lld, 2^31 - 1 elements are taken", name, (long long)rows, (long long)columns);
  return CT_OK;
}

// What both entry points check, and the products.
int run(const char* name, hipStream_t s, Request r) {
  const int64_t size = dtype_size(r.dtype);
  CT_REQUIRE(r.steps >= 1 && r.steps <= kMostSteps, "%s: %d steps, 1 to %d are taken", name, r.steps, kMostSteps);
  CT_REQUIRE(r.coefficients, "%s: null coefficients", name);
  CT_REQUIRE(r.start.epsilon >= 0, "%s: epsilon must not be negative", name);
  double bound = 1.0, before_last = 1.0, change = 1.0;   // of the largest singular value; of what X X^T is off by
  for (int step = 0; step < r.steps; ++step) {
    const double* k = r.coefficients + 3 * step;
    CT_REQUIRE(std::isfinite(k[0]) && std::isfinite(k[1]) && std::isfinite(k[2]), "%s: coefficients must be finite", name);
    before_last = std::max(before_last, bound);
    const double factor = most_of_factor(k[0], k[1], k[2], bound * bound);
    change *= std::max(1.0, factor * most_of_factor(k[0], 3 * k[1], 5 * k[2], bound * bound));   // (s (a + b s + c s^2)^2)' is that
    bound = most_of_step(k[0], k[1], k[2], bound * bound);
    CT_REQUIRE(factor <= kMostValue && bound <= kMostValue, "%s: with these coefficients singular values grow beyond 2^40", name);
  }
  CT_REQUIRE(r.dtype == CT_F64 || before_last <= kMostFloat, "%s: with these coefficients singular values grow beyond 2^30 before the last step", name);
  if (r.count == 0 || r.rows == 0 || r.columns == 0) return CT_OK;
  const Layout l(r.rows, r.columns, r.dtype);
  CT_REQUIRE(r.workspace && (reinterpret_cast<uintptr_t>(r.workspace) & 15) == 0, "%s: the workspace must be a buffer, aligned to 16 bytes", name);
  CT_REQUIRE(r.workspace_bytes >= l.matrix, "%s: a workspace of %lld bytes, a matrix takes %lld", name, (long long)r.workspace_bytes, (long long)l.matrix);
  // a launch of 2^32 lanes or more is refused, and a block has up to 512
  const int64_t most = (int64_t(1) << 22) / tiles_of(1, r.rows, r.columns, 32, false);
  const int64_t at_once = std::min({r.count, r.workspace_bytes / l.matrix, std::max<int64_t>(1, most)});
  const Run work{r.workspace, r.workspace_bytes};
  auto run_of = [&](const void* p, int64_t ld, int64_t stride) { return Run{p, ((r.count - 1) * stride + (r.rows - 1) * ld + r.columns) * size}; };
  const Run x = run_of(r.start.x, r.start.ld, r.start.stride), gradient = run_of(r.start.gradient, r.start.ld, r.start.stride);
  const Run out = run_of(r.out, r.ldo, r.out_stride);
  CT_REQUIRE(!runs_meet(work, x) && !runs_meet(work, gradient) && !runs_meet(work, out), "%s: the workspace overlaps an operand", name);
  if (r.dtype == CT_F64) return run_double(s, r, l, at_once);
  if (l.m > kMostFew || change > kMostFewChange) return run_float(s, r, l, at_once);
  FewMatrices few{r.start, static_cast<char*>(r.workspace), l.matrix, static_cast<float*>(r.out), r.ldo, r.out_stride, (float)r.alpha, (float)r.beta, r.coefficients,
                  r.steps};
  for (int64_t first = 0; first < r.count; first += at_once) {
    ortho_few(s, few, std::min(at_once, r.count - first));
    few.start.move(at_once * few.start.stride * 4);
    few.out += at_once * few.out_stride;
  }
  note_kernel("orthogonalize_few");
  return after_launch(s);
}

}  // namespace

#define CT_ORTHO_FLOATING(name) CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, name ": datatype must be float or double")

extern "C" {

int ct_orthogonalize_workspace(int64_t count, int64_t rows, int64_t columns, int dtype, int64_t* bytes) {
  CT_ORTHO_FLOATING("ct_orthogonalize_workspace");
  CT_REQUIRE(bytes, "ct_orthogonalize_workspace: null result");
  CT_REQUIRE(count >= 0 && rows >= 0 && columns >= 0 && rows <= kMostSide && columns <= kMostSide && rows * columns < int64_t(1) << 31,
             "ct_orthogonalize_workspace: bad extent");
  *bytes = 0;
  if (count == 0 || rows == 0 || columns == 0) return CT_OK;
  *bytes = std::min(count, std::max<int64_t>(1, kCellsAtOnce / (rows * columns))) * Layout(rows, columns, dtype).matrix;
  return CT_OK;
}

int ct_orthogonalize(void* stream, void* output, int64_t output_colstride, int64_t output_stride, double alpha, const void* input,
                     int64_t input_colstride, int64_t input_stride, double beta, int64_t count, int64_t rows, int64_t columns,
                     const double* coefficients, int steps, double epsilon, void* workspace, int64_t workspace_bytes, int dtype) {
  CT_ORTHO_FLOATING("ct_orthogonalize");
  if (int rc = check_extents("ct_orthogonalize", count, rows, columns)) return rc;
  if (count > 0 && rows > 0 && columns > 0) {
    CT_REQUIRE(output && input, "ct_orthogonalize: null buffer");
    CT_REQUIRE(output_colstride >= columns && input_colstride >= columns, "ct_orthogonalize: a column stride below the row's length");
    CT_REQUIRE(std::max({output_colstride, input_colstride, output_stride, input_stride}) <= kMostStride, "ct_orthogonalize: a stride beyond 2^40");
    CT_REQUIRE(count == 1 || input_stride >= 0, "ct_orthogonalize: negative stride of matrices");
    CT_REQUIRE(count == 1 || output_stride >= (rows - 1) * output_colstride + columns, "ct_orthogonalize: results overlap one another");
    const int64_t size = dtype_size(dtype);
    const bool in_place = output == input && output_colstride == input_colstride && (count == 1 || output_stride == input_stride);
    CT_REQUIRE(in_place || !runs_meet({output, ((count - 1) * output_stride + (rows - 1) * output_colstride + columns) * size},
                                      {input, ((count - 1) * input_stride + (rows - 1) * input_colstride + columns) * size}),
               "ct_orthogonalize: output overlaps the input");
  }
  Request r{};
  r.start.x = input;
  r.start.ld = input_colstride;
  r.start.stride = count > 1 ? input_stride : 0;
  r.start.rows = (uint32_t)rows;
  r.start.columns = (uint32_t)columns;
  r.start.epsilon = epsilon;
  r.out = output;
  r.ldo = output_colstride;
  r.out_stride = count > 1 ? output_stride : 0;
  r.alpha = alpha;
  r.beta = beta;
  r.coefficients = coefficients;
  r.steps = steps;
  r.count = count;
  r.rows = rows;
  r.columns = columns;
  r.workspace = workspace;
  r.workspace_bytes = workspace_bytes;
  r.dtype = dtype;
  return run("ct_orthogonalize", static_cast<hipStream_t>(stream), r);
}

int ct_muon_step(void* stream, int dtype, double alpha, double momentum, int nesterov, double weight_decay, double gradient_alpha,
                 const double* coefficients, int steps, double epsilon, const void* gradient, void* parameters, void* momentum_vals,
                 int64_t count, int64_t rows, int64_t columns, void* workspace, int64_t workspace_bytes) {
  CT_ORTHO_FLOATING("ct_muon_step");
  if (int rc = check_extents("ct_muon_step", count, rows, columns)) return rc;
  if (count > 0 && rows > 0 && columns > 0) {
    CT_REQUIRE(gradient && parameters && momentum_vals, "ct_muon_step: null buffer");
    const int64_t bytes = count * rows * columns * dtype_size(dtype);
    CT_REQUIRE(!runs_meet({gradient, bytes}, {parameters, bytes}) && !runs_meet({gradient, bytes}, {momentum_vals, bytes}) &&
                   !runs_meet({parameters, bytes}, {momentum_vals, bytes}),
               "ct_muon_step: the gradient, the parameters and the momentum overlap");
  }
  Request r{};
  r.start.x = momentum_vals;
  r.start.gradient = gradient;
  r.start.momentum = momentum_vals;
  r.start.ld = columns;
  r.start.stride = rows * columns;
  r.start.rows = (uint32_t)rows;
  r.start.columns = (uint32_t)columns;
  r.start.gradient_alpha = gradient_alpha;
  r.start.decay = momentum;
  r.start.epsilon = epsilon;
  r.start.nesterov = nesterov != 0;
  r.out = parameters;
  r.ldo = columns;
  r.out_stride = rows * columns;
  r.alpha = columns > 0 ? -alpha * std::sqrt(std::max(1.0, (double)rows / (double)columns)) : 0.0;
  r.beta = 1.0 - alpha * weight_decay;
  r.coefficients = coefficients;
  r.steps = steps;
  r.count = count;
  r.rows = rows;
  r.columns = columns;
  r.workspace = workspace;
  r.workspace_bytes = workspace_bytes;
  r.dtype = dtype;
  return run("ct_muon_step", static_cast<hipStream_t>(stream), r);
}

}  // extern "C"
