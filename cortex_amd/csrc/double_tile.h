// double_tile.h -- a tile of a product of doubles on the matrix cores, of operands that lie by rows or by columns.
#pragma once

#include "common.h"

namespace cthip {

// A tile of S x S by four waves, S / 2 a side each, in products of 16 x 16 x 4: a wave's operands are 16 rows (or columns) by
// lane % 16 of k lane / 16, its results rows lane / 16 + 4 r.  BK k are staged in LDS at a time, the next two lots on their way
// into registers meanwhile.  An operand gives a lane four elements of a lot.  Its loads have no branches that lanes take apart:
// behind one, every load would be waited for before the next is used (30 us in place of 21, 2026 rows of 7 groups, 301 by 517).
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));
typedef f64x2 f64x2_at_8 __attribute__((aligned(8)));

constexpr int double_depth(int side) { return side == 64 ? 16 : 32; }

// Four k of a row, which is the same for all k; `end` k, at least one.
template <int S>
struct DoubleRow {
  static constexpr int BK = double_depth(S);
  static constexpr bool kByRow = true;
  const double* p;
  uint32_t end;
  bool present;
  static __device__ __forceinline__ uint32_t row() { return threadIdx.x / (BK / 4); }
  static __device__ __forceinline__ uint32_t k() { return threadIdx.x % (BK / 4) * 4; }
  __device__ __forceinline__ void load(uint32_t k0, f64x2 (&x)[2]) const {
    if (k0 + BK <= end) {
      x[0] = *reinterpret_cast<const f64x2_at_8*>(p + k0 + k());
      x[1] = *reinterpret_cast<const f64x2_at_8*>(p + k0 + k() + 2);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e / 2][e % 2] = p[min(k0 + k() + e, end - 1)];
    }
  }
  __device__ __forceinline__ void mend(uint32_t k0, f64x2 (&x)[2]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e / 2][e % 2] = present && k0 + k() + e < end ? x[e / 2][e % 2] : 0.0;
  }
};

// Four columns, from `column` on of `width`, of the rows that k goes over: row `first` + k, or the one that an index names there.
template <int S>
struct DoubleColumns {
  static constexpr int BK = double_depth(S);
  static constexpr bool kByRow = false;
  const double* p;
  int64_t ld;
  const int32_t* index;
  uint32_t first, end, rows;   // k below end, at least one; rows of p
  uint32_t left;               // columns from the tile's first on
  uint32_t next, absent;
  static __device__ __forceinline__ uint32_t column() { return threadIdx.x % (S / 4) * 4; }
  static __device__ __forceinline__ uint32_t k() { return threadIdx.x / (S / 4); }
  __device__ __forceinline__ DoubleColumns(const double* p, int64_t ld, const int32_t* index, uint32_t first, uint32_t end, uint32_t rows, uint32_t left)
      : p(p), ld(ld), index(index), first(first), end(end), rows(rows), left(left), absent(0) {
    look_up(0);
  }
  __device__ __forceinline__ void look_up(uint32_t k0) {
    const uint32_t row = first + min(k0 + k(), end - 1);
    next = index ? (uint32_t)index[row] : row;
  }
  __device__ __forceinline__ void load(uint32_t k0, f64x2 (&x)[2]) {
    const bool outside = next >= rows;
    absent = absent << 1 | outside;   // of this lot, and of the one before
    const double* row = p + (int64_t)(outside ? 0 : next) * ld;
    if (left >= S) {
      x[0] = *reinterpret_cast<const f64x2_at_8*>(row + column());
      x[1] = *reinterpret_cast<const f64x2_at_8*>(row + column() + 2);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e / 2][e % 2] = row[min(column() + e, left - 1)];
    }
    look_up(k0 + BK);
  }
  // after the load of the next lot
  __device__ __forceinline__ void mend(uint32_t k0, f64x2 (&x)[2]) const {
    const bool zero = (absent >> 1 & 1) || k0 + k() >= end;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e / 2][e % 2] = zero ? 0.0 : x[e / 2][e % 2];
  }
};

// Where an element of k lies in its row of S in LDS: half a wave's stores of one k of each of its rows, and its reads of 16
// rows of two k, fall on different banks each.  Runs of four stay together.
template <int S> __device__ __forceinline__ uint32_t double_at(uint32_t k, uint32_t row) {
  if constexpr (S == 32) return row ^ ((k >> 2 & 3) << 2 | ((k ^ k >> 4) & 1) << 4);
  else return row ^ ((k >> 2 & 1) << 3 | ((k ^ k >> 3) & 1) << 4);
}

template <int S, class Left, class Right, class Store>
__device__ __forceinline__ void double_tile(uint32_t depth, Left left, Right right, Store store) {
  constexpr int BK = double_depth(S), MT = S / 32;
  static_assert(S * BK / 4 == 256, "four elements of each operand to a lane");
  __shared__ __attribute__((aligned(16))) double lds_a[BK][S], lds_b[BK][S];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wave_m = wave / 2 * (S / 2), wave_n = wave % 2 * (S / 2);
  auto put_in = [&](auto& operand, double (&lds)[BK][S], uint32_t k0, f64x2 (&x)[2]) {
    using Operand = std::remove_reference_t<decltype(operand)>;
    operand.mend(k0, x);
    if constexpr (Operand::kByRow) {
#pragma unroll
      for (int e = 0; e < 4; ++e) lds[Operand::k() + e][double_at<S>(Operand::k() + e, Operand::row())] = x[e / 2][e % 2];
    } else {
      f64x2* to = reinterpret_cast<f64x2*>(&lds[Operand::k()][double_at<S>(Operand::k(), Operand::column())]);
      to[0] = x[0];
      to[1] = x[1];
    }
  };
  f64x4 sum[MT][MT] = {};
  f64x2 a[2][2], b[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    left.load(h * BK, a[h]);
    right.load(h * BK, b[h]);
  }
  auto step = [&](uint32_t k0, int h) {
    put_in(left, lds_a, k0, a[h]);
    put_in(right, lds_b, k0, b[h]);
    __syncthreads();
    left.load(k0 + 2 * BK, a[h]);
    right.load(k0 + 2 * BK, b[h]);
#pragma unroll
    for (int k = 0; k < BK; k += 4) {
      double l[MT], r[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        l[t] = lds_a[k + lane / 16][double_at<S>(k + lane / 16, wave_m + t * 16 + lane % 16)];
        r[t] = lds_b[k + lane / 16][double_at<S>(k + lane / 16, wave_n + t * 16 + lane % 16)];
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < MT; ++u) sum[t][u] = __builtin_amdgcn_mfma_f64_16x16x4f64(l[t], r[u], sum[t][u], 0, 0, 0);
    }
    __syncthreads();
  };
  for (uint32_t k0 = 0; k0 < depth; k0 += 2 * BK) {   // lots beyond the last one are zeros
    step(k0, 0);
    step(k0 + BK, 1);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) store(wave_m + t * 16 + lane / 16 + 4 * r, wave_n + u * 16 + lane % 16, sum[t][u][r]);
}

// Small products: a block owns 32 x 32, its W waves take every W-th run of 16 k each, straight from memory into the matrix cores'
// operands, the next run's loads on their way meanwhile, and leave their sums in LDS.  Nothing waits for another wave before that: five of
// 301 x 517 times their transposes 16 us, in tiles of 32 by way of LDS 19 (with eight waves 18.6).  A lane's four k of a run are
// lane / 16 * 4 and those behind it; sixteen lanes' rows, or columns, of t are t * 16 and those behind it.
constexpr uint32_t kDirectSide = 32, kDirectPitch = 33, kDirectRun = 16;

template <bool kByRow>
struct DoubleDirect {
  const double* p[2];   // a lane's row, from k 0 on, or its column
  int64_t ld;           // of columns
  bool present[2];
  // `row(i)`: which one is row i of the tile's, none if it is negative
  template <class Row>
  static __device__ __forceinline__ DoubleDirect rows(const double* p, int64_t ld, Row row) {
    DoubleDirect d;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t i = row(t * 16 + threadIdx.x % 16);
      d.present[t] = i >= 0;
      d.p[t] = p + (i < 0 ? 0 : i) * ld;
    }
    d.ld = ld;
    return d;
  }
  static __device__ __forceinline__ DoubleDirect columns(const double* p, int64_t ld, uint32_t left) {   // of `left` columns
    DoubleDirect d;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      d.present[t] = true;
      d.p[t] = p + min(t * 16 + threadIdx.x % 16, left - 1);
    }
    d.ld = ld;
    return d;
  }
  __device__ __forceinline__ void load(uint32_t k0, uint32_t end, double (&x)[2][4]) const {
    const uint32_t k = k0 + threadIdx.x % 64 / 16 * 4;
    if (kByRow && k0 + kDirectRun <= end) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (uint32_t e = 0; e < 4; e += 2) {
          const f64x2 two = *reinterpret_cast<const f64x2_at_8*>(p[t] + k + e);
          x[t][e] = two[0];
          x[t][e + 1] = two[1];
        }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) x[t][e] = p[t][min(k + e, end - 1) * (kByRow ? 1 : ld)];
    }
  }
  __device__ __forceinline__ void mend(uint32_t k0, uint32_t end, double (&x)[2][4]) const {
    const uint32_t k = k0 + threadIdx.x % 64 / 16 * 4;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) x[t][e] = present[t] && k + e < end ? x[t][e] : 0.0;
  }
};

// Of `depth` k, at least one.  The waves' sums are in `partial` afterwards, for all lanes to read.
template <int W, class Left, class Right>
__device__ __forceinline__ void double_direct(uint32_t depth, const Left& left, const Right& right, double (&partial)[W][kDirectSide * kDirectPitch]) {
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool all_present = __all(left.present[0] && left.present[1]);
  double x[2][2][4], y[2][2][4];   // of two runs
  f64x4 sum[2][2] = {};
  auto load = [&](uint32_t k0, int slot) {
    left.load(k0, depth, x[slot]);
    right.load(k0, depth, y[slot]);
  };
  auto multiply = [&](uint32_t k0, int slot) {
    if (k0 + kDirectRun > depth || !all_present) {
      asm volatile("");   // stays a branch
      left.mend(k0, depth, x[slot]);
      right.mend(k0, depth, y[slot]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 2; ++u) sum[t][u] = __builtin_amdgcn_mfma_f64_16x16x4f64(x[slot][t][e], y[slot][u][e], sum[t][u], 0, 0, 0);
  };
  constexpr uint32_t kStep = W * kDirectRun;
  uint32_t k0 = wave * kDirectRun;
  if (k0 < depth) {
    load(k0, 0);
    for (; k0 + 2 * kStep < depth; k0 += 2 * kStep) {   // no load behind a branch, which would be waited for at once
      load(k0 + kStep, 1);
      multiply(k0, 0);
      load(k0 + 2 * kStep, 0);
      multiply(k0 + kStep, 1);
    }
    if (k0 + kStep < depth) {
      load(k0 + kStep, 1);
      multiply(k0, 0);
      multiply(k0 + kStep, 1);
    } else {
      multiply(k0, 0);
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) partial[wave][(t * 16 + lane / 16 + 4 * r) * kDirectPitch + u * 16 + lane % 16] = sum[t][u][r];
  __syncthreads();
}

// The sum of cell (r, n), in the order of the waves.
template <int W>
__device__ __forceinline__ double direct_sum(const double (&partial)[W][kDirectSide * kDirectPitch], uint32_t r, uint32_t n) {
  double sum = partial[0][r * kDirectPitch + n];
#pragma unroll
  for (int w = 1; w < W; ++w) sum += partial[w][r * kDirectPitch + n];
  return sum;
}

}  // namespace cthip
