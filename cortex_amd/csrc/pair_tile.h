// pair_tile.h -- products of matrices with bounded elements on the half-precision matrix cores, two pieces to a float.
//
// v_mfma_f32_32x32x16_f16 takes as long as its bfloat16 form, and a half has eleven significant bits in place of eight: of a
// float x, hi = x rounded to a half and lo = x - hi rounded to a half leave at most 2^-23 of the power of two below x, the last
// of the float's bits, and
//   a * b = hi hi + (hi lo + lo hi) + lo lo
// without its last term (at most 2^-22 of the product, 2^-24.6 in the root mean square, of either sign) is three products where
// three bfloat16 pieces take six.  What a half lacks is range, 2^-24 to 2^16, so this is for matrices whose elements have a known
// bound: they are multiplied by a power of two that takes the bound to 2^14 at most, and what is below the least half is then
// 2^-39 of the bound.  Sums are held in float.
//
// A matrix of pieces is stored in rows of runs of 32 k, 128 bytes to a run: the 32 leading pieces, then the 32 others.  Beyond its
// columns a row is zeros up to a whole run.
#pragma once

#include "common.h"

namespace cthip {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef float pair_f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t pair_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kPairRun = 32, kPairRunBytes = 128;
// 2^kPairTop is the most that a bound is taken to.
constexpr int kPairTop = 14;

__device__ __forceinline__ void split_pair(float x, _Float16* hi, _Float16* lo) {
  *hi = (_Float16)x;
  *lo = (_Float16)(x - (float)*hi);
}

// Of matrices without a known bound a row has a power of two of its own, which takes its largest element below 2^15, and the other
// pieces are 2^kPairApart times as large as they are, so that they are no denormals before the element is 2^-28 of its row's largest:
// what is below 2^-51 of that is zero.  Their products are summed apart.
constexpr int kPairApart = 11;
__device__ __forceinline__ void split_pair_apart(float x, _Float16* hi, _Float16* lo) {
  *hi = (_Float16)x;
  *lo = (_Float16)((x - (float)*hi) * (float)(1 << kPairApart));
}

constexpr int pair_tile_lds(int bm, int bn) { return 2 * (bm + bn) * kPairRunBytes; }

// Rows of two matrices of pieces, those beyond the last ones repeated: where they begin and how far apart rows are.
template <int BM, int BN, int T>
struct PairMatrices {
  static constexpr int UA = BM * 8 / T, U = UA + BN * 8 / T;
  const char *a, *b;
  uint32_t offset[U];
  __device__ __forceinline__ PairMatrices(const char* a, uint32_t last_a, const char* b, uint32_t last_b, uint32_t row_bytes, uint32_t tid) : a(a), b(b) {
#pragma unroll
    for (int i = 0; i < U; ++i) offset[i] = min(((i < UA ? i : i - UA) * T + tid) / 8, i < UA ? last_a : last_b) * row_bytes + tid % 8 * 16;
  }
  __device__ __forceinline__ pair_u32x4 load(int i, uint32_t run) const {
    return *reinterpret_cast<const pair_u32x4*>((i < UA ? a : b) + (int64_t)run * kPairRunBytes + offset[i]);
  }
};

// Rows that lie anywhere: `left(r)` and `right(r)` say where those of the tile begin.
template <int BM, int BN, int T>
struct PairRows {
  static constexpr int UA = BM * 8 / T, U = UA + BN * 8 / T;
  const char* row[U];
  template <class Left, class Right>
  __device__ __forceinline__ PairRows(Left left, Right right, uint32_t tid) {
#pragma unroll
    for (int i = 0; i < U; ++i) row[i] = (i < UA ? left((i * T + tid) / 8) : right(((i - UA) * T + tid) / 8)) + tid % 8 * 16;
  }
  __device__ __forceinline__ pair_u32x4 load(int i, uint32_t run) const {
    return *reinterpret_cast<const pair_u32x4*>(row[i] + (int64_t)run * kPairRunBytes);
  }
};

// The sums over all runs of k (at least one) of BM rows of the source's left matrix with BN rows of its right one, over WM x WN waves of 64 lanes:
// a lane's results of 32 x 32 cells, [.][.][.][r] row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32.  All of a block's waves call it.
// kApart: the products of the leading pieces in sum[0], those of one leading piece in sum[1]; else all of them in sum[0].
//
// Chunks of 16 bytes of a row are permuted by half the row's number, so that sixteen rows' reads of one chunk cover the banks once.  A
// fragment is read a product or two ahead of its use into the registers of the one that was used last, and a run's loads are kAhead runs
// ahead of their way into LDS.
template <int BM, int BN, int WM, int WN, int kAhead, bool kApart, class Source, int MT = BM / WM / 32, int NT = BN / WN / 32>
__device__ __forceinline__ void pair_tile(const Source& source, uint32_t runs, char* lds, uint32_t tid, pair_f32x16 (&sum)[kApart ? 2 : 1][MT][NT]) {
  constexpr int T = 64 * WM * WN, UA = Source::UA, U = Source::U, kBuffer = (BM + BN) * kPairRunBytes;
  static_assert(UA * T == BM * 8 && (U - UA) * T == BN * 8 && T % 128 == 0, "lanes share the tiles evenly");
  const uint32_t lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wave_m = wave / WN * (MT * 32), wave_n = wave % WN * (NT * 32), row = lane & 31, half = lane >> 5;
#pragma unroll
  for (int s = 0; s < (kApart ? 2 : 1); ++s)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[s][t][u][r] = 0.f;
  const uint32_t put = tid / 8 * kPairRunBytes + ((tid ^ tid / 16) & 7) * 16;
  pair_u32x4 raw[kAhead][U];
  auto load = [&](uint32_t run, int slot) {   // a run behind the last one is not used
#pragma unroll
    for (int i = 0; i < U; ++i) raw[slot][i] = source.load(i, min(run, runs - 1));
  };
  auto stage = [&](uint32_t buffer, int slot) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      *reinterpret_cast<pair_u32x4*>(lds + buffer * kBuffer + (i < UA ? 0 : BM * kPairRunBytes) + (i < UA ? i : i - UA) * (T / 8 * kPairRunBytes) + put) = raw[slot][i];
  };
  // [][0] leading pieces, [][1] others; a wave of one product has registers for both halves of a run
  constexpr bool kBoth = MT * NT == 1;
  f16x8 left[kBoth ? 2 : 1][2][MT], right[kBoth ? 2 : 1][2][NT];
  auto fetch_left = [&](uint32_t buffer, int part, int p) {
    const uint32_t chunk = p * 4 + part * 2 + half;
#pragma unroll
    for (int t = 0; t < MT; ++t)
      left[kBoth ? part : 0][p][t] = *reinterpret_cast<const f16x8*>(lds + buffer * kBuffer + (wave_m + t * 32 + row) * kPairRunBytes + ((chunk ^ row / 2) & 7) * 16);
  };
  auto fetch_right = [&](uint32_t buffer, int part, int p) {
    const uint32_t chunk = p * 4 + part * 2 + half;
#pragma unroll
    for (int u = 0; u < NT; ++u)
      right[kBoth ? part : 0][p][u] =
          *reinterpret_cast<const f16x8*>(lds + buffer * kBuffer + (BM + wave_n + u * 32 + row) * kPairRunBytes + ((chunk ^ row / 2) & 7) * 16);
  };
  auto multiply = [&](int part, int l, int r) {
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        pair_f32x16& to = sum[kApart ? l | r : 0][t][u];
        to = __builtin_amdgcn_mfma_f32_32x32x16_f16(left[kBoth ? part : 0][l][t], right[kBoth ? part : 0][r][u], to, 0, 0, 0);
      }
  };
  auto fetch = [&](uint32_t buffer, int part) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      fetch_left(buffer, part, p);
      fetch_right(buffer, part, p);
    }
  };
  auto multiply_all = [&](int part) {
    multiply(part, 1, 0);
    multiply(part, 0, 0);
    multiply(part, 0, 1);
  };
  // run 0 in LDS, runs 1 .. kAhead on their way
  load(0, 0);
  stage(0, 0);
#pragma unroll
  for (int i = 1; i <= kAhead; ++i) {
    load(i, i % kAhead);
    __builtin_amdgcn_sched_barrier(0);   // in the order in which they are waited for
  }
  __syncthreads();
  if constexpr (kBoth) {
    fetch(0, 0);
  } else {
    fetch_left(0, 0, 1);
    fetch_right(0, 0, 0);
  }
  auto step = [&](uint32_t run, uint32_t buffer, int slot) {
    if constexpr (kBoth) {
      fetch(buffer, 1);
      stage(buffer ^ 1, slot);
      load(run + 1 + kAhead, slot);
      multiply_all(0);
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
      fetch(buffer ^ 1, 0);
      multiply_all(1);
      __builtin_amdgcn_sched_barrier(0);
      return;
    }
    fetch_left(buffer, 0, 0);
    fetch_right(buffer, 0, 1);
    multiply(0, 1, 0);
    __builtin_amdgcn_sched_barrier(0);
    fetch_left(buffer, 1, 1);
    stage(buffer ^ 1, slot);
    multiply(0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    fetch_right(buffer, 1, 0);
    load(run + 1 + kAhead, slot);
    multiply(0, 0, 1);
    __builtin_amdgcn_sched_barrier(0);
    fetch_left(buffer, 1, 0);
    fetch_right(buffer, 1, 1);
    multiply(1, 1, 0);
    __builtin_amdgcn_sched_barrier(0);
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
    fetch_left(buffer ^ 1, 0, 1);
    multiply(1, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    fetch_right(buffer ^ 1, 0, 0);
    multiply(1, 0, 1);
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int kTurn = kAhead % 2 ? 2 * kAhead : kAhead;
  // Without a branch in the loop, behind which all loads would be waited for, those that are not needed yet too (1024 x 1024 in tiles of 64 15.9
  // us, and 13.9).  One run ahead there are no others, and the longer code costs large tiles 2 %.
  uint32_t run = 0;
  if constexpr (kAhead > 1) {
    for (; run + kTurn <= runs; run += kTurn) {
#pragma unroll
      for (int i = 0; i < kTurn; ++i) step(run + i, i & 1, (i + 1) % kAhead);
    }
  }
  for (; run < runs; run += kTurn) {
#pragma unroll
    for (int i = 0; i < kTurn; ++i)
      if (i == 0 || run + i < runs) step(run + i, i & 1, (i + 1) % kAhead);
  }
}

}  // namespace cthip
