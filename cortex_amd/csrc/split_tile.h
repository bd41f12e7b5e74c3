// split_tile.h -- a tile of a float product on the bfloat16 matrix cores, three pieces to a float (split_mfma.h), of operands
// that a Source loads: a block's waves stage runs of eight k into LDS, split on the way, and multiply them.
#pragma once

#include "split_mfma.h"

namespace cthip {

// Element `chunk` (of eight k) of row `row` of a tile in LDS, rows of 32 k: the chunks of a row are permuted so that eight
// consecutive rows' reads of one chunk cover 128 bytes' worth of banks once.
__device__ __forceinline__ uint32_t tile_at(uint32_t row, uint32_t chunk) { return row * 32 + ((chunk ^ (row >> 1)) & 3) * 8; }

// Eight consecutive k of one row of an operand: kRowMajor has them side by side, else a leading dimension apart.  `base` is
// uniform and stays in scalar registers, `offset` is the lane's, in bytes.
template <bool kRowMajor>
__device__ __forceinline__ void load8(const float* base, uint32_t offset, int64_t ld, f32x4 (&to)[2]) {
  uint64_t bits = reinterpret_cast<uint64_t>(base);
  asm("" : "+s"(bits));   // or the loop keeps a 64-bit address per lane and load, for which there are no registers
  typedef __attribute__((address_space(1))) const char* Global;
  typedef f32x4 f32x4_at_4 __attribute__((aligned(4)));
  const Global p = reinterpret_cast<Global>(bits);
  if constexpr (kRowMajor) {
    to[0] = *reinterpret_cast<__attribute__((address_space(1))) const f32x4_at_4*>(p + offset);
    to[1] = *reinterpret_cast<__attribute__((address_space(1))) const f32x4_at_4*>(p + 16 + offset);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      to[e / 4][e % 4] = *reinterpret_cast<__attribute__((address_space(1))) const float*>(p + 4 * e * ld + offset);
  }
}

// Of tiles of BM x BN, in halfwords: two buffers of each operand's pieces.
constexpr int kTileDepth = 32;
constexpr int split_tile_lds(int bm, int bn) { return 2 * kSplitPieces * (bm + bn) * kTileDepth; }

// Where a block's T lanes load the operands of a tile: UA runs of eight k of the left one to each lane, then UB of the right.
template <int BM, int BN, int T, bool kA, bool kB>
struct TileShare {
  static constexpr int BK = kTileDepth, kChunks = BK / 8, UA = BM * kChunks / T, UB = BN * kChunks / T, U = UA + UB, kThreads = T;
  static_assert(UA * T == BM * kChunks && UB * T == BN * kChunks, "lanes share the tiles evenly");
  uint32_t tid;
  __device__ __forceinline__ uint32_t row_of(int i) const {
    return (i < UA ? kA : kB) ? ((i < UA ? i : i - UA) * T + tid) / kChunks : ((i < UA ? i : i - UA) * T + tid) % (i < UA ? BM : BN);
  }
  __device__ __forceinline__ uint32_t chunk_of(int i) const {
    return (i < UA ? kA : kB) ? ((i < UA ? i : i - UA) * T + tid) % kChunks : ((i < UA ? i : i - UA) * T + tid) / (i < UA ? BM : BN);
  }
};

// Two matrices; at least 32 k.  Rows beyond the last ones (of either tile) repeat them: their results are not for use.  The
// last tile of k, if it is a partial one, is loaded from 32 k before the end on; what an earlier tile had is set to zero, in
// both operands, before it is used.  Tiles beyond it are all zeros.
template <int BM, int BN, int T, bool kA, bool kB>
struct MatrixSource : TileShare<BM, BN, T, kA, kB> {
  using Share = TileShare<BM, BN, T, kA, kB>;
  using Share::BK;
  using Share::UA;
  using Share::U;
  const float *base_a, *base_b;
  int64_t lda, ldb;
  uint32_t k, first;
  uint32_t offset[U];
  __device__ __forceinline__ MatrixSource(const float* base_a, int64_t lda, const float* base_b, int64_t ldb, uint32_t last_a,
                                          uint32_t last_b, uint32_t k, uint32_t first, uint32_t tid)
      : Share{tid}, base_a(base_a), base_b(base_b), lda(lda), ldb(ldb), k(k), first(first) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const uint32_t r = min(this->row_of(i), i < UA ? last_a : last_b);
      const uint32_t ld = (uint32_t)(i < UA ? lda : ldb);
      offset[i] = 4 * ((i < UA ? kA : kB) ? r * ld + this->chunk_of(i) * 8 : this->chunk_of(i) * 8 * ld + r);
    }
  }
  __device__ __forceinline__ void rewind() {}
  __device__ __forceinline__ void load(int i, uint32_t tile, f32x4 (&to)[2]) const {
    const int64_t k0 = min((first + tile) * BK, k - BK);
    if (i < UA) load8<kA>(base_a + (kA ? k0 : k0 * lda), offset[i], lda, to);
    else load8<kB>(base_b + (kB ? k0 : k0 * ldb), offset[i], ldb, to);
  }
  __device__ __forceinline__ void drop(int i, uint32_t tile, f32x4 (&r)[2]) const {
    const uint32_t k0 = (first + tile) * BK;
    if (k0 + BK <= k) return;
    asm volatile("");   // stays a branch: as selects it would cost every tile
    const uint32_t repeated = k0 - (k - BK);   // of the tile's k; all of them beyond the last tile
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e / 4][e % 4] = this->chunk_of(i) * 8 + e < repeated ? 0.f : r[e / 4][e % 4];
  }
};

// A source's load(i, tile, to) is called with the tiles in their order for each i, beginning with 0 again after rewind();
// drop(i, tile, r) sets to zero what load left of that tile and is not of it, before the next load of that i.
//
// The sums of `tiles` tiles of k (an even number) of the source's tile of BM x BN over WM x WN waves: lane's results of
// 32 x 32 cells, [.][.][r] row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32.  All of a block's waves call it, each group
// of them with an LDS of its own.
template <int BM, int BN, int WM, int WN, class Source, int MT = BM / WM / 32, int NT = BN / WN / 32>
__device__ __forceinline__ void split_tile(Source& source, uint32_t tiles, uint16_t* lds, uint32_t tid,
                                           float (&result)[MT][NT][16]) {
  constexpr int BK = kTileDepth, UA = Source::UA, U = Source::U;
  constexpr int kLeft = 2 * kSplitPieces * BM * BK, kRight = 2 * kSplitPieces * BN * BK;
  const uint32_t lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  f32x16 sums[2][MT][NT];   // the products of the leading pieces; all others
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u) sums[s][t][u] = zero16();
  const uint32_t wave_m = wave / WN * (MT * 32), wave_n = wave % WN * (NT * 32), row = lane & 31, half = lane >> 5;

  {
    const SplitWeights weights;
    f32x4 raw[U][2];
    u32x4 pieces[kSplitPieces];
    auto piece_of = [&](int i, int buffer, int p) {
      return i < UA ? &lds[(buffer * kSplitPieces + p) * BM * BK] : &lds[kLeft + (buffer * kSplitPieces + p) * BN * BK];
    };
    // half h of run i: the pieces go to LDS with the second one
    auto stage = [&](int i, int h, int buffer, uint32_t tile) {
      if (h == 0) source.drop(i, tile, raw[i]);
      split4(raw[i][h], pieces, 4 * h, weights);
      if (h == 0) return;
#pragma unroll
      for (int p = 0; p < kSplitPieces; ++p)
        *reinterpret_cast<u32x4*>(piece_of(i, buffer, p) + tile_at(source.row_of(i), source.chunk_of(i))) = pieces[p];
    };
    bf16x8 left[2][MT][kSplitPieces], right[2][NT][kSplitPieces];
    // piece p of an operand, k 16 * part .. + 15 of the tile
    auto fetch_left = [&](int buffer, int part, int p) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
        left[part][t][p] = *reinterpret_cast<const bf16x8*>(piece_of(0, buffer, p) + tile_at(wave_m + t * 32 + row, part * 2 + half));
    };
    auto fetch_right = [&](int buffer, int part, int p) {
#pragma unroll
      for (int u = 0; u < NT; ++u)
        right[part][u][p] = *reinterpret_cast<const bf16x8*>(piece_of(UA, buffer, p) + tile_at(wave_n + u * 32 + row, part * 2 + half));
    };
    auto multiply = [&](int part, int i) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          f32x16& to = sums[i + 1 < kSplitProducts][t][u];
          to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(left[part][t][kSplitLeft[i]], right[part][u][kSplitRight[i]], to, 0, 0, 0);
        }
    };
    // After product i of a half: pieces of the next half, those that its first product needs early, the others as the
    // present half's last use frees their registers.
    auto fetch_next = [&](int i, int buffer, int part) {
      if (i == 0) {
        fetch_left(buffer, part, 0);
        fetch_right(buffer, part, 0);
        fetch_right(buffer, part, 2);
      }
      if (i == 1) fetch_left(buffer, part, 2);
      if (i == 3) fetch_right(buffer, part, 1);
      if (i == 4) fetch_left(buffer, part, 1);
    };
    // One tile of k.  Its first half's fragments are in registers when it begins.  The products of that half run beside
    // the splitting of the next tile into the other buffer, those of the second beside the reads of the next tile's first
    // fragments: one barrier a tile, and no product waits for a read that was just issued.
    auto step = [&](uint32_t tile, int buffer) {
#pragma unroll
      for (int i = 0; i < kSplitProducts; ++i) {
        multiply(0, i);
        fetch_next(i, buffer, 1);
#pragma unroll
        for (int j = i * 2 * U / kSplitProducts; j < (i + 1) * 2 * U / kSplitProducts; ++j) {
          stage(j / 2, j % 2, buffer ^ 1, tile + 1);
          if (j % 2) source.load(j / 2, tile + 2, raw[j / 2]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kSplitProducts; ++i) {
        multiply(1, i);
        fetch_next(i, buffer ^ 1, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
#pragma unroll
    for (int i = 0; i < U; ++i) source.load(i, 0, raw[i]);
#pragma unroll
    for (int j = 0; j < 2 * U; ++j) stage(j / 2, j % 2, 0, 0);
#pragma unroll
    for (int i = 0; i < U; ++i) source.load(i, 1, raw[i]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSplitProducts; ++i) fetch_next(i, 0, 0);
    for (uint32_t tile = 0; tile < tiles; tile += 2) {
      step(tile, 0);
      step(tile + 1, 1);
    }
  }

  bool found = false;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float sum = sums[0][t][u][r] + sums[1][t][u][r];
        found |= not_finite(sum);
        result[t][u][r] = sum * kSplitUnscale;
      }
  if (__syncthreads_or(found)) {
    // In float: chains of a tile's 32 products, added up.
    constexpr int LD = BK + 4;
    float* left = reinterpret_cast<float*>(lds);
    float* right = left + BM * LD;
    static_assert((BM + BN) * LD * 4 <= (kLeft + kRight) * 2, "the floats fit where their pieces were");
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) result[t][u][r] = 0.f;
    source.rewind();
    for (uint32_t tile = 0; tile < tiles; ++tile) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        f32x4 raw[2];
        source.load(i, tile, raw);
        source.drop(i, tile, raw);
        float* to = (i < UA ? left : right) + source.row_of(i) * LD + source.chunk_of(i) * 8;
        *reinterpret_cast<f32x4*>(to) = raw[0];
        *reinterpret_cast<f32x4*>(to + 4) = raw[1];
      }
      __syncthreads();
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          f32x16 sum = zero16();
          for (int k = 0; k < BK; k += 8) {
            const f32x4 l = *reinterpret_cast<const f32x4*>(left + (wave_m + t * 32 + row) * LD + k + 4 * half);
            const f32x4 r = *reinterpret_cast<const f32x4*>(right + (wave_n + u * 32 + row) * LD + k + 4 * half);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_32x32x2f32(l[e], r[e], sum, 0, 0, 0);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) result[t][u][r] += sum[r];
        }
      __syncthreads();
    }
  }
}

}  // namespace cthip
