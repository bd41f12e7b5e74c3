// grouped.h -- what products of rows with the matrix of their group have in common: where groups and tiles are, the operands
// of a tile, and the choice of a kernel.
//
// Groups are runs of rows between offsets in device memory, or all rows where there are none.  A call launches as many blocks as the
// tiles can be at most: the tiles of all rows and one more to each group.  A block finds its group by adding up the groups' tiles;
// blocks beyond the last tile end.  Offsets are clamped as they are read, so that no content of theirs leads outside a buffer.
#pragma once

#include <algorithm>
#include <optional>

#include "common.h"
#include "split_tile.h"

namespace cthip {

struct GroupedArgs {
  const void* a;
  const void* b;
  void* c;
  const int32_t* index_a;
  const int32_t* index_b;
  const int32_t* offsets;
  int64_t lda, ldb, ldc, b_stride, c_stride, c_split;   // c_split: between the results of a launch's parts of k
  double alpha, beta;
  uint32_t groups, rows, a_rows, b_rows, m, n, k;   // m, k: of the weights' products only where rows are not
  uint32_t part;   // k of a part
  bool trans_b;
};

struct Group {
  uint32_t index, first, rows, tile;
};

__device__ __forceinline__ uint2 group_rows(const GroupedArgs& a, uint32_t g) {
  if (!a.offsets) return make_uint2(0, a.rows);
  const int32_t most = (int32_t)a.rows;
  const int32_t first = min(max(a.offsets[g], 0), most), end = min(max(a.offsets[g + 1], first), most);
  return make_uint2((uint32_t)first, (uint32_t)(end - first));
}

// The group of row tile `tile`, of `height` rows: found by every wave, 64 groups at a time.
__device__ __forceinline__ bool find_group(const GroupedArgs& a, uint32_t tile, uint32_t height, Group* out) {
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t g0 = 0; g0 < a.groups; g0 += 64) {
    const uint32_t g = g0 + lane;
    uint2 r = make_uint2(0, 0);
    if (g < a.groups) r = group_rows(a, g);
    const uint32_t tiles = (r.y + height - 1) / height;
    uint32_t upto = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t y = __shfl_up(upto, d);
      if (lane >= (uint32_t)d) upto += y;
    }
    const uint64_t over = __ballot(upto > tile);
    if (over) {
      const int at = __ffsll((unsigned long long)over) - 1;
      out->index = g0 + at;
      out->first = __shfl(r.x, at);
      out->rows = __shfl(r.y, at);
      out->tile = tile - (__shfl(upto, at) - __shfl(tiles, at));
      return true;
    }
    tile -= __shfl(upto, 63);
  }
  return false;
}

template <class T>
__device__ __forceinline__ void put(T* cell, T sum, double alpha, double beta) {
  const T value = (T)alpha * sum;
  *cell = beta == 0 ? value : value + (T)beta * *cell;
}

// Tiles in bands of kBand rows, column after column, part of k after part, dealt to the dies in runs: what a die works on at a
// time is as square as it can be and mostly of one group, and each die has a part of every group.  Runs of kRun, or as many as
// give every die one (64 tiles in runs of 16 would leave four dies idle).
constexpr uint32_t kBand = 8, kRun = 16;

struct GroupedPlan {
  uint32_t m_tiles, n_tiles, units, parts, run_shift;   // m_tiles: as many as there can be; units: of all parts
  uint32_t first;                                       // unit of this launch
  uint32_t band;                                        // rows of tiles of a band
  FastDiv part_fd, band_fd;
};

struct TilePlace {
  uint32_t m_tile, n_tile, part;
};

__device__ __forceinline__ bool place_of(const GroupedPlan& p, TilePlace* out) {
  const uint32_t at = blockIdx.x / kXcds, run = at >> p.run_shift;
  uint32_t unit = p.first + ((run * kXcds + blockIdx.x % kXcds) << p.run_shift) + (at - (run << p.run_shift));
  if (unit >= p.units) return false;
  uint32_t band, rest;
  p.part_fd.divmod(unit, out->part, unit);
  p.band_fd.divmod(unit, band, rest);
  const uint32_t rows = min(p.band, p.m_tiles - band * p.band);
  out->n_tile = rest / rows;
  out->m_tile = band * p.band + rest - out->n_tile * rows;
  return true;
}

// Rows of a by their indexes, 32 k and more; the matrix of the group.  Rows beyond the group's last one repeat it.  As in ct_gemm six
// bfloat16 products to a float product bound the tiles: 16 groups of 1024 rows, 1024 by 2048, 430 us (160 TFLOP/s), its rows' gradient 396, the
// weights' 440.
template <int BM, int BN, int T, bool kB>
struct GroupedSource : TileShare<BM, BN, T, true, kB> {
  using Share = TileShare<BM, BN, T, true, kB>;
  using Share::BK;
  using Share::U;
  using Share::UA;
  using Share::UB;
  const float* row_a[UA];
  bool absent[UA], any_absent;   // an index outside a: zeros in the place of its row
  const float* base_b;
  int64_t ldb;
  uint32_t k, begin;
  uint32_t offset[UB];
  __device__ __forceinline__ GroupedSource(const GroupedArgs& a, const Group& g, uint32_t row0, uint32_t col0, uint32_t begin, uint32_t tid)
      : Share{tid}, any_absent(false), ldb(a.ldb), k(a.k), begin(begin) {
#pragma unroll
    for (int i = 0; i < UA; ++i) {
      const uint32_t row = g.first + min(row0 + this->row_of(i), g.rows - 1), from = a.index_a ? (uint32_t)a.index_a[row] : row;
      absent[i] = from >= a.a_rows;
      any_absent |= absent[i];
      row_a[i] = static_cast<const float*>(a.a) + (int64_t)(absent[i] ? 0 : from) * a.lda + this->chunk_of(i) * 8;
    }
    any_absent = __ballot(any_absent) != 0;
    base_b = static_cast<const float*>(a.b) + (int64_t)g.index * a.b_stride + (int64_t)col0 * (kB ? a.ldb : 1);
#pragma unroll
    for (int i = 0; i < UB; ++i) {
      const uint32_t r = min(this->row_of(UA + i), a.n - 1 - col0), chunk = this->chunk_of(UA + i);
      offset[i] = 4 * (kB ? r * (uint32_t)a.ldb + chunk * 8 : chunk * 8 * (uint32_t)a.ldb + r);
    }
  }
  __device__ __forceinline__ void rewind() {}
  __device__ __forceinline__ void load(int i, uint32_t tile, f32x4 (&to)[2]) const {
    const int64_t k0 = min(begin + tile * BK, k - BK);
    if (i < UA) {
      __builtin_memcpy(&to[0], row_a[i] + k0, 16);
      __builtin_memcpy(&to[1], row_a[i] + k0 + 4, 16);
    } else {
      load8<kB>(base_b + (kB ? k0 : k0 * ldb), offset[i - UA], ldb, to);
    }
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

// The sums of 16 rows by 16 NT columns in the float instructions: W waves take every W-th run of 32 k each, straight from memory into the
// operands of v_mfma_f32_16x16x4_f32, and leave their sums in LDS, [wave][row][column].  `left` is row lane % 16, zeros if it is absent;
// `right` if kB column u * 16 + lane % 16 of each u, else the row of k 0, of which a lane takes the NT columns from lane % 16 * NT on,
// side by side; there are `columns` of them.
template <int W, int NT, bool kB>
__device__ __forceinline__ void thin_sums(const float* left, bool absent, const float* const (&right)[kB ? NT : 1], int64_t ldb, uint32_t columns,
                                          uint32_t k_end, float (&partial)[W][256 * NT]) {
  constexpr uint32_t BN = 16 * NT, BK = 32;
  static_assert(NT == 1 || NT == 4, "loads of one column or four");
  const uint32_t lane = threadIdx.x & 63, at16 = lane % 16, quarter = lane / 16, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool any_absent = __ballot(absent) != 0, whole = kB || at16 * NT + NT - 1 < columns;
  // eight k from k0 + 8 * quarter on: of a row, of a column, of all columns where they are side by side
  auto load_eight = [&](const float* from, uint32_t k0, f32x4 (&x)[2]) {
    const uint32_t k = k0 + quarter * 8;
    if (k0 + BK <= k_end) {
      __builtin_memcpy(&x[0], from + k, 16);
      __builtin_memcpy(&x[1], from + k + 4, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = from[min(k + e, k_end - 1)];
        x[e / 4][e % 4] = k + e < k_end ? y : 0.f;
      }
    }
  };
  auto load_columns = [&](uint32_t k0, f32x4 (&r)[NT][2]) {
    const uint32_t k = k0 + quarter * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float* at = right[0] + (int64_t)min(k + e, k_end - 1) * ldb;
      if constexpr (NT == 1) {
        r[0][e / 4][e % 4] = at[min(at16, columns - 1)];
      } else {
        f32x4 four;
        if (whole) __builtin_memcpy(&four, at + at16 * 4, 16);
        else {
#pragma unroll
          for (int u = 0; u < NT; ++u) four[u] = at[min(at16 * NT + u, columns - 1)];
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) r[u][e / 4][e % 4] = four[u];
      }
    }
    if (k0 + BK > k_end) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int u = 0; u < NT; ++u) r[u][e / 4][e % 4] = k + e < k_end ? r[u][e / 4][e % 4] : 0.f;
    }
  };
  auto load_left = [&](uint32_t k0, f32x4 (&l)[2]) {
    load_eight(left, k0, l);
    if (any_absent && absent) l[0] = l[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  f32x4 sums[NT] = {}, l[2], l_next[2], r[NT][2];
  const uint32_t mine = wave * BK;
  if (mine < k_end) {
    load_left(mine, l);
    if constexpr (kB) {
#pragma unroll
      for (int u = 0; u < NT; ++u) load_eight(right[u], mine, r[u]);
    } else {
      load_columns(mine, r);
    }
  }
  auto multiply = [&](int u) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(l[e / 4][e % 4], r[u][e / 4][e % 4], sums[u], 0, 0, 0);
  };
  uint32_t next = mine + W * BK;
  for (; next < k_end; next += W * BK) {   // no load behind a branch, which would be waited for at once
    load_left(next, l_next);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      multiply(u);
      // the column's next run into the registers of this one
      if constexpr (kB) load_eight(right[u], next, r[u]);
    }
    if constexpr (!kB) load_columns(next, r);
    l[0] = l_next[0];
    l[1] = l_next[1];
  }
  if (mine < k_end) {
#pragma unroll
    for (int u = 0; u < NT; ++u) multiply(u);
  }
#pragma unroll
  for (int u = 0; u < NT; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) partial[wave][(quarter * 4 + e) * BN + (kB ? u * 16 + at16 : at16 * NT + u)] = sums[u][e];
  __syncthreads();
}

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A launch of 2^32 lanes or more is refused, and a block has up to 1024: more tiles than this take several launches.
constexpr int64_t kMostUnits = int64_t(1) << 21, kMostTiles = (int64_t(1) << 31) - 1;
static_assert(kMostUnits % (kXcds * kRun) == 0, "a launch ends with a round of runs");

// Calls `launch(grid, plan)` for launches that together have a block for every unit.  Bands of one row of tiles leave the blocks
// without a tile for the end: between the others they would leave every other unit of the chip without work (16 rows by 8192 gates and
// ups of 4096: 82 us, 54 of 12 rows).
template <class F>
void for_launches(int64_t m_tiles, int64_t n_tiles, int64_t parts, F launch, uint32_t band = kBand) {
  GroupedPlan p;
  p.m_tiles = (uint32_t)m_tiles;
  p.n_tiles = (uint32_t)n_tiles;
  p.units = (uint32_t)(m_tiles * n_tiles * parts);
  p.parts = (uint32_t)parts;
  p.run_shift = 0;
  while ((uint32_t(2) << p.run_shift) <= std::min(kRun, p.units / kXcds)) ++p.run_shift;
  p.part_fd = FastDiv((uint32_t)(m_tiles * n_tiles));
  p.band = band;
  p.band_fd = FastDiv((uint32_t)(band * n_tiles));
  const int64_t round = (int64_t)kXcds << p.run_shift;
  for (int64_t first = 0; first < p.units; first += kMostUnits) {
    p.first = (uint32_t)first;
    launch(dim3((uint32_t)(ceil_div(std::min(p.units - first, kMostUnits), round) * round)), p);
  }
}

// Sums whose k is divided among blocks: their products go to scratch, and a second launch adds them up.
template <class T>
class Parts {
 public:
  // As many as asked for, or one where no scratch is to be had: while the stream is being captured, or for want of memory.
  Parts(hipStream_t s, int64_t parts, int64_t cells) : cells_(cells), count_(1) {
    if (parts == 1) return;
    scratch_.emplace(s, (size_t)(parts * cells) * sizeof(T));
    partial_ = static_cast<T*>(scratch_->get());
    if (partial_) count_ = parts;
  }
  int64_t count() const { return count_; }
  // Of the first launch; matrices of `m` rows, or none.
  GroupedArgs args(GroupedArgs a, int64_t m) const {
    if (!partial_) return a;
    a.c = partial_;
    a.ldc = a.n;
    a.c_stride = m * a.n;
    a.c_split = cells_;
    a.alpha = 1.0;
    a.beta = 0.0;
    return a;
  }
  const T* partial() const { return partial_; }
  int64_t cells() const { return cells_; }

 private:
  std::optional<ProductScratch> scratch_;   // until both launches are made
  T* partial_ = nullptr;
  int64_t cells_, count_;
};

// The second launch, and its bytes at 3.3 TB/s; no more than the scratch there may be.
inline double time_of_sum(int64_t parts, int64_t cells, int64_t size) {
  if (parts == 1) return 0.0;
  return parts * cells * size > (int64_t)kMostProductScratch ? 1e9 : 4.5 + 0.3e-6 * (double)((parts + 1) * cells * size);
}

// Microseconds of `blocks` tiles of 64 or of 128 a side over k_tiles of 32 k: the lines of ct_gemm's kernels.
constexpr int64_t kUnits = 256;
inline double time_of_medium(int64_t blocks, int64_t k_tiles) {
  const int64_t full = blocks / (3 * kUnits), rest = blocks - full * 3 * kUnits, shared = full * 3 + ceil_div(rest, kUnits);
  return 3.3 + 1.3 * (double)shared + (double)k_tiles * (0.31 * (double)(full + (rest > 0)) + 0.33 * (double)shared);
}
inline double time_of_large(int64_t blocks, int64_t k_tiles) { return 1.8 + (double)ceil_div(blocks, 256) * (3.7 + 1.19 * (double)k_tiles); }
struct Choice {
  int64_t height, width, parts;
  double us;
};

// Of k_tiles tiles of k, divided evenly and in pairs of tiles: those of a part.
inline int64_t tiles_of_part(int64_t k_tiles, int64_t parts) { return ceil_div(ceil_div(k_tiles, parts), 2) * 2; }

constexpr int64_t kMostParts = 32;
// Large tiles of parts, a round of blocks at a time, are written at once.
inline double write_of_parts(int64_t parts, int64_t blocks) { return parts > 1 ? 6.0 * (double)ceil_div(blocks * parts, kUnits) : 0.0; }

// Tiles of 64 and 128 a side, with k in one part or several, against the best so far.  The times of 64 products of 2 and 8 even groups,
// 64 to 1024 rows each, k 1024 to 4096: 5 % above the best plan's of each.  Us of one part and of what is chosen: 2 groups of 128 rows,
// k 4096, n 1024: 89 and 29; 8 groups of 64, k 4096, n 1024: 88 and 52; of the weights' products 8 groups of 4096 rows, 128 by 128: 110 and 47.
inline void consider_parts(Choice* best, int64_t blocks64, int64_t blocks128, int64_t k_tiles, int64_t cells, int64_t most_parts) {
  for (int64_t parts = 1; parts <= most_parts; parts *= 2) {
    const int64_t tiles = parts == 1 ? k_tiles : tiles_of_part(k_tiles, parts);
    if (parts > 1 && tiles * (parts - 1) >= k_tiles) break;   // the last part would have none
    const double sum = time_of_sum(parts, cells, sizeof(float));
    const double medium = time_of_medium(blocks64 * parts, tiles) + sum, large = time_of_large(blocks128 * parts, tiles) + sum + write_of_parts(parts, blocks128);
    if (medium < best->us) *best = {64, 64, parts, medium};
    if (large < best->us) *best = {128, 128, parts, large};
  }
}

// The same of double, tiles of 32 and 64 a side: one block's steps over the longest sum, or those of all blocks over the mean one.  Of
// the weights' products the longest is taken to be twice the mean, for groups are seldom even (7 groups of 290 rows in the mean, 301 by
// 517: 35 us in tiles of 32, 56 in tiles of 64, which take 18 where they are even).
inline double time_of_double(int64_t side, int64_t blocks, double mean_k, double longest_k) {
  const double one = side == 32 ? 0.020 : 0.054;
  const double all = side == 32 ? 0.010 + 0.0000475 * (double)blocks : 0.015 + 0.037 * (double)ceil_div(blocks, kUnits);
  return 4.0 + std::max(longest_k * one, mean_k * all);
}
inline void consider_double_parts(Choice* best, int64_t blocks32, int64_t blocks64, int64_t mean_k, int64_t longest_k, int64_t cells, int64_t most_parts) {
  for (int64_t parts = 1; parts <= most_parts && (parts == 1 || mean_k >= parts * 64); parts *= 2) {
    const double sum = time_of_sum(parts, cells, sizeof(double)), mean = (double)mean_k / (double)parts, longest = (double)longest_k / (double)parts;
    const double small = time_of_double(32, blocks32 * parts, mean, longest) + sum, large = time_of_double(64, blocks64 * parts, mean, longest) + sum + write_of_parts(parts, blocks64);
    if (small < best->us) *best = {32, 32, parts, small};
    if (large < best->us) *best = {64, 64, parts, large};
  }
}

constexpr int64_t kMostSplitLd = int64_t(1) << 22, kMostWeightsLd = int64_t(1) << 30;

constexpr int64_t kMostExtent = (int64_t(1) << 31) - 1;
inline bool extent(int64_t n) { return n >= 0 && n <= kMostExtent; }
constexpr int64_t kMostGroups = 65535;

}  // namespace cthip
