// ops_grouped.hip -- products of rows with the matrix of their group (ct_grouped_gemm), and the products over the rows of
// each group that are those matrices' gradients (ct_grouped_gemm_weights).
#include "common.h"
#include "double_tile.h"
#include "grouped.h"
#include "rows.h"
#include "split_tile.h"

using namespace cthip;

namespace {

constexpr int kSide = 64, kDepth = 16;

// One tile of kSide x kSide: `left(row, k)` and `right(k, column)` are elements, zero outside.
template <class T, class Left, class Right, class Store>
__device__ __forceinline__ void tile_product(uint32_t depth, Left left, Right right, Store store) {
  __shared__ T lds_a[kDepth][kSide + 1], lds_b[kDepth][kSide + 1];
  const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  T sum[4][4] = {};
  for (uint32_t k0 = 0; k0 < depth; k0 += kDepth) {
    for (uint32_t i = threadIdx.x; i < kSide * kDepth; i += 256) {
      lds_a[i % kDepth][i / kDepth] = left(i / kDepth, k0 + i % kDepth);
      lds_b[i / kSide][i % kSide] = right(k0 + i / kSide, i % kSide);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = fma(lds_a[k][ty * 4 + i], lds_b[k][tx * 4 + j], sum[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) store(ty * 4 + i, tx * 4 + j, sum[i][j]);
}

// Of operands without rows, and of sums without terms.  A block takes every so manieth tile of rows and of columns, here and below.
template <class T>
__global__ void __launch_bounds__(256) grouped_kernel(const GroupedArgs a) {
  Group g;
  for (uint32_t tile = blockIdx.y; find_group(a, tile, kSide, &g); tile += gridDim.y) {
    const uint32_t row0 = g.tile * kSide;
    const T* b = static_cast<const T*>(a.b) + (int64_t)g.index * a.b_stride;
    for (uint32_t col0 = blockIdx.x * kSide; col0 < a.n; col0 += gridDim.x * kSide) {
      T* c = static_cast<T*>(a.c) + (int64_t)(g.first + row0) * a.ldc + col0;
      tile_product<T>(
          a.k,
          [&](uint32_t r, uint32_t k) -> T {
            if (row0 + r >= g.rows || k >= a.k) return 0;
            const uint32_t i = g.first + row0 + r, from = a.index_a ? (uint32_t)a.index_a[i] : i;
            return from < a.a_rows ? static_cast<const T*>(a.a)[(int64_t)from * a.lda + k] : T(0);
          },
          [&](uint32_t k, uint32_t n) -> T {
            if (k >= a.k || col0 + n >= a.n) return 0;
            return a.trans_b ? b[(int64_t)(col0 + n) * a.ldb + k] : b[(int64_t)k * a.ldb + col0 + n];
          },
          [&](uint32_t r, uint32_t n, T sum) {
            if (row0 + r < g.rows && col0 + n < a.n) put(c + (int64_t)r * a.ldc + n, sum, a.alpha, a.beta);
          });
    }
  }
}

// Of floats whose rows lie further apart than the tiles' offsets reach.
__global__ void __launch_bounds__(256) grouped_weights_kernel(const GroupedArgs a) {
  const uint32_t group = blockIdx.z;
  const uint2 rows = group_rows(a, group);
  float* c = static_cast<float*>(a.c) + (int64_t)group * a.c_stride;
  auto element = [&](const void* p, const int32_t* index, uint32_t count, int64_t ld, uint32_t k, uint32_t column, uint32_t width) -> float {
    if (k >= rows.y || column >= width) return 0;
    const uint32_t i = rows.x + k, from = index ? (uint32_t)index[i] : i;
    return from < count ? static_cast<const float*>(p)[(int64_t)from * ld + column] : 0.f;
  };
  for (uint32_t row0 = blockIdx.y * kSide; row0 < a.m; row0 += gridDim.y * kSide)
    for (uint32_t col0 = blockIdx.x * kSide; col0 < a.n; col0 += gridDim.x * kSide)
      tile_product<float>(
          rows.y, [&](uint32_t r, uint32_t k) { return element(a.a, a.index_a, a.a_rows, a.lda, k, row0 + r, a.m); },
          [&](uint32_t k, uint32_t n) { return element(a.b, a.index_b, a.b_rows, a.ldb, k, col0 + n, a.n); },
          [&](uint32_t r, uint32_t n, float sum) {
            if (row0 + r < a.m && col0 + n < a.n) put(c + (int64_t)(row0 + r) * a.ldc + col0 + n, sum, a.alpha, a.beta);
          });
}

// ------------------------------------------------------------------ float: the matrix cores, three pieces to a float

template <int MT, int NT>
__device__ __forceinline__ void store_tile(const GroupedArgs& a, float* c, uint32_t rows, uint32_t columns, uint32_t wave_m, uint32_t wave_n,
                                           uint32_t lane, const float (&result)[MT][NT][16]) {
  const uint32_t column = lane & 31, half = lane >> 5;
  const float alpha = (float)a.alpha, beta = (float)a.beta;
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const uint32_t n = wave_n + u * 32 + column;
    if (n >= columns) continue;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t m = wave_m + t * 32 + 8 * (r / 4) + 4 * half + r % 4;
        if (m >= rows) continue;
        float& cell = c[(int64_t)m * a.ldc + n];
        const float value = alpha * result[t][u][r];
        cell = beta == 0.f ? value : value + beta * cell;
      }
  }
}

template <int BM, int BN, int WM, int WN, bool kB>
__global__ void __launch_bounds__(64 * WM * WN, 2) grouped_split_kernel(const GroupedArgs a, const GroupedPlan p) {
  constexpr int T = 64 * WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
  __shared__ __attribute__((aligned(16))) uint16_t lds[split_tile_lds(BM, BN)];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a, at.m_tile, BM, &g)) return;
  const uint32_t row0 = g.tile * BM, col0 = at.n_tile * BN, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t begin = at.part * a.part, count = min(a.part, a.k - begin);
  GroupedSource<BM, BN, T, kB> source(a, g, row0, col0, begin, tid);
  float result[MT][NT][16];
  split_tile<BM, BN, WM, WN>(source, (count + 2 * kTileDepth - 1) / (2 * kTileDepth) * 2, lds, tid, result);
  store_tile(a, static_cast<float*>(a.c) + at.part * a.c_split + (int64_t)(g.first + row0) * a.ldc + col0, g.rows - row0, a.n - col0, wave / WN * (MT * 32),
             wave % WN * (NT * 32), tid & 63, result);
}

// The rows of a group whose products a block adds up: an even share, of whole tiles, for each of the parts.
__device__ __forceinline__ uint2 part_of(uint2 rows, uint32_t part, uint32_t parts) {
  if (parts == 1) return rows;
  const uint32_t each = ((rows.y + parts - 1) / parts + 2 * kTileDepth - 1) / (2 * kTileDepth) * (2 * kTileDepth), from = min(part * each, rows.y);
  return make_uint2(rows.x + from, min(each, rows.y - from));
}

// Columns of the rows of a group, over which the products' sums run.  A wave loads eight rows at a time: its lanes 0 to 7
// hold where they begin, read a tile ahead where there are indexes, and each load takes one as a scalar.  Rows beyond the
// group's last one, and those of indexes outside the operand, are zeros.
// kWide: operands of 4 GiB and more, with 64 bits to a row's place.  (Indexes read into scalar registers, and 64-bit scalar
// addresses, took three times as long: 1500 and 470 us of 16 groups of 1024 rows, 2048 by 1024; the scalar loads were waited
// for with all of LDS, and the addresses spilled.)
template <int BM, int BN, int T, bool kWide>
struct GroupedWeightsSource : TileShare<BM, BN, T, false, false> {
  using Share = TileShare<BM, BN, T, false, false>;
  using Share::BK;
  using Share::U;
  using Share::UA;
  using Place = std::conditional_t<kWide, uint64_t, uint32_t>;
  const float *base_a, *base_b;
  const int32_t *index_a, *index_b;
  uint32_t lda, ldb, rows_a, rows_b, first, rows;
  uint32_t offset[U], chunk[U], absent[U], next[U];
  __device__ __forceinline__ GroupedWeightsSource(const GroupedArgs& a, uint32_t first, uint32_t rows, uint32_t row0, uint32_t col0, uint32_t tid)
      : Share{tid}, base_a(static_cast<const float*>(a.a) + row0), base_b(static_cast<const float*>(a.b) + col0), index_a(a.index_a),
        index_b(a.index_b), lda((uint32_t)a.lda), ldb((uint32_t)a.ldb), rows_a(a.a_rows), rows_b(a.b_rows), first(first), rows(rows) {
    static_assert(BM % 64 == 0 && BN % 64 == 0, "a wave's lanes are columns of one run");
#pragma unroll
    for (int i = 0; i < U; ++i) {
      offset[i] = 4 * min(this->row_of(i), i < UA ? a.m - 1 - row0 : a.n - 1 - col0);
      chunk[i] = __builtin_amdgcn_readfirstlane(this->chunk_of(i));
      absent[i] = 0;
    }
    rewind();
  }
  __device__ __forceinline__ uint32_t row_at(uint32_t i, uint32_t tile) const { return tile * BK + chunk[i] * 8 + (this->tid & 7); }
  __device__ __forceinline__ void look_up(int i, uint32_t tile) {
    const uint32_t row = first + min(row_at(i, tile), rows - 1);
    const int32_t* index = i < UA ? index_a : index_b;
    next[i] = index ? (uint32_t)index[row] : row;
  }
  __device__ __forceinline__ void rewind() {
#pragma unroll
    for (int i = 0; i < U; ++i) look_up(i, 0);
  }
  __device__ __forceinline__ void load(int i, uint32_t tile, f32x4 (&to)[2]) {
    const bool outside = next[i] >= (i < UA ? rows_a : rows_b);
    absent[i] = (uint32_t)__ballot(outside || row_at(i, tile) >= rows) & 0xff;
    const Place begin = (Place)(outside ? 0 : next[i]) * (4 * (Place)(i < UA ? lda : ldb));
    uint64_t base = reinterpret_cast<uint64_t>(i < UA ? base_a : base_b);
    asm("" : "+s"(base));
    typedef __attribute__((address_space(1))) const char* Global;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      Place at = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)begin, e);
      if constexpr (kWide) at |= (Place)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(begin >> 32), e) << 32;
      to[e / 4][e % 4] = *reinterpret_cast<__attribute__((address_space(1))) const float*>(reinterpret_cast<Global>(base) + (Place)(at + offset[i]));
    }
    look_up(i, tile + 1);
  }
  __device__ __forceinline__ void drop(int i, uint32_t, f32x4 (&r)[2]) const {
    if (absent[i] == 0) return;
    asm volatile("");   // stays a branch
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e / 4][e % 4] = absent[i] >> e & 1 ? 0.f : r[e / 4][e % 4];
  }
};

template <int BM, int BN, int WM, int WN, bool kWide>
__global__ void __launch_bounds__(64 * WM * WN, 2) grouped_weights_split_kernel(const GroupedArgs a, const GroupedPlan p) {
  constexpr int T = 64 * WM * WN, MT = BM / WM / 32, NT = BN / WN / 32;
  __shared__ __attribute__((aligned(16))) uint16_t lds[split_tile_lds(BM, BN)];
  TilePlace at;
  if (!place_of(p, &at)) return;
  const uint32_t tiles = (a.m + BM - 1) / BM, group = at.m_tile / tiles, row0 = (at.m_tile - group * tiles) * BM, col0 = at.n_tile * BN;
  const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint2 rows = part_of(group_rows(a, group), at.part, p.parts);
  const uint32_t first = __builtin_amdgcn_readfirstlane(rows.x), count = __builtin_amdgcn_readfirstlane(rows.y);
  float result[MT][NT][16] = {};
  if (count > 0 && a.a_rows > 0 && a.b_rows > 0) {
    GroupedWeightsSource<BM, BN, T, kWide> source(a, first, count, row0, col0, tid);
    split_tile<BM, BN, WM, WN>(source, (count + 2 * kTileDepth - 1) / (2 * kTileDepth) * 2, lds, tid, result);
  }
  store_tile(a, static_cast<float*>(a.c) + at.part * a.c_split + (int64_t)group * a.c_stride + (int64_t)row0 * a.ldc + col0, a.m - row0, a.n - col0,
             wave / WN * (MT * 32), wave % WN * (NT * 32), tid & 63, result);
}

// ------------------------------------------------------------------ float, a few rows to a group

// What a few tokens ask of their experts is bound by reading the matrices: a block owns 16 rows by 16 NT columns, its W waves
// take every W-th run of 32 k each, straight from memory into the operands of v_mfma_f32_16x16x4_f32, and their sums are added in LDS in
// their order.  That instruction is a sixteenth as fast as those of the split products, but takes the floats as they are: 537 MB
// of 32 matrices, 4096 by 1024, one row each, in 128 us with split products, of which the splitting took what reading left (94 us with
// nothing but the loads).  Of a matrix stored [k][n] a lane takes its NT columns side by side.
template <int W, int NT, bool kB>
__global__ void __launch_bounds__(64 * W, 4) grouped_thin_kernel(const GroupedArgs a, const GroupedPlan p) {
  constexpr uint32_t BM = 16, BN = 16 * NT;
  __shared__ float partial[W][BM * BN];
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a, at.m_tile, BM, &g)) return;
  const uint32_t row0 = g.tile * BM, col0 = at.n_tile * BN, at16 = threadIdx.x % 16;
  const uint32_t row = g.first + min(row0 + at16, g.rows - 1), from = a.index_a ? (uint32_t)a.index_a[row] : row;
  const bool absent = from >= a.a_rows;   // an index outside a: zeros in the place of its row
  const float* left = static_cast<const float*>(a.a) + (int64_t)(absent ? 0 : from) * a.lda;
  const float* b = static_cast<const float*>(a.b) + (int64_t)g.index * a.b_stride;
  const float* right[kB ? NT : 1];
#pragma unroll
  for (int u = 0; u < (kB ? NT : 1); ++u) right[u] = b + (int64_t)(kB ? min(col0 + u * 16 + at16, a.n - 1) : col0) * (kB ? a.ldb : 1);
  thin_sums<W, NT, kB>(left, absent, right, a.ldb, a.n - col0, a.k, partial);
  float* c = static_cast<float*>(a.c) + (int64_t)(g.first + row0) * a.ldc + col0;
  const uint32_t rows = g.rows - row0, columns = a.n - col0;
  for (uint32_t i = threadIdx.x; i < BM * BN; i += 64 * W) {
    float sum = partial[0][i];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += partial[w][i];
    if (i / BN < rows && i % BN < columns) put(c + (int64_t)(i / BN) * a.ldc + i % BN, sum, a.alpha, a.beta);
  }
}

// ------------------------------------------------------------------ double: the matrix cores

template <int S, bool kB>
__global__ void __launch_bounds__(256, 2) grouped_double_kernel(const GroupedArgs a, const GroupedPlan p) {
  TilePlace at;
  Group g;
  if (!place_of(p, &at) || !find_group(a, at.m_tile, S, &g)) return;
  const uint32_t row0 = g.tile * S, col0 = at.n_tile * S;
  const double* b = static_cast<const double*>(a.b) + (int64_t)g.index * a.b_stride;
  double* c = static_cast<double*>(a.c) + at.part * a.c_split + (int64_t)(g.first + row0) * a.ldc + col0;
  const uint32_t begin = at.part * a.part, count = min(a.part, a.k - begin);
  const uint32_t row = g.first + min(row0 + DoubleRow<S>::row(), g.rows - 1), from = a.index_a ? (uint32_t)a.index_a[row] : row;
  const bool present = from < a.a_rows;
  const DoubleRow<S> left{static_cast<const double*>(a.a) + (int64_t)(present ? from : 0) * a.lda + begin, count, present};
  auto store = [&](uint32_t r, uint32_t n, double sum) {
    if (row0 + r < g.rows && col0 + n < a.n) put(c + (int64_t)r * a.ldc + n, sum, a.alpha, a.beta);
  };
  if constexpr (kB) {
    const uint32_t column = min(col0 + DoubleRow<S>::row(), a.n - 1);
    double_tile<S>(count, left, DoubleRow<S>{b + (int64_t)column * a.ldb + begin, count, true}, store);
  } else {
    double_tile<S>(count, left, DoubleColumns<S>(b + (int64_t)begin * a.ldb + col0, a.ldb, nullptr, 0, count, count, a.n - col0), store);
  }
}

template <int S>
__global__ void __launch_bounds__(256, 2) grouped_weights_double_kernel(const GroupedArgs a, const GroupedPlan p) {
  TilePlace at;
  if (!place_of(p, &at)) return;
  const uint32_t tiles = (a.m + S - 1) / S, group = at.m_tile / tiles, row0 = (at.m_tile - group * tiles) * S, col0 = at.n_tile * S;
  const uint2 rows = part_of(group_rows(a, group), at.part, p.parts);
  double* c = static_cast<double*>(a.c) + at.part * a.c_split + (int64_t)group * a.c_stride + (int64_t)row0 * a.ldc + col0;
  auto store = [&](uint32_t r, uint32_t n, double sum) {
    if (row0 + r < a.m && col0 + n < a.n) put(c + (int64_t)r * a.ldc + n, sum, a.alpha, a.beta);
  };
  if (rows.y > 0 && a.a_rows > 0 && a.b_rows > 0) {
    double_tile<S>(rows.y, DoubleColumns<S>(static_cast<const double*>(a.a) + row0, a.lda, a.index_a, rows.x, rows.y, a.a_rows, a.m - row0),
                   DoubleColumns<S>(static_cast<const double*>(a.b) + col0, a.ldb, a.index_b, rows.x, rows.y, a.b_rows, a.n - col0), store);
  } else {
    for (uint32_t i = threadIdx.x; i < S * S; i += 256) store(i / S, i % S, 0.0);
  }
}

// ------------------------------------------------------------------ the parts of k brought together

// partial [parts][c's cells, dense], added in their order: of rows of c (those from the first group's to the last one's only),
// or of matrices.
template <class T, bool kWeights>
__global__ void __launch_bounds__(256) grouped_sum_kernel(const GroupedArgs a, const T* partial, uint32_t parts, uint32_t cells, FastDiv n_fd, FastDiv m_fd) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= cells) return;
  uint32_t row, column, group = 0;
  n_fd.divmod(i, row, column);
  if constexpr (kWeights) {
    m_fd.divmod(row, group, row);
  } else {
    const uint2 last = group_rows(a, a.groups - 1);
    if (row < group_rows(a, 0).x || row >= last.x + last.y) return;
  }
  double sum = 0.0;
  for (uint32_t s0 = 0; s0 < parts; s0 += 8) {   // loads of eight parts on their way
    T x[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = partial[(int64_t)min(s0 + s, parts - 1) * cells + i];
#pragma unroll
    for (int s = 0; s < 8; ++s) sum += s0 + s < parts ? x[s] : T(0);
  }
  put(static_cast<T*>(a.c) + (int64_t)group * a.c_stride + (int64_t)row * a.ldc + column, (T)sum, a.alpha, a.beta);
}

// The second launch, of the parts of the first.
template <bool kWeights, class T>
void add_up(hipStream_t s, const Parts<T>& parts, const GroupedArgs& a) {
  if (!parts.partial()) return;
  hipLaunchKernelGGL((grouped_sum_kernel<T, kWeights>), dim3((uint32_t)ceil_div(parts.cells(), 256)), dim3(256), 0, s, a, parts.partial(),
                     (uint32_t)parts.count(), (uint32_t)parts.cells(), FastDiv(a.n), FastDiv(kWeights ? a.m : 1));
}

// Of the kernel for a few rows, blocks of 64 and of 16 columns.
double time_of_thin64(int64_t blocks, int64_t k_tiles) { return 3.0 + (double)ceil_div(blocks, kUnits) * (0.5 + 0.28 * (double)k_tiles); }
double time_of_thin16(int64_t blocks, int64_t k_tiles) { return 3.0 + (double)ceil_div(blocks, 2 * kUnits) * (0.5 + 0.22 * (double)k_tiles); }

// Up to here a block of the kernel for a few rows has four waves: 64 matrices, 768 by 768 [k][n], 12 rows each, in 30 us, against 36 with eight;
// from 1024 on eight or sixteen are as fast or faster.
constexpr int64_t kFewK = 768;

// Of the kernels whose blocks walk over tiles: as many as one launch may have along each side.
inline dim3 plain_grid(int64_t columns, int64_t row_tiles, int64_t groups) {
  return dim3((uint32_t)std::min(ceil_div(columns, kSide), kMostUnits), (uint32_t)std::min<int64_t>(row_tiles, 65535), (uint32_t)groups);
}

}  // namespace

#define CT_GROUPED_FLOATING(name) CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, name ": datatype must be float or double")

extern "C" {

int ct_grouped_gemm(void* stream, void* c, int64_t c_colstride, int trans_b, double alpha, const void* a, int64_t a_row_count,
                    int64_t a_col_count, int64_t a_colstride, const int32_t* index, const void* b, int64_t b_col_count,
                    int64_t b_colstride, int64_t b_stride, const int32_t* offsets, int64_t n_groups, int64_t row_count,
                    double beta, int dtype) {
  CT_GROUPED_FLOATING("ct_grouped_gemm");
  CT_REQUIRE(extent(a_row_count) && extent(a_col_count) && extent(b_col_count) && extent(row_count), "ct_grouped_gemm: bad extent");
  CT_REQUIRE(n_groups >= 0 && n_groups <= kMostGroups, "ct_grouped_gemm: %lld groups, at most %lld are taken", (long long)n_groups,
             (long long)kMostGroups);
  if (n_groups == 0 || row_count == 0 || b_col_count == 0) return CT_OK;
  CT_REQUIRE(c && offsets && (a_col_count == 0 || (b && (a || a_row_count == 0))), "ct_grouped_gemm: null buffer");
  CT_REQUIRE(index || a_row_count >= row_count, "ct_grouped_gemm: a has %lld rows of %lld", (long long)a_row_count, (long long)row_count);
  const int64_t b_rows = trans_b ? b_col_count : a_col_count, b_cols = trans_b ? a_col_count : b_col_count;
  CT_REQUIRE(c_colstride >= b_col_count && a_colstride >= a_col_count && b_colstride >= b_cols, "ct_grouped_gemm: a column stride below the row's length");
  CT_REQUIRE(b_stride >= 0, "ct_grouped_gemm: negative stride of matrices");
  const int64_t size = dtype_size(dtype);
  const RowRange result{c, row_count, b_col_count, c_colstride};
  CT_REQUIRE(!rows_meet(result, {a_col_count ? a : nullptr, a_row_count, a_col_count, a_colstride}, size) &&
                 !run_meets({a_col_count ? b : nullptr, ((n_groups - 1) * b_stride + (b_rows - 1) * b_colstride + b_cols) * size}, result, size),
             "ct_grouped_gemm: c overlaps an operand");
  CT_REQUIRE(!run_meets({offsets, (n_groups + 1) * 4}, result, size) && !run_meets({index, row_count * 4}, result, size),
             "ct_grouped_gemm: c overlaps the offsets or the index");
  hipStream_t s = static_cast<hipStream_t>(stream);
  GroupedArgs g{};
  g.a = a; g.b = b; g.c = c; g.index_a = index; g.offsets = offsets;
  g.lda = a_colstride; g.ldb = b_colstride; g.ldc = c_colstride; g.b_stride = b_stride;
  g.alpha = alpha; g.beta = beta;
  g.groups = (uint32_t)n_groups; g.rows = (uint32_t)row_count; g.a_rows = (uint32_t)a_row_count;
  g.n = (uint32_t)b_col_count; g.k = (uint32_t)a_col_count;
  g.trans_b = trans_b != 0;
  const int64_t even_groups = std::min(n_groups, row_count);
  const int64_t cells = row_count * b_col_count;
  auto row_tiles_of = [&](int64_t height) { return even_groups * ceil_div(row_count / even_groups, height); };   // if the groups are even
  auto blocks_of = [&](int64_t side) { return row_tiles_of(side) * ceil_div(b_col_count, side); };
  if (dtype == CT_F64 && a_row_count > 0 && a_col_count > 0) {
    auto choose = [&](int64_t most_parts) {
      Choice best{32, 32, 1, 1e12};
      consider_double_parts(&best, blocks_of(32), blocks_of(64), a_col_count, a_col_count, cells, most_parts);
      return best;
    };
    Choice best = choose(kMostParts);
    const Parts<double> parts(s, best.parts, cells);
    if (parts.count() < best.parts) best = choose(1);
    const int64_t side = best.height, m_tiles = row_count / side + even_groups, n_tiles = ceil_div(b_col_count, side);
    CT_REQUIRE(m_tiles <= kMostTiles / parts.count() / n_tiles, "ct_grouped_gemm: %lld rows of %lld columns", (long long)row_count, (long long)b_col_count);
    GroupedArgs of_parts = parts.args(g, 0);
    of_parts.part = (uint32_t)ceil_div(a_col_count, parts.count());
    for_launches(m_tiles, n_tiles, parts.count(), [&](dim3 grid, const GroupedPlan& plan) {
      if (side == 64 && trans_b) hipLaunchKernelGGL((grouped_double_kernel<64, true>), grid, dim3(256), 0, s, of_parts, plan);
      else if (side == 64) hipLaunchKernelGGL((grouped_double_kernel<64, false>), grid, dim3(256), 0, s, of_parts, plan);
      else if (trans_b) hipLaunchKernelGGL((grouped_double_kernel<32, true>), grid, dim3(256), 0, s, of_parts, plan);
      else hipLaunchKernelGGL((grouped_double_kernel<32, false>), grid, dim3(256), 0, s, of_parts, plan);
    });
    add_up<false>(s, parts, g);
    note_kernel(parts.count() > 1 ? "grouped_double+grouped_sum" : "grouped_double");
    return after_launch(s);
  }
  if (dtype == CT_F32 && a_row_count > 0 && a_col_count > 0) {
    // The tiles that there are if the groups are even, and the kernel that takes them soonest.  With 4096 by 1024 [n][k] and 8 groups,
    // us with 16 columns to a block, 64, and tiles of 64 and 128 a side: of one row 28, 34, 88 and 151; of 32 rows 60, 40, 88 and 153; of
    // 128 rows 228, 145, 89 and 150; with 32 groups of 128 rows 910, 568, 286 and 217.
    const int64_t k_tiles = ceil_div(a_col_count, kTileDepth);
    const double thin64 = time_of_thin64(row_tiles_of(16) * ceil_div(b_col_count, 64), k_tiles);
    const double thin16 = time_of_thin16(row_tiles_of(16) * ceil_div(b_col_count, 16), k_tiles);
    auto choose = [&](int64_t most_parts) {
      Choice best{16, thin16 < thin64 ? 16 : 64, 1, std::min(thin64, thin16)};
      if (a_col_count >= kTileDepth && b_colstride <= kMostSplitLd) consider_parts(&best, blocks_of(64), blocks_of(128), k_tiles, cells, most_parts);
      return best;
    };
    Choice best = choose(kMostParts);
    const Parts<float> parts(s, best.parts, cells);
    if (parts.count() < best.parts) best = choose(1);
    const bool thin = best.height == 16;
    const int64_t m_tiles = row_count / best.height + even_groups, n_tiles = ceil_div(b_col_count, best.width);
    CT_REQUIRE(m_tiles <= kMostTiles / parts.count() / n_tiles, "ct_grouped_gemm: %lld rows of %lld columns", (long long)row_count, (long long)b_col_count);
    GroupedArgs of_parts = parts.args(g, 0);
    of_parts.part = (uint32_t)(tiles_of_part(k_tiles, parts.count()) * kTileDepth);
    auto launch = [&](auto of_b, auto of_not_b, int waves) {
      for_launches(m_tiles, n_tiles, parts.count(), [&](dim3 grid, const GroupedPlan& plan) {
        if (trans_b) hipLaunchKernelGGL(of_b, grid, dim3(64 * waves), 0, s, of_parts, plan);
        else hipLaunchKernelGGL(of_not_b, grid, dim3(64 * waves), 0, s, of_parts, plan);
      });
    };
    const bool few = a_col_count <= kFewK;
    if (thin && best.width == 64 && few) launch(grouped_thin_kernel<4, 4, true>, grouped_thin_kernel<4, 4, false>, 4);
    else if (thin && best.width == 64) launch(grouped_thin_kernel<8, 4, true>, grouped_thin_kernel<8, 4, false>, 8);
    else if (thin && few) launch(grouped_thin_kernel<4, 1, true>, grouped_thin_kernel<4, 1, false>, 4);
    else if (thin) launch(grouped_thin_kernel<16, 1, true>, grouped_thin_kernel<16, 1, false>, 16);
    else if (best.height == 128) launch(grouped_split_kernel<128, 128, 2, 4, true>, grouped_split_kernel<128, 128, 2, 4, false>, 8);
    else launch(grouped_split_kernel<64, 64, 2, 2, true>, grouped_split_kernel<64, 64, 2, 2, false>, 4);
    add_up<false>(s, parts, g);
    static const char* const kNames[] = {"grouped_medium", "grouped_large", "grouped_medium+grouped_sum", "grouped_large+grouped_sum"};
    note_kernel(thin ? "grouped_thin" : kNames[(best.height == 128) + 2 * (parts.count() > 1)]);
    return after_launch(s);
  }
  const dim3 grid = plain_grid(b_col_count, row_count / kSide + std::min(n_groups, row_count), 1);
  if (dtype == CT_F32) hipLaunchKernelGGL((grouped_kernel<float>), grid, dim3(256), 0, s, g);
  else hipLaunchKernelGGL((grouped_kernel<double>), grid, dim3(256), 0, s, g);
  note_kernel("grouped");
  return after_launch(s);
}

int ct_grouped_gemm_weights(void* stream, void* c, int64_t c_colstride, int64_t c_stride, double alpha, const void* a,
                            int64_t a_row_count, int64_t a_col_count, int64_t a_colstride, const int32_t* a_index,
                            const void* b, int64_t b_row_count, int64_t b_col_count, int64_t b_colstride,
                            const int32_t* b_index, const int32_t* offsets, int64_t n_groups, int64_t row_count, double beta,
                            int dtype) {
  CT_GROUPED_FLOATING("ct_grouped_gemm_weights");
  CT_REQUIRE(extent(a_row_count) && extent(a_col_count) && extent(b_row_count) && extent(b_col_count) && extent(row_count),
             "ct_grouped_gemm_weights: bad extent");
  CT_REQUIRE(n_groups >= 0 && n_groups <= kMostGroups, "ct_grouped_gemm_weights: %lld groups, at most %lld are taken",
             (long long)n_groups, (long long)kMostGroups);
  if (n_groups == 0 || a_col_count == 0 || b_col_count == 0) return CT_OK;
  CT_REQUIRE(c && offsets && (row_count == 0 || ((a || a_row_count == 0) && (b || b_row_count == 0))), "ct_grouped_gemm_weights: null buffer");
  CT_REQUIRE((a_index || a_row_count >= row_count) && (b_index || b_row_count >= row_count),
             "ct_grouped_gemm_weights: an operand has fewer rows than %lld", (long long)row_count);
  CT_REQUIRE(c_colstride >= b_col_count && a_colstride >= a_col_count && b_colstride >= b_col_count,
             "ct_grouped_gemm_weights: a column stride below the row's length");
  CT_REQUIRE(n_groups == 1 || c_stride >= (a_col_count - 1) * c_colstride + b_col_count, "ct_grouped_gemm_weights: results overlap one another");
  const int64_t size = dtype_size(dtype);
  const Run result{c, ((n_groups - 1) * c_stride + (a_col_count - 1) * c_colstride + b_col_count) * size};
  CT_REQUIRE(!run_meets(result, {a, a_row_count, a_col_count, a_colstride}, size) && !run_meets(result, {b, b_row_count, b_col_count, b_colstride}, size),
             "ct_grouped_gemm_weights: c overlaps an operand");
  CT_REQUIRE(!runs_meet(result, {offsets, (n_groups + 1) * 4}) && !runs_meet(result, {a_index, row_count * 4}) && !runs_meet(result, {b_index, row_count * 4}),
             "ct_grouped_gemm_weights: c overlaps the offsets or an index");
  hipStream_t s = static_cast<hipStream_t>(stream);
  GroupedArgs g{};
  g.a = a; g.b = b; g.c = c; g.index_a = a_index; g.index_b = b_index; g.offsets = offsets;
  g.lda = a_colstride; g.ldb = b_colstride; g.ldc = c_colstride; g.c_stride = c_stride;
  g.alpha = alpha; g.beta = beta;
  g.groups = (uint32_t)n_groups; g.rows = (uint32_t)row_count; g.a_rows = (uint32_t)a_row_count; g.b_rows = (uint32_t)b_row_count;
  g.m = (uint32_t)a_col_count; g.n = (uint32_t)b_col_count;
  const int64_t cells = n_groups * a_col_count * b_col_count, mean = std::max<int64_t>(row_count / n_groups, 1);
  auto blocks_of = [&](int64_t side) { return n_groups * ceil_div(a_col_count, side) * ceil_div(b_col_count, side); };
  if (dtype == CT_F32 && std::max(a_colstride, b_colstride) <= kMostWeightsLd) {
    auto choose = [&](int64_t most_parts) {
      Choice best{0, 0, 1, 1e12};
      consider_parts(&best, blocks_of(64), blocks_of(128), ceil_div(mean, kTileDepth), cells, most_parts);
      return best;
    };
    Choice best = choose(kMostParts);
    const Parts<float> parts(s, best.parts, cells);
    if (parts.count() < best.parts) best = choose(1);
    const int64_t m_tiles = n_groups * ceil_div(a_col_count, best.height), n_tiles = ceil_div(b_col_count, best.width);
    CT_REQUIRE(m_tiles <= kMostTiles / parts.count() / n_tiles, "ct_grouped_gemm_weights: %lld by %lld results of %lld groups", (long long)a_col_count,
               (long long)b_col_count, (long long)n_groups);
    const GroupedArgs of_parts = parts.args(g, a_col_count);
    const bool wide = std::max(a_row_count * a_colstride, b_row_count * b_colstride) * size >= int64_t(1) << 32, large = best.height == 128;
    for_launches(m_tiles, n_tiles, parts.count(), [&](dim3 grid, const GroupedPlan& plan) {
      if (large && !wide) hipLaunchKernelGGL((grouped_weights_split_kernel<128, 128, 2, 4, false>), grid, dim3(512), 0, s, of_parts, plan);
      else if (large) hipLaunchKernelGGL((grouped_weights_split_kernel<128, 128, 2, 4, true>), grid, dim3(512), 0, s, of_parts, plan);
      else if (!wide) hipLaunchKernelGGL((grouped_weights_split_kernel<64, 64, 2, 2, false>), grid, dim3(256), 0, s, of_parts, plan);
      else hipLaunchKernelGGL((grouped_weights_split_kernel<64, 64, 2, 2, true>), grid, dim3(256), 0, s, of_parts, plan);
    });
    add_up<true>(s, parts, g);
    static const char* const kNames[] = {"grouped_weights_medium", "grouped_weights_large", "grouped_weights_medium+grouped_sum", "grouped_weights_large+grouped_sum"};
    note_kernel(kNames[large + 2 * (parts.count() > 1)]);
    return after_launch(s);
  }
  if (dtype == CT_F64) {
    auto choose = [&](int64_t most_parts) {
      Choice best{32, 32, 1, 1e12};
      consider_double_parts(&best, blocks_of(32), blocks_of(64), mean, 2 * mean, cells, most_parts);
      return best;
    };
    Choice best = choose(kMostParts);
    const Parts<double> parts(s, best.parts, cells);
    if (parts.count() < best.parts) best = choose(1);
    const int64_t side = best.height, m_tiles = n_groups * ceil_div(a_col_count, side), n_tiles = ceil_div(b_col_count, side);
    CT_REQUIRE(m_tiles <= kMostTiles / parts.count() / n_tiles, "ct_grouped_gemm_weights: %lld by %lld results of %lld groups", (long long)a_col_count,
               (long long)b_col_count, (long long)n_groups);
    const GroupedArgs of_parts = parts.args(g, a_col_count);
    for_launches(m_tiles, n_tiles, parts.count(), [&](dim3 grid, const GroupedPlan& plan) {
      if (side == 64) hipLaunchKernelGGL((grouped_weights_double_kernel<64>), grid, dim3(256), 0, s, of_parts, plan);
      else hipLaunchKernelGGL((grouped_weights_double_kernel<32>), grid, dim3(256), 0, s, of_parts, plan);
    });
    add_up<true>(s, parts, g);
    note_kernel(parts.count() > 1 ? "grouped_weights_double+grouped_sum" : "grouped_weights_double");
    return after_launch(s);
  }
  hipLaunchKernelGGL(grouped_weights_kernel, plain_grid(b_col_count, ceil_div(a_col_count, kSide), n_groups), dim3(256), 0, s, g);
  note_kernel("grouped_weights");
  return after_launch(s);
}

}  // extern "C"
