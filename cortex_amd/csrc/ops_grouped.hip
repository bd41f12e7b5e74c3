// ops_grouped.hip -- products of rows with the matrix of their group (ct_grouped_gemm), and the products over the rows of
// each group that are those matrices' gradients (ct_grouped_gemm_weights).
//
// Groups are runs of rows between offsets in device memory.  A launch has as many blocks as the tiles can be at most: the
// tiles of all rows and one more to each group.  A block finds its group by adding up the groups' tiles; blocks beyond the
// last tile end.  Offsets are clamped as they are read, so that no content of theirs leads outside a buffer.
#include <algorithm>

#include "common.h"
#include "rows.h"

using namespace cthip;

namespace {

struct GroupedArgs {
  const void* a;
  const void* b;
  void* c;
  const int32_t* index_a;
  const int32_t* index_b;
  const int32_t* offsets;
  int64_t lda, ldb, ldc, b_stride, c_stride;
  double alpha, beta;
  uint32_t groups, rows, a_rows, b_rows, m, n, k;   // m, k: of the weights' products only where rows are not
  bool trans_b;
};

struct Group {
  uint32_t index, first, rows, tile;
};

__device__ __forceinline__ uint2 group_rows(const GroupedArgs& a, uint32_t g) {
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

template <class T>
__device__ __forceinline__ void put(T* cell, T sum, double alpha, double beta) {
  const T value = (T)alpha * sum;
  *cell = beta == 0 ? value : value + (T)beta * *cell;
}

template <class T>
__global__ void __launch_bounds__(256) grouped_kernel(const GroupedArgs a) {
  Group g;
  if (!find_group(a, blockIdx.y, kSide, &g)) return;
  const uint32_t row0 = g.tile * kSide, col0 = blockIdx.x * kSide;
  const T* b = static_cast<const T*>(a.b) + (int64_t)g.index * a.b_stride;
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

template <class T>
__global__ void __launch_bounds__(256) grouped_weights_kernel(const GroupedArgs a) {
  const uint32_t group = blockIdx.z, row0 = blockIdx.y * kSide, col0 = blockIdx.x * kSide;
  const uint2 rows = group_rows(a, group);
  T* c = static_cast<T*>(a.c) + (int64_t)group * a.c_stride;
  auto element = [&](const void* p, const int32_t* index, uint32_t count, int64_t ld, uint32_t k, uint32_t column, uint32_t width) -> T {
    if (k >= rows.y || column >= width) return 0;
    const uint32_t i = rows.x + k, from = index ? (uint32_t)index[i] : i;
    return from < count ? static_cast<const T*>(p)[(int64_t)from * ld + column] : T(0);
  };
  tile_product<T>(
      rows.y, [&](uint32_t r, uint32_t k) { return element(a.a, a.index_a, a.a_rows, a.lda, k, row0 + r, a.m); },
      [&](uint32_t k, uint32_t n) { return element(a.b, a.index_b, a.b_rows, a.ldb, k, col0 + n, a.n); },
      [&](uint32_t r, uint32_t n, T sum) {
        if (row0 + r < a.m && col0 + n < a.n) put(c + (int64_t)(row0 + r) * a.ldc + col0 + n, sum, a.alpha, a.beta);
      });
}

uint32_t tiles_of(int64_t n, int64_t side) { return (uint32_t)((n + side - 1) / side); }

constexpr int64_t kMostExtent = (int64_t(1) << 31) - 1;
bool extent(int64_t n) { return n >= 0 && n <= kMostExtent; }
constexpr int64_t kMostGroups = 65535;

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
                 !rows_meet(result, {a_col_count ? b : nullptr, 1, (n_groups - 1) * b_stride + (b_rows - 1) * b_colstride + b_cols, 1}, size),
             "ct_grouped_gemm: c overlaps an operand");
  hipStream_t s = static_cast<hipStream_t>(stream);
  GroupedArgs g{};
  g.a = a; g.b = b; g.c = c; g.index_a = index; g.offsets = offsets;
  g.lda = a_colstride; g.ldb = b_colstride; g.ldc = c_colstride; g.b_stride = b_stride;
  g.alpha = alpha; g.beta = beta;
  g.groups = (uint32_t)n_groups; g.rows = (uint32_t)row_count; g.a_rows = (uint32_t)a_row_count;
  g.n = (uint32_t)b_col_count; g.k = (uint32_t)a_col_count;
  g.trans_b = trans_b != 0;
  const int64_t tiles = row_count / kSide + std::min(n_groups, row_count);
  CT_REQUIRE(tiles <= 65535, "ct_grouped_gemm: %lld rows", (long long)row_count);
  const dim3 grid(tiles_of(b_col_count, kSide), (uint32_t)tiles);
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
  const RowRange result{c, 1, (n_groups - 1) * c_stride + (a_col_count - 1) * c_colstride + b_col_count, 1};
  CT_REQUIRE(!rows_meet(result, {a, a_row_count, a_col_count, a_colstride}, size) && !rows_meet(result, {b, b_row_count, b_col_count, b_colstride}, size),
             "ct_grouped_gemm_weights: c overlaps an operand");
  hipStream_t s = static_cast<hipStream_t>(stream);
  GroupedArgs g{};
  g.a = a; g.b = b; g.c = c; g.index_a = a_index; g.index_b = b_index; g.offsets = offsets;
  g.lda = a_colstride; g.ldb = b_colstride; g.ldc = c_colstride; g.c_stride = c_stride;
  g.alpha = alpha; g.beta = beta;
  g.groups = (uint32_t)n_groups; g.rows = (uint32_t)row_count; g.a_rows = (uint32_t)a_row_count; g.b_rows = (uint32_t)b_row_count;
  g.m = (uint32_t)a_col_count; g.n = (uint32_t)b_col_count;
  CT_REQUIRE(tiles_of(a_col_count, kSide) <= 65535, "ct_grouped_gemm_weights: %lld columns of a", (long long)a_col_count);
  const dim3 grid(tiles_of(b_col_count, kSide), tiles_of(a_col_count, kSide), (uint32_t)n_groups);
  if (dtype == CT_F32) hipLaunchKernelGGL((grouped_weights_kernel<float>), grid, dim3(256), 0, s, g);
  else hipLaunchKernelGGL((grouped_weights_kernel<double>), grid, dim3(256), 0, s, g);
  note_kernel("grouped_weights");
  return after_launch(s);
}

}  // extern "C"
