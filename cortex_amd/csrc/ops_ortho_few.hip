// ops_ortho_few.hip -- float matrices of up to 64 rows (or columns) made orthogonal in three launches.
//
// With X X^T = A, which is small here, a step X' = B X, B = a I + b A + c A A, makes A' = B A B: after A the steps need X no more, and what
// they come to is a matrix Q, the product of all B, by which X is multiplied in the end.  A matrix is read twice, once for A and once
// for Q X, where the steps as they are written read and write it once each.
//
// In A a singular value is squared, and a step multiplies a small one by a: what A is off by grows by a^2, 2.3e5 times in five of the
// usual steps.  So A, the steps and Q X are in double, and coefficients and steps by which it would grow to a float's last bit
// are not taken here (kMostFewChange).  For matrices of doubles there is no such wider type, and none of this.
//
// Bound by latency: 4 x 9 takes 17 us, 64 x 64 54, 64 x 8000 74 (65 x 65, in the products of halves, 81).  Of 64 rows 40 us are the steps,
// which one unit makes.  The products are v_mfma_f64_16x16x4_f64: of a lane's operands the row (or column) is lane % 16 and k lane / 16, of
// its results the rows lane / 16 + 4 r and the column lane % 16.
#include <algorithm>

#include "common.h"
#include "ortho.h"

using namespace cthip;

namespace {

typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kSide = 64, kPitch = kSide + 1;   // of tiles in LDS
constexpr int kMostSteps = 64;

struct FewArgs {
  StartArgs start;
  char* workspace;
  int64_t workspace_stride, ldo, out_stride;
  float* out;
  float alpha, beta;
  uint32_t m, n, blocks, parts, each;   // blocks: of 16 rows; each: columns of a part
  int steps;
  double coefficients[kMostSteps][3];
};

__host__ __device__ inline uint32_t pairs_of(uint32_t blocks) { return blocks * (blocks + 1) / 2; }

// [part][pair of blocks of rows][16][16], and behind them Q / (|X| + epsilon).
__device__ __forceinline__ double* sums_of(const FewArgs& a, uint32_t matrix) { return reinterpret_cast<double*>(a.workspace + matrix * a.workspace_stride); }
__device__ __forceinline__ double* factor_of(const FewArgs& a, uint32_t matrix) { return sums_of(a, matrix) + a.parts * pairs_of(a.blocks) * 256; }

// Of `depth` k, a multiple of 16.
__device__ __forceinline__ f64x4 product16(const double* l, uint32_t l_row, uint32_t l_k, const double* r, uint32_t r_column, uint32_t r_k, uint32_t depth, f64x4 sum) {
  const uint32_t lane = threadIdx.x & 63;
  l += lane % 16 * l_row + lane / 16 * l_k;
  r += lane % 16 * r_column + lane / 16 * r_k;
#pragma unroll 1
  for (uint32_t k0 = 0; k0 < depth; k0 += 16) {
    double x[4], y[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      x[i] = l[(k0 + 4 * i) * l_k];
      y[i] = r[(k0 + 4 * i) * r_k];
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f64_16x16x4f64(x[i], y[i], sum, 0, 0, 0);
  }
  return sum;
}

// Element (r, c) of the matrix on its shorter side: r of m, c of n.
template <bool kTall> __device__ __forceinline__ int64_t place(const FewArgs& a, uint32_t matrix, uint32_t r, uint32_t c) {
  return (int64_t)matrix * a.start.stride + (kTall ? (int64_t)c * a.start.ld + r : (int64_t)r * a.start.ld + c);
}

// A lane's elements of 64 columns from c0 on: e of 16, of row r and column c.
template <bool kTall> __device__ __forceinline__ uint32_t row_of(uint32_t e) { return kTall ? threadIdx.x % 64 : e * 4 + threadIdx.x / 64; }
template <bool kTall> __device__ __forceinline__ uint32_t column_of(uint32_t e) { return kTall ? e * 4 + threadIdx.x / 64 : threadIdx.x % 64; }

struct Pair {
  uint32_t row, column;
};
__device__ __forceinline__ Pair pair_at(uint32_t pair) {
  const uint32_t row = pair >= 6 ? 3 : pair >= 3 ? 2 : pair >= 1 ? 1 : 0;
  return {row * 16, (pair - row * (row + 1) / 2) * 16};
}

// The sums of products of pairs of rows over a part of the columns; of a step, the momentum before them.
template <bool kTall, bool kStep>
__global__ void __launch_bounds__(256) few_gram_kernel(const FewArgs a) {
  __shared__ double tile[kSide * kPitch];
  const uint32_t matrix = blockIdx.y, first = blockIdx.x * a.each, end = min(first + a.each, a.n), wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const float* x = static_cast<const float*>(a.start.x);
  const float* gradient = static_cast<const float*>(a.start.gradient);
  float v[16], g[16];
  auto load = [&](uint32_t c0) {   // what is outside repeats the last ones
#pragma unroll
    for (uint32_t e = 0; e < 16; ++e) {
      const int64_t at = place<kTall>(a, matrix, min(row_of<kTall>(e), a.m - 1), min(c0 + column_of<kTall>(e), a.n - 1));
      v[e] = x[at];
      if constexpr (kStep) g[e] = gradient[at];
    }
  };
  f64x4 sums[3] = {};
  const uint32_t pairs = pairs_of(a.blocks);
  load(first);
  for (uint32_t c0 = first; c0 < end; c0 += 64) {
#pragma unroll
    for (uint32_t e = 0; e < 16; ++e) {
      const uint32_t r = row_of<kTall>(e), c = column_of<kTall>(e);
      const bool inside = r < a.m && c0 + c < end;
      float value = v[e];
      if constexpr (kStep) {
        const float step = (float)a.start.gradient_alpha * g[e];
        value = (float)a.start.decay * value + step;
        if (inside) static_cast<float*>(a.start.momentum)[place<kTall>(a, matrix, r, c0 + c)] = value;
        if (a.start.nesterov) value = step + (float)a.start.decay * value;
      }
      tile[r * kPitch + c] = inside ? (double)value : 0.0;
    }
    __syncthreads();
    if (c0 + 64 < end) load(c0 + 64);
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i) {
      const uint32_t pair = i * 4 + wave;
      if (pair >= pairs) break;
      const Pair at = pair_at(pair);
      sums[i] = product16(tile + at.row * kPitch, kPitch, 1, tile + at.column * kPitch, kPitch, 1, 64, sums[i]);
    }
    __syncthreads();
  }
  double* to = sums_of(a, matrix) + (int64_t)blockIdx.x * pairs * 256;
#pragma unroll
  for (uint32_t i = 0; i < 3; ++i) {
    if (i * 4 + wave >= pairs) continue;
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) to[(i * 4 + wave) * 256 + (lane / 16 + 4 * r) * 16 + lane % 16] = sums[i][r];
  }
}

// The steps of a matrix.  All that is multiplied here is a polynomial of A, and so is the product: symmetric, 16 x 16 at and below the
// diagonal are formed, to a wave each, and stored twice.  64 x 64 in 0.3 TFLOP/s of a unit's matrix cores are 1.1 us a product.
__global__ void __launch_bounds__(1024) few_steps_kernel(const FewArgs a) {
  __shared__ double gram[kSide * kPitch], factor[kSide * kPitch], total[kSide * kPitch], other[kSide * kPitch];
  __shared__ double inverse;
  const uint32_t matrix = blockIdx.x, wave = threadIdx.x / 64, lane = threadIdx.x % 64, pairs = pairs_of(a.blocks), side = a.blocks * 16;
  const double* sums = sums_of(a, matrix);
  for (uint32_t i = threadIdx.x; i < pairs * 256; i += 1024) {
    double sum = 0.0;
    for (uint32_t part0 = 0; part0 < a.parts; part0 += 8) {   // loads of eight parts on their way
      double y[8];
#pragma unroll
      for (uint32_t p = 0; p < 8; ++p) y[p] = sums[(int64_t)min(part0 + p, a.parts - 1) * pairs * 256 + i];
#pragma unroll
      for (uint32_t p = 0; p < 8; ++p) sum += part0 + p < a.parts ? y[p] : 0.0;
    }
    const Pair at = pair_at(i / 256);
    const uint32_t r = at.row + i / 16 % 16, c = at.column + i % 16;
    gram[r * kPitch + c] = sum;
    if (at.row != at.column) gram[c * kPitch + r] = sum;
  }
  __syncthreads();
  if (wave == 0) {
    double squares = lane < a.m ? gram[lane * kPitch + lane] : 0.0;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) squares += __shfl_xor(squares, d);
    if (lane == 0) inverse = 1.0 / (sqrt(squares) + a.start.epsilon);
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < side * side; i += 1024) gram[i / side * kPitch + i % side] = gram[i / side * kPitch + i % side] * inverse * inverse;
  __syncthreads();
  auto product = [&](Pair at, const double* l, const double* r) {
    return product16(l + at.row * kPitch, kPitch, 1, r + at.column * kPitch, kPitch, 1, side, f64x4{});
  };
  auto store = [&](Pair at, double* to, f64x4 x) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t r = at.row + lane / 16 + 4 * i, c = at.column + lane % 16;
      if (r < c) continue;   // above the diagonal it is what is below
      to[r * kPitch + c] = x[i];
      to[c * kPitch + r] = x[i];
    }
  };
  for (int step = 0; step < a.steps; ++step) {
    const double* k = a.coefficients[step];
    const bool more = step + 1 < a.steps;
    if (wave < pairs) {
      const Pair at = pair_at(wave);
      f64x4 x = product(at, gram, gram);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t r = at.row + lane / 16 + 4 * i, c = at.column + lane % 16;
        x[i] = k[2] * x[i] + k[1] * gram[r * kPitch + c] + (r == c ? k[0] : 0.0);
      }
      store(at, factor, x);
      if (step == 0) store(at, total, x);
    }
    __syncthreads();
    // B Q and B A, of which a wave may have two
    f64x4 found[2];
    const uint32_t of_total = step > 0 ? pairs : 0, tasks = of_total + (more ? pairs : 0);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t task = i * 16 + wave;
      if (task < tasks) found[i] = task < of_total ? product(pair_at(task), factor, total) : product(pair_at(task - of_total), factor, gram);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      const uint32_t task = i * 16 + wave;
      if (task < tasks) store(pair_at(task < of_total ? task : task - of_total), task < of_total ? total : other, found[i]);
    }
    __syncthreads();
    if (!more) break;
    if (wave < pairs) store(pair_at(wave), gram, product(pair_at(wave), other, factor));
    __syncthreads();
  }
  double* to = factor_of(a, matrix);
  for (uint32_t i = threadIdx.x; i < side * side; i += 1024) to[i] = total[i / side * kPitch + i % side] * inverse;
}

// Q X of 64 columns.
template <bool kTall>
__global__ void __launch_bounds__(256) few_apply_kernel(const FewArgs a) {
  __shared__ double tile[kSide * kPitch], factor[kSide * kPitch];
  const uint32_t matrix = blockIdx.y, c0 = blockIdx.x * 64, wave = threadIdx.x / 64, lane = threadIdx.x % 64, side = a.blocks * 16;
  float v[16];
#pragma unroll
  for (uint32_t e = 0; e < 16; ++e)
    v[e] = start_value<float>(a.start, place<kTall>(a, matrix, min(row_of<kTall>(e), a.m - 1), min(c0 + column_of<kTall>(e), a.n - 1)));
  const double* q = factor_of(a, matrix);
  for (uint32_t i = threadIdx.x; i < side * side; i += 256) factor[i / side * kPitch + i % side] = q[i];
#pragma unroll
  for (uint32_t e = 0; e < 16; ++e) {
    const uint32_t r = row_of<kTall>(e), c = column_of<kTall>(e);
    tile[r * kPitch + c] = r < a.m && c0 + c < a.n ? (double)v[e] : 0.0;
  }
  __syncthreads();
  float* out = a.out + matrix * a.out_stride;
  for (uint32_t block = 0; block < a.blocks; ++block) {
    // 16 of the shorter side by 16 of the columns, as they lie in the result
    const f64x4 sum = kTall ? product16(tile + wave * 16, 1, kPitch, factor + block * 16 * kPitch, kPitch, 1, side, f64x4{})
                            : product16(factor + block * 16 * kPitch, kPitch, 1, tile + wave * 16, 1, kPitch, side, f64x4{});
    float before[4];
    int64_t at[4];
    bool inside[4];
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) {
      const uint32_t i = lane / 16 + 4 * r, j = lane % 16;   // of the product
      const uint32_t shorter = block * 16 + (kTall ? j : i), longer = c0 + wave * 16 + (kTall ? i : j);
      inside[r] = shorter < a.m && longer < a.n;
      at[r] = kTall ? (int64_t)longer * a.ldo + shorter : (int64_t)shorter * a.ldo + longer;
      before[r] = a.beta != 0.f && inside[r] ? out[at[r]] : 0.f;
    }
#pragma unroll
    for (uint32_t r = 0; r < 4; ++r) {
      const float value = a.alpha * (float)sum[r];
      if (inside[r]) out[at[r]] = a.beta == 0.f ? value : value + a.beta * before[r];
    }
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// So many that neither a part's columns nor the sum of the parts, which one block forms, takes long.
int64_t parts_of(int64_t n) { return std::min<int64_t>(32, ceil_div(n, 128)); }

}  // namespace

namespace cthip {

int64_t few_bytes(int64_t m, int64_t n) {
  const int64_t blocks = ceil_div(m, 16);
  return (parts_of(n) * pairs_of((uint32_t)blocks) + blocks * blocks) * 256 * 8;
}

void ortho_few(hipStream_t s, const FewMatrices& f, int64_t count) {
  FewArgs a{};
  const bool tall = f.start.rows > f.start.columns;
  a.start = f.start;
  a.workspace = f.workspace;
  a.workspace_stride = f.workspace_stride;
  a.out = f.out;
  a.ldo = f.ldo;
  a.out_stride = f.out_stride;
  a.alpha = f.alpha;
  a.beta = f.beta;
  a.m = std::min(f.start.rows, f.start.columns);
  a.n = std::max(f.start.rows, f.start.columns);
  a.blocks = (uint32_t)ceil_div(a.m, 16);
  a.parts = (uint32_t)parts_of(a.n);
  a.each = (uint32_t)(ceil_div(ceil_div(a.n, a.parts), 64) * 64);
  a.parts = (uint32_t)ceil_div(a.n, a.each);
  a.steps = f.steps;
  for (int step = 0; step < f.steps; ++step)
    for (int i = 0; i < 3; ++i) a.coefficients[step][i] = f.coefficients[3 * step + i];
  const dim3 of_parts(a.parts, (uint32_t)count), of_columns((uint32_t)ceil_div(a.n, 64), (uint32_t)count);
  const bool step = f.start.gradient != nullptr;
  if (tall && step) hipLaunchKernelGGL((few_gram_kernel<true, true>), of_parts, dim3(256), 0, s, a);
  else if (tall) hipLaunchKernelGGL((few_gram_kernel<true, false>), of_parts, dim3(256), 0, s, a);
  else if (step) hipLaunchKernelGGL((few_gram_kernel<false, true>), of_parts, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((few_gram_kernel<false, false>), of_parts, dim3(256), 0, s, a);
  hipLaunchKernelGGL(few_steps_kernel, dim3((uint32_t)count), dim3(1024), 0, s, a);
  if (tall) hipLaunchKernelGGL((few_apply_kernel<true>), of_columns, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((few_apply_kernel<false>), of_columns, dim3(256), 0, s, a);
}

}  // namespace cthip
