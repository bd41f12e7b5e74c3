// ops_norm.hip -- the norms after a block and before the next one, fused with the block's gate and residual
// (ct_norm_residual), and their gradients.
//
// Forward, for a row z of the block and r of the residual:  zh = (z - m) s,  u = zh wp + bp,  out = c r + g u,
// oh = (out - m') s',  h = oh wn + bn, s = 1 / sqrt(mean of (z - m)^2 + epsilon), m the mean or 0.
// Backward, from dout and dh:  with the norm's transpose N^T(y) = s (y - [mean(y)] - xh mean(y xh)),
//   d = dout + N'^T(dh wn),  dr = c d,  dg = d u,  du = d g,  dz = N^T(du wp),
// and sums over the rows: S1 of du zh, S0 of du, T1 of dh oh, T0 of dh: the gradients of wp, bp, wn, bn.  A gate that is the
// same for all rows is taken out of S1 and S0: its own gradient is wp S1 + bp S0, and wp's is g S1.
//
// A row is held in registers by LANES lanes, VPT pieces of 16 bytes to each, so that every operand is read once and every
// result written once.  Rows that do not fit (more than 16384 floats), and those shorter than a piece, take the kernels at
// the end, which read again.  Memory bounds it: 16384 x 2048 floats, two root-mean-square norms and a column gate, 94 us (5.7 TB/s) and 151 of
// the gradient (5.3), where a copy of 2 GiB reaches 4.9.
#include <algorithm>
#include <cmath>

#include "elementwise.h"
#include "rows.h"

using namespace cthip;

namespace {

constexpr int kNormBlock = 256;
// Lanes of a block: rows of a wave or less share one, others have one to themselves.
constexpr int block_of(int lanes) { return lanes > 64 ? lanes : kNormBlock; }

enum GateKind { kNoGate, kScalarGate, kColumnGate, kRowGate, kFullGate };

struct Matrix {
  void* p;
  int64_t ld;
};

struct NormArgs {
  Matrix output, normalized, input, residual, gate;   // ld of the gate: of a full one
  const void *post_scale, *post_bias, *pre_scale, *pre_bias;
  void* statistics;
  int64_t rows;
  uint32_t width;
  int post, pre, gate_kind;
  double residual_scale, epsilon;
};

template <class T> __device__ __forceinline__ const T* row_of(const Matrix& m, int64_t row) { return static_cast<const T*>(m.p) + row * m.ld; }
template <class T> __device__ __forceinline__ T* row_to(const Matrix& m, int64_t row) { return static_cast<T*>(m.p) + row * m.ld; }

// The lanes that hold a row of N elements or more, and what each of them holds: VPT pieces of N elements.  Piece t belongs at
// element N * (lane + t * LANES); one that would pass the end of the row is the row's last N elements instead, of which the
// lane owns what lies behind its place, perhaps nothing.  So loads have no branches, and none is waited for before the next.
template <class T, int LANES, int VPT, bool kStreaming>
struct Row {
  static constexpr int N = Quad<T>::N, E = N * VPT;
  uint32_t lane, width;
  __device__ __forceinline__ uint32_t place(int t) const { return N * (lane + t * LANES); }
  __device__ __forceinline__ uint32_t start(int t) const { return min(place(t), width - N); }
  __device__ __forceinline__ bool owns(int t, int e) const { return start(t) + e >= place(t); }
  __device__ __forceinline__ Quad<T> piece(const T* p, int t) const { return load_quad(p + start(t)); }
  // of an operand that may be absent: `fill` then
  __device__ __forceinline__ Quad<T> piece_or(const void* p, T fill, int t) const {
    Quad<T> q;
    if (p) return piece(static_cast<const T*>(p), t);
#pragma unroll
    for (int e = 0; e < N; ++e) q.v[e] = fill;
    return q;
  }
  __device__ __forceinline__ void load(const T* p, Quad<T> (&x)[VPT]) const {
#pragma unroll
    for (int t = 0; t < VPT; ++t) x[t] = load_quad<kStreaming>(p + start(t));
  }
  __device__ __forceinline__ T owned(int t, int e, T x) const { return owns(t, e) ? x : T(0); }
  __device__ __forceinline__ void store(T* p, int t, const Quad<T>& q) const {
    if (place(t) + N <= width) {
      store_quad<kStreaming>(p + place(t), q);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (owns(t, e)) p[start(t) + e] = q.v[e];
    }
  }
};

#define CT_EACH                        \
  _Pragma("unroll") for (int t = 0; t < VPT; ++t) _Pragma("unroll") for (int e = 0; e < N; ++e)

// Sums of K values over the LANES lanes of a row, in all of them.  A row of more than a wave is a whole block's; `lds` holds
// K values to a wave, twice, used in turn so that one barrier a call is enough.
template <class T, int LANES, int K>
__device__ __forceinline__ void row_sum(T (&v)[K], T* lds, int& turn) {
#pragma unroll
  for (int m = (LANES < 64 ? LANES : 64) / 2; m > 0; m >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], m);
  if constexpr (LANES > 64) {
    constexpr int W = LANES / 64;
    T* mine = lds + turn * (3 * W);
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) mine[k * W + threadIdx.x / 64] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = mine[k * W];
#pragma unroll
      for (int w = 1; w < W; ++w) v[k] += mine[k * W + w];
    }
  }
}

template <class T> __device__ __forceinline__ T rate_of(T mean_square, T epsilon) { return T(1) / (T)sqrt(mean_square + epsilon); }

template <class T, int LANES, int VPT, bool kStreaming>
__global__ void __launch_bounds__(block_of(LANES)) norm_kernel(const NormArgs a) {
  constexpr int kThreads = block_of(LANES), kRows = kThreads / LANES;
  using R = Row<T, LANES, VPT, kStreaming>;
  constexpr int N = R::N;
  __shared__ T lds[LANES > 64 ? 2 * 3 * (LANES / 64) : 1];
  int turn = 0;
  const R at{threadIdx.x % LANES, a.width};
  const T inverse = T(1) / (T)a.width, epsilon = (T)a.epsilon;
  for (int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES; row < a.rows; row += (int64_t)gridDim.x * kRows) {
    Quad<T> x[VPT], y[VPT];
    at.load(row_of<T>(a.input, row), x);
    at.load(row_of<T>(a.residual.p ? a.residual : a.input, row), y);
    // the norm of x in place, its statistics to `place`
    auto norm = [&](int kind, const void* scale, const void* bias, int place) {
      T mean[1] = {0}, square[1] = {0};
      // The parameters are on their way while the sums are formed: rows of 256, layer norms before and after, 43 us a 65536, were 61; of
      // 1531 doubles 45 us a 5003, were 51.  Not with 1024 lanes, which have no registers for them (rows of 16384 134 us, and 97 so).
      constexpr bool kAhead = LANES <= 256;
      Quad<T> w_ahead[kAhead ? VPT : 1], b_ahead[kAhead ? VPT : 1];
      if constexpr (kAhead) {
#pragma unroll
        for (int t = 0; t < VPT; ++t) {
          w_ahead[t] = at.piece_or(scale, T(1), t);
          b_ahead[t] = at.piece_or(bias, T(0), t);
        }
      }
      if (kind == CT_NORM_LAYER) {
        CT_EACH mean[0] += at.owned(t, e, x[t].v[e]);
        row_sum<T, LANES>(mean, lds, turn);
        mean[0] *= inverse;
        CT_EACH x[t].v[e] -= mean[0];
      }
      CT_EACH square[0] += at.owned(t, e, x[t].v[e] * x[t].v[e]);
      row_sum<T, LANES>(square, lds, turn);
      const T rate = rate_of(square[0] * inverse, epsilon);
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        const Quad<T> w = kAhead ? w_ahead[kAhead ? t : 0] : at.piece_or(scale, T(1), t);
#pragma unroll
        for (int e = 0; e < N; ++e) x[t].v[e] = x[t].v[e] * rate * w.v[e];
        if (bias) {
          const Quad<T> b = kAhead ? b_ahead[kAhead ? t : 0] : at.piece(static_cast<const T*>(bias), t);
#pragma unroll
          for (int e = 0; e < N; ++e) x[t].v[e] += b.v[e];
        }
      }
      if (a.statistics && at.lane == 0) {
        T* to = static_cast<T*>(a.statistics) + place * a.rows + row;
        to[0] = mean[0];
        to[a.rows] = rate;
      }
    };
    auto no_norm = [&](int place) {
      if (!a.statistics || at.lane != 0) return;
      T* to = static_cast<T*>(a.statistics) + place * a.rows + row;
      to[0] = 0;
      to[a.rows] = 1;
    };
    if (a.post != CT_NORM_NONE) norm(a.post, a.post_scale, a.post_bias, 0);
    else no_norm(0);
    if (a.gate_kind == kScalarGate || a.gate_kind == kRowGate) {
      const T g = static_cast<const T*>(a.gate.p)[a.gate_kind == kRowGate ? row * a.gate.ld : 0];
      CT_EACH x[t].v[e] *= g;
    } else if (a.gate_kind != kNoGate) {
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        const Quad<T> g = at.piece(static_cast<const T*>(a.gate.p) + (a.gate_kind == kFullGate ? row * a.gate.ld : 0), t);
#pragma unroll
        for (int e = 0; e < N; ++e) x[t].v[e] *= g.v[e];
      }
    }
    if (a.residual.p) {
      const T c = (T)a.residual_scale;
      CT_EACH x[t].v[e] = c * y[t].v[e] + x[t].v[e];
    }
#pragma unroll
    for (int t = 0; t < VPT; ++t) at.store(row_to<T>(a.output, row), t, x[t]);
    if (a.pre == CT_NORM_NONE) {
      no_norm(2);
      continue;
    }
    norm(a.pre, a.pre_scale, a.pre_bias, 2);
#pragma unroll
    for (int t = 0; t < VPT; ++t) at.store(row_to<T>(a.normalized, row), t, x[t]);
  }
}

// ------------------------------------------------------------------ gradient

struct NormGradientArgs {
  Matrix input_gradient, residual_gradient, gate_gradient, output_gradient, normalized_gradient, input, output, gate;
  const void *post_scale, *post_bias, *pre_scale;
  const void* statistics;
  void* partial;             // [slots][blocks][width]
  int64_t rows;
  uint32_t width, blocks;
  int post, pre, gate_kind;
  int slot[4], slots;        // of S1, S0, T1, T0 in partial; negative: not wanted
  double residual_scale;
};

// Whether the gate is a factor of all rows' sums: then it is left out of them.
__device__ __forceinline__ bool common_gate(int kind) { return kind == kNoGate || kind == kScalarGate || kind == kColumnGate; }

// The sums over the rows stay in LDS, a value to each lane and element, so that registers are left for what is on its way: the
// next row's operands are loaded into the registers of this one's as those are used up.
// kSums: 0 none, 1 S1 and T1, 2 all.  An absent gradient of the results is read from `input` and not used.
template <class T, int LANES, int VPT, int kSums, bool kStreaming>
__global__ void __launch_bounds__(block_of(LANES), VPT >= 3 ? 3 : 4) norm_gradient_kernel(const NormGradientArgs a) {
  constexpr int kThreads = block_of(LANES), kRows = kThreads / LANES;
  using R = Row<T, LANES, VPT, kStreaming>;
  constexpr int N = R::N;
  __shared__ T lds[LANES > 64 ? 2 * 3 * (LANES / 64) : 1];
  extern __shared__ __attribute__((aligned(16))) char sums_lds[];
  int turn = 0;
  const R at{threadIdx.x % LANES, a.width};
  const T inverse = T(1) / (T)a.width;
  // the pieces of sum `slot` of a group of lanes, side by side
  Quad<T>* const sums = reinterpret_cast<Quad<T>*>(sums_lds);
  const uint32_t pieces = (a.width + N - 1) / N;
  auto has = [&](int t) { return at.lane + t * LANES < pieces; };
  auto sum_at = [&](int slot, int group, int t) -> Quad<T>& { return sums[(slot * kRows + group) * pieces + at.lane + t * LANES]; };
  const int group = threadIdx.x / LANES;
  // value(t, e) to every sum of a slot
  auto add_to = [&](int slot, auto value) {
    if (slot < 0) return;
#pragma unroll
    for (int t = 0; t < VPT; ++t) {
      if (!has(t)) continue;
      Quad<T> q = sum_at(slot, group, t);
#pragma unroll
      for (int e = 0; e < N; ++e) q.v[e] += value(t, e);
      sum_at(slot, group, t) = q;
    }
  };
  if constexpr (kSums > 0) {
#pragma unroll
    for (int slot = 0; slot < 2 * kSums; ++slot)
      if (slot < a.slots) {
#pragma unroll
        for (int t = 0; t < VPT; ++t)
          if (has(t)) sum_at(slot, group, t) = Quad<T>{};
      }
  }
  const T* statistics = static_cast<const T*>(a.statistics);
  const bool post = a.post != CT_NORM_NONE, pre = a.pre != CT_NORM_NONE && a.normalized_gradient.p;
  const Matrix& of_d = a.output_gradient.p ? a.output_gradient : a.input;
  const Matrix& of_dh = pre ? a.normalized_gradient : a.input;
  const Matrix& of_oh = pre ? a.output : a.input;
  const int64_t stride = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / LANES;
  Quad<T> d[VPT], z[VPT], dh[VPT], oh[VPT];
  if (row < a.rows) {
    at.load(row_of<T>(of_dh, row), dh);
    at.load(row_of<T>(of_oh, row), oh);
    at.load(row_of<T>(of_d, row), d);
    at.load(row_of<T>(a.input, row), z);
  }
  for (; row < a.rows; row += stride) {
    const int64_t next = min(row + stride, a.rows - 1);
    if (!a.output_gradient.p) CT_EACH d[t].v[e] = 0;
    if (pre) {
      const T mean = statistics[2 * a.rows + row], rate = statistics[3 * a.rows + row];
      CT_EACH oh[t].v[e] = (oh[t].v[e] - mean) * rate;
      if constexpr (kSums > 0) add_to(a.slot[2], [&](int t, int e) { return dh[t].v[e] * oh[t].v[e]; });
      if constexpr (kSums > 1) add_to(a.slot[3], [&](int t, int e) { return dh[t].v[e]; });
      T sums[2] = {0, 0};
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        const Quad<T> w = at.piece_or(a.pre_scale, T(1), t);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          dh[t].v[e] *= w.v[e];
          sums[0] += at.owned(t, e, dh[t].v[e]);
          sums[1] += at.owned(t, e, dh[t].v[e] * oh[t].v[e]);
        }
      }
      row_sum<T, LANES>(sums, lds, turn);
      const T first = a.pre == CT_NORM_LAYER ? sums[0] * inverse : T(0), second = sums[1] * inverse;
      CT_EACH d[t].v[e] += rate * (dh[t].v[e] - first - oh[t].v[e] * second);
    }
    at.load(row_of<T>(of_dh, next), dh);
    at.load(row_of<T>(of_oh, next), oh);
    if (a.residual_gradient.p) {
      const T c = (T)a.residual_scale;
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        Quad<T> q;
#pragma unroll
        for (int e = 0; e < N; ++e) q.v[e] = c * d[t].v[e];
        at.store(row_to<T>(a.residual_gradient, row), t, q);
      }
    }
    // zh; its sums; the gate's gradient; dz
    const T mean = post ? statistics[row] : T(0), rate = post ? statistics[a.rows + row] : T(1);
    CT_EACH z[t].v[e] = (z[t].v[e] - mean) * rate;
    const bool of_columns = common_gate(a.gate_kind), of_row = a.gate_kind == kRowGate && a.gate_gradient.p;
    if (kSums > 0 && of_columns) {
      add_to(a.slot[0], [&](int t, int e) { return d[t].v[e] * z[t].v[e]; });
      if constexpr (kSums > 1) add_to(a.slot[1], [&](int t, int e) { return d[t].v[e]; });
    }
    T sums[3] = {0, 0, 0};
    if (of_row || (a.gate_kind == kFullGate && a.gate_gradient.p)) {
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        const Quad<T> w = at.piece_or(post ? a.post_scale : nullptr, T(1), t);
        Quad<T> u = at.piece_or(post ? a.post_bias : nullptr, T(0), t);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          u.v[e] = d[t].v[e] * (z[t].v[e] * w.v[e] + u.v[e]);
          sums[2] += at.owned(t, e, u.v[e]);
        }
        if (!of_row) at.store(row_to<T>(a.gate_gradient, row), t, u);
      }
    }
    if (a.gate_kind == kColumnGate || a.gate_kind == kFullGate) {
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        const Quad<T> g = at.piece(static_cast<const T*>(a.gate.p) + (a.gate_kind == kFullGate ? row * a.gate.ld : 0), t);
#pragma unroll
        for (int e = 0; e < N; ++e) d[t].v[e] *= g.v[e];
      }
    } else if (a.gate_kind != kNoGate) {
      const T g = static_cast<const T*>(a.gate.p)[a.gate_kind == kRowGate ? row * a.gate.ld : 0];
      CT_EACH d[t].v[e] *= g;
    }
    if (kSums > 0 && !of_columns) {
      add_to(a.slot[0], [&](int t, int e) { return d[t].v[e] * z[t].v[e]; });
      if constexpr (kSums > 1) add_to(a.slot[1], [&](int t, int e) { return d[t].v[e]; });
    }
    if (post || of_row) {
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        const Quad<T> w = at.piece_or(post ? a.post_scale : nullptr, T(1), t);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          d[t].v[e] *= w.v[e];
          sums[0] += at.owned(t, e, d[t].v[e]);
          sums[1] += at.owned(t, e, d[t].v[e] * z[t].v[e]);
        }
      }
      row_sum<T, LANES>(sums, lds, turn);
      if (of_row && at.lane == 0) static_cast<T*>(a.gate_gradient.p)[row * a.gate_gradient.ld] = sums[2];
      if (post) {
        const T first = a.post == CT_NORM_LAYER ? sums[0] * inverse : T(0), second = sums[1] * inverse;
        CT_EACH d[t].v[e] = rate * (d[t].v[e] - first - z[t].v[e] * second);
      }
    }
    if (a.input_gradient.p) {
#pragma unroll
      for (int t = 0; t < VPT; ++t) at.store(row_to<T>(a.input_gradient, row), t, d[t]);
    }
    at.load(row_of<T>(of_d, next), d);
    at.load(row_of<T>(a.input, next), z);
  }
  if constexpr (kSums > 0) {
    // of the block's rows, in the order of their groups of lanes
    __syncthreads();
    if (threadIdx.x >= LANES) return;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (a.slot[s] < 0 || (kSums == 1 && s % 2 == 1)) continue;
      T* to = static_cast<T*>(a.partial) + ((int64_t)a.slot[s] * a.blocks + blockIdx.x) * a.width;
#pragma unroll
      for (int t = 0; t < VPT; ++t) {
        if (!has(t)) continue;
        Quad<T> q = sum_at(a.slot[s], 0, t);
        for (int r = 1; r < kRows; ++r) {
          const Quad<T> other = sum_at(a.slot[s], r, t);
#pragma unroll
          for (int e = 0; e < N; ++e) q.v[e] += other.v[e];
        }
        at.store(to, t, q);
      }
    }
  }
}

struct NormFinishArgs {
  const void* partial;
  const void *post_scale, *post_bias;
  const void* gate;
  void *gate_gradient, *post_scale_gradient, *post_bias_gradient, *pre_scale_gradient, *pre_bias_gradient;
  void* by_column;   // of a scalar gate's gradient: its part of each column
  uint32_t width, blocks;
  int slot[4];
  int gate_kind;
};

// The blocks' sums of 32 columns, added in their order within each of 32 runs of blocks, in double.
template <class T>
__device__ __forceinline__ void finish_columns(const NormFinishArgs& a, uint32_t column0, double (&lds)[2][32][32]) {
  const uint32_t column = column0 + threadIdx.x % 32, run = threadIdx.x / 32;
  // S1 and S0 by one half of the blocks, T1 and T0 by the other
  const int half = 2 * blockIdx.y;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    double sum = 0;
    if (a.slot[half + s] >= 0 && column < a.width) {
      const T* from = static_cast<const T*>(a.partial) + (int64_t)a.slot[half + s] * a.blocks * a.width + column;
#pragma unroll 8
      for (uint32_t b = run; b < a.blocks; b += 32) sum += (double)from[(int64_t)b * a.width];
    }
    lds[s][run][threadIdx.x % 32] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= 32 || column >= a.width) return;
  double sums[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    sums[s] = lds[s][0][threadIdx.x];
    for (int r = 1; r < 32; ++r) sums[s] += lds[s][r][threadIdx.x];
  }
  auto store = [&](void* to, double v) {
    if (to) static_cast<T*>(to)[column] = (T)v;
  };
  if (half) {
    store(a.pre_scale_gradient, sums[0]);
    store(a.pre_bias_gradient, sums[1]);
    return;
  }
  double gate = 1;
  if (a.gate_kind == kScalarGate) gate = (double)*static_cast<const T*>(a.gate);
  if (a.gate_kind == kColumnGate) gate = (double)static_cast<const T*>(a.gate)[column];
  store(a.post_scale_gradient, gate * sums[0]);
  store(a.post_bias_gradient, gate * sums[1]);
  const double scale = a.post_scale ? (double)static_cast<const T*>(a.post_scale)[column] : 1.0;
  const double bias = a.post_bias ? (double)static_cast<const T*>(a.post_bias)[column] : 0.0;
  const double of_gate = scale * sums[0] + (a.slot[1] >= 0 ? bias * sums[1] : 0.0);
  if (a.gate_kind == kColumnGate) store(a.gate_gradient, of_gate);
  if (a.by_column) static_cast<double*>(a.by_column)[column] = of_gate;
}

// A launch of 2^32 lanes is refused: blocks take more than one run of columns of rows that long.
constexpr int64_t kMostFinishBlocks = int64_t(1) << 21;
template <class T>
__global__ void __launch_bounds__(1024) norm_finish_kernel(const NormFinishArgs a) {
  __shared__ double lds[2][32][32];
  for (uint32_t column0 = blockIdx.x * 32; column0 < a.width; column0 += gridDim.x * 32) {
    finish_columns<T>(a, column0, lds);
    __syncthreads();
  }
}

template <class T>
__global__ void __launch_bounds__(256) norm_scalar_gate_kernel(const double* by_column, uint32_t width, T* gradient) {
  __shared__ double lds[4];
  double sum = 0;
  for (uint32_t c = threadIdx.x; c < width; c += 256) sum += by_column[c];
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) *gradient = (T)(lds[0] + lds[1] + lds[2] + lds[3]);
}

// ------------------------------------------------------------------ rows that do not fit registers

constexpr int kLongBlock = 1024;

template <int K> __device__ __forceinline__ void long_sum(double (&v)[K], double* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) lds[k * 16 + threadIdx.x / 64] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = lds[k * 16];
    for (int w = 1; w < 16; ++w) v[k] += lds[k * 16 + w];
  }
}

template <class T> __device__ __forceinline__ T or_else(const void* p, int64_t i, T absent) { return p ? static_cast<const T*>(p)[i] : absent; }
template <class T> __device__ __forceinline__ T gate_at(const Matrix& gate, int kind, int64_t row, uint32_t c) {
  const T* g = static_cast<const T*>(gate.p);
  return kind == kNoGate ? T(1) : kind == kScalarGate ? g[0] : kind == kColumnGate ? g[c] : kind == kRowGate ? g[row * gate.ld] : g[row * gate.ld + c];
}

template <class T>
__global__ void __launch_bounds__(kLongBlock) norm_long_kernel(const NormArgs a) {
  __shared__ double lds[16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    auto statistics = [&](const T* x, int kind, int place, T* mean, T* rate) {
      double m[1] = {0}, q[1] = {0};
      *mean = 0;
      *rate = 1;
      if (kind == CT_NORM_LAYER) {
        for (uint32_t c = threadIdx.x; c < a.width; c += kLongBlock) m[0] += (double)x[c];
        long_sum(m, lds);
        *mean = (T)(m[0] / a.width);
      }
      if (kind != CT_NORM_NONE) {
        for (uint32_t c = threadIdx.x; c < a.width; c += kLongBlock) {
          const double y = (double)x[c] - (kind == CT_NORM_LAYER ? m[0] / a.width : 0.0);
          q[0] += y * y;
        }
        long_sum(q, lds);
        *rate = (T)(1.0 / sqrt(q[0] / a.width + a.epsilon));
      }
      if (a.statistics && threadIdx.x == 0) {
        T* to = static_cast<T*>(a.statistics) + place * a.rows + row;
        to[0] = *mean;
        to[a.rows] = *rate;
      }
    };
    const T* z = row_of<T>(a.input, row);
    T* out = row_to<T>(a.output, row);
    T mean, rate;
    statistics(z, a.post, 0, &mean, &rate);
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.width; c += kLongBlock) {
      T u = z[c];
      if (a.post != CT_NORM_NONE) u = (u - mean) * rate * or_else<T>(a.post_scale, c, 1) + or_else<T>(a.post_bias, c, 0);
      u *= gate_at<T>(a.gate, a.gate_kind, row, c);
      out[c] = a.residual.p ? (T)a.residual_scale * row_of<T>(a.residual, row)[c] + u : u;
    }
    __syncthreads();   // a lane reads again only what it wrote
    statistics(out, a.pre, 2, &mean, &rate);
    if (a.pre == CT_NORM_NONE) continue;
    T* h = row_to<T>(a.normalized, row);
    for (uint32_t c = threadIdx.x; c < a.width; c += kLongBlock)
      h[c] = (out[c] - mean) * rate * or_else<T>(a.pre_scale, c, 1) + or_else<T>(a.pre_bias, c, 0);
  }
}

// means [4][rows]: of y and y oh of the norm before the next block, of y and y zh of the one after this
template <class T>
struct LongRow {
  const NormGradientArgs& a;
  const double* means;
  int64_t row;
  T post_mean, post_rate, pre_mean, pre_rate;
  __device__ __forceinline__ LongRow(const NormGradientArgs& a, const double* means, int64_t row) : a(a), means(means), row(row) {
    const T* s = static_cast<const T*>(a.statistics);
    post_mean = a.post != CT_NORM_NONE ? s[row] : T(0);
    post_rate = a.post != CT_NORM_NONE ? s[a.rows + row] : T(1);
    pre_mean = before() ? s[2 * a.rows + row] : T(0);
    pre_rate = before() ? s[3 * a.rows + row] : T(1);
  }
  __device__ __forceinline__ bool before() const { return a.pre != CT_NORM_NONE && a.normalized_gradient.p; }
  __device__ __forceinline__ T dh(uint32_t c) const { return row_of<T>(a.normalized_gradient, row)[c]; }
  __device__ __forceinline__ T oh(uint32_t c) const { return (row_of<T>(a.output, row)[c] - pre_mean) * pre_rate; }
  __device__ __forceinline__ T zh(uint32_t c) const { return (row_of<T>(a.input, row)[c] - post_mean) * post_rate; }
  __device__ __forceinline__ T post_scale(uint32_t c) const { return a.post != CT_NORM_NONE ? or_else<T>(a.post_scale, c, 1) : T(1); }
  __device__ __forceinline__ T u(uint32_t c) const {
    return zh(c) * post_scale(c) + (a.post != CT_NORM_NONE ? or_else<T>(a.post_bias, c, 0) : T(0));
  }
  __device__ __forceinline__ T gate(uint32_t c) const { return gate_at<T>(a.gate, a.gate_kind, row, c); }
  __device__ __forceinline__ double d(uint32_t c) const {
    double v = a.output_gradient.p ? (double)row_of<T>(a.output_gradient, row)[c] : 0.0;
    if (before()) {
      const double y = (double)dh(c) * (double)or_else<T>(a.pre_scale, c, 1);
      v += (double)pre_rate * (y - (a.pre == CT_NORM_LAYER ? means[row] : 0.0) - (double)oh(c) * means[a.rows + row]);
    }
    return v;
  }
};

template <class T>
__global__ void __launch_bounds__(kLongBlock) norm_long_means_kernel(const NormGradientArgs a, double* means) {
  __shared__ double lds[48];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const LongRow<T> r(a, means, row);
    double p[2] = {0, 0}, q[3] = {0, 0, 0};
    if (r.before()) {
      for (uint32_t c = threadIdx.x; c < a.width; c += kLongBlock) {
        const double y = (double)r.dh(c) * (double)or_else<T>(a.pre_scale, c, 1);
        p[0] += y;
        p[1] += y * (double)r.oh(c);
      }
      long_sum(p, lds);
    }
    if (threadIdx.x == 0) {
      means[row] = p[0] / a.width;
      means[a.rows + row] = p[1] / a.width;
    }
    __threadfence_block();
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.width; c += kLongBlock) {
      const double d = r.d(c), y = d * (double)(r.gate(c) * r.post_scale(c));
      q[0] += y;
      q[1] += y * (double)r.zh(c);
      q[2] += d * (double)r.u(c);
    }
    long_sum(q, lds);
    if (threadIdx.x == 0) {
      means[2 * a.rows + row] = q[0] / a.width;
      means[3 * a.rows + row] = q[1] / a.width;
      if (a.gate_kind == kRowGate && a.gate_gradient.p) static_cast<T*>(a.gate_gradient.p)[row * a.gate_gradient.ld] = (T)q[2];
    }
  }
}

// Block (x, y): 256 columns of every a.blocks-th row.
template <class T>
__global__ void __launch_bounds__(256) norm_long_sums_kernel(const NormGradientArgs a, const double* means) {
  const uint32_t c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.width) return;
  double sums[4] = {0, 0, 0, 0};
  for (int64_t row = blockIdx.y; row < a.rows; row += a.blocks) {
    const LongRow<T> r(a, means, row);
    const double d = r.d(c) * (common_gate(a.gate_kind) ? 1.0 : (double)r.gate(c));
    sums[0] += d * (double)r.zh(c);
    sums[1] += d;
    if (r.before()) {
      sums[2] += (double)r.dh(c) * (double)r.oh(c);
      sums[3] += (double)r.dh(c);
    }
  }
#pragma unroll
  for (int s = 0; s < 4; ++s)
    if (a.slot[s] >= 0) static_cast<T*>(a.partial)[((int64_t)a.slot[s] * a.blocks + blockIdx.y) * a.width + c] = (T)sums[s];
}

template <class T>
__global__ void __launch_bounds__(256) norm_long_apply_kernel(const NormGradientArgs a, const double* means) {
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const LongRow<T> r(a, means, row);
    const uint32_t c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.width) continue;
    const double d = r.d(c), gate = (double)r.gate(c);
    double dz = d * gate;
    const T u = r.u(c);
    if (a.post != CT_NORM_NONE) {
      dz *= (double)r.post_scale(c);
      dz = (double)r.post_rate * (dz - (a.post == CT_NORM_LAYER ? means[2 * a.rows + row] : 0.0) - (double)r.zh(c) * means[3 * a.rows + row]);
    }
    if (a.gate_kind == kFullGate && a.gate_gradient.p) row_to<T>(a.gate_gradient, row)[c] = (T)(d * (double)u);
    if (a.residual_gradient.p) row_to<T>(a.residual_gradient, row)[c] = (T)((double)(T)a.residual_scale * d);
    if (a.input_gradient.p) row_to<T>(a.input_gradient, row)[c] = (T)dz;
  }
}

// ------------------------------------------------------------------ host

// Calls f with the lanes of a row and the pieces to a lane that hold `width` elements; false if none do.  (Three pieces beside two and
// four: 32768 x 768 floats 75 us and 116 of the gradient, with four 87 and 121; 3000 x 5000 doubles 99 and 289, with four 145 and 389.)
template <class T, class F>
bool with_shape(uint32_t width, F f) {
  constexpr uint32_t N = Quad<T>::N;
  const uint32_t pieces = (width + N - 1) / N;
  if (width < N) return false;
#define CT_SHAPE(L, V) \
  if (pieces <= L * V) return f(std::integral_constant<int, L>(), std::integral_constant<int, V>()), true
  CT_SHAPE(16, 1); CT_SHAPE(16, 2); CT_SHAPE(16, 3); CT_SHAPE(16, 4);
  CT_SHAPE(64, 2); CT_SHAPE(64, 3); CT_SHAPE(64, 4);
  CT_SHAPE(256, 2); CT_SHAPE(256, 3); CT_SHAPE(256, 4);
  CT_SHAPE(1024, 2); CT_SHAPE(1024, 3); CT_SHAPE(1024, 4);
#undef CT_SHAPE
  return false;
}

constexpr int64_t kMostNormBlocks = 1 << 20;
constexpr int64_t kUnits = 256, kLdsOfAUnit = 160 << 10, kBytesAhead = 128 << 10;
constexpr int64_t kMostSumLds = 128 << 10;   // of a block, for its sums
constexpr int64_t kMostSumBytes = int64_t(64) << 20;

// Operands and results that the last-level cache does not hold together go past the caches.
bool streaming(int64_t rows, int64_t width, int64_t matrices, int64_t size) { return rows * width * matrices * size > int64_t(256) << 20; }

template <class T>
int norm_typed(hipStream_t s, const NormArgs& a) {
  const bool taken = with_shape<T>(a.width, [&](auto lanes, auto pieces) {
    constexpr int L = decltype(lanes)::value, V = decltype(pieces)::value, kThreads = block_of(L), kRows = kThreads / L;
    const int64_t blocks = std::min((a.rows + kRows - 1) / kRows, kMostNormBlocks);
    if (streaming(a.rows, a.width, 3 + (a.pre != CT_NORM_NONE), sizeof(T)))
      hipLaunchKernelGGL((norm_kernel<T, L, V, true>), dim3((uint32_t)blocks), dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((norm_kernel<T, L, V, false>), dim3((uint32_t)blocks), dim3(kThreads), 0, s, a);
  });
  if (!taken) hipLaunchKernelGGL((norm_long_kernel<T>), dim3((uint32_t)std::min(a.rows, kMostNormBlocks)), dim3(kLongBlock), 0, s, a);
  note_kernel(taken ? "norm_residual" : "norm_residual_long");
  return after_launch(s);
}

// Blocks to a compute unit whose operands are on their way at the same time: 128 KiB in all.  (16384 x 2048 floats, three, four
// and five blocks of 256 lanes: 157, 151 and 163 us; 8192 x 4096, two, three and four: 150, 155 and 177; more blocks also leave more sums.)
int64_t blocks_of_a_unit(int64_t bytes_of_a_block, int waves, int pieces) {
  const int64_t of_registers = (pieces >= 3 ? 12 : pieces == 2 ? 16 : 24) / waves;
  return std::max<int64_t>(1, std::min(kBytesAhead / bytes_of_a_block, of_registers));
}

template <class T>
int norm_gradient_typed(hipStream_t s, NormGradientArgs a, NormFinishArgs f) {
  const int slots = std::max({a.slot[0], a.slot[1], a.slot[2], a.slot[3]}) + 1;
  const bool sums = slots > 0, biases = a.slot[1] >= 0 || a.slot[3] >= 0;
  a.slots = slots;
  // Sums that LDS does not hold together are formed in two passes, those of the biases first: it stores no other result, and so may results be in
  // the place of operands.  (2048 rows of 10000 floats, layer norms and biases: 212 us; the long kernels 559.)
  const bool together = (int64_t)slots * a.width * (int64_t)sizeof(T) <= kMostSumLds;
  const int of_a_pass = together ? slots : 2, stored = together ? std::max(slots, 1) : 4;
  const bool fits = with_shape<T>(a.width, [](auto, auto) {}) && (int64_t)of_a_pass * a.width * (int64_t)sizeof(T) <= kMostSumLds;
  const size_t of_columns = (size_t)a.width * sizeof(double), of_means = fits ? 0 : (size_t)4 * a.rows * sizeof(double);
  double *by_column = nullptr, *means = nullptr;
  // Scratch for the sums of `blocks` blocks, which the last launch adds.
  auto with_sums_of = [&](int64_t blocks) {
    a.blocks = f.blocks = (uint32_t)blocks;
    void* scratch = nullptr;
    if (int rc = stream_scratch(s, of_columns + of_means + (size_t)stored * blocks * a.width * sizeof(T), &scratch)) return rc;
    by_column = static_cast<double*>(scratch);
    means = by_column + a.width;
    a.partial = means + (fits ? 0 : 4 * a.rows);
    f.partial = a.partial;
    return (int)CT_OK;
  };
  const int64_t most_blocks = std::max<int64_t>(1, kMostSumBytes / ((int64_t)stored * a.width * (int64_t)sizeof(T)));
  int rc = CT_OK;
  if (a.rows == 0) {
    rc = with_sums_of(0);
  } else if (fits) {
    with_shape<T>(a.width, [&](auto lanes, auto pieces) {
      constexpr int L = decltype(lanes)::value, V = decltype(pieces)::value, kThreads = block_of(L), kRows = kThreads / L;
      const size_t lds = (size_t)of_a_pass * kRows * ((a.width + Quad<T>::N - 1) / Quad<T>::N) * sizeof(Quad<T>);
      // each block of as many rows as the others
      const int64_t ahead = (int64_t)4 * kRows * a.width * sizeof(T), of_lds = lds ? std::max<int64_t>(1, kLdsOfAUnit / (int64_t)(lds + 1024)) : 32;
      const int64_t at_once = kUnits * std::min(blocks_of_a_unit(ahead, kThreads / 64, V), of_lds), groups = (a.rows + kRows - 1) / kRows;
      const int64_t turns = (groups + at_once - 1) / at_once;
      if ((rc = with_sums_of(std::min((groups + turns - 1) / turns, most_blocks)))) return;
      auto launch = [&](auto kernel, const NormGradientArgs& pass) {
        if (lds > (48 << 10)) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        hipLaunchKernelGGL(kernel, dim3(a.blocks), dim3(kThreads), lds, s, pass);
      };
      const bool past = streaming(a.rows, a.width, 6, sizeof(T));
      auto launch_pass = [&](const NormGradientArgs& pass, int of_sums) {
        if (of_sums == 2 && past) launch(norm_gradient_kernel<T, L, V, 2, true>, pass);
        else if (of_sums == 2) launch(norm_gradient_kernel<T, L, V, 2, false>, pass);
        else if (of_sums == 1 && past) launch(norm_gradient_kernel<T, L, V, 1, true>, pass);
        else if (of_sums == 1) launch(norm_gradient_kernel<T, L, V, 1, false>, pass);
        else if (past) launch(norm_gradient_kernel<T, L, V, 0, true>, pass);
        else launch(norm_gradient_kernel<T, L, V, 0, false>, pass);
      };
      a.slots = of_a_pass;
      if (together) {
        launch_pass(a, biases ? 2 : sums ? 1 : 0);
      } else {
        for (int first : {1, 0}) {
          NormGradientArgs pass = a;
          if (first == 1) pass.input_gradient.p = pass.residual_gradient.p = pass.gate_gradient.p = nullptr;
          pass.partial = static_cast<T*>(a.partial) + (first == 1 ? (int64_t)2 * a.blocks * a.width : 0);
          for (int i = 0; i < 4; ++i) {
            pass.slot[i] = i % 2 == first && a.slot[i] >= 0 ? i / 2 : -1;
            if (i % 2 == first && a.slot[i] >= 0) f.slot[i] = 2 * first + i / 2;
          }
          launch_pass(pass, first + 1);
        }
      }
    });
  } else if (!(rc = with_sums_of(std::min<int64_t>({a.rows, most_blocks, 512})))) {
    const uint32_t columns = (a.width + 255) / 256;
    hipLaunchKernelGGL((norm_long_means_kernel<T>), dim3((uint32_t)std::min(a.rows, kMostNormBlocks)), dim3(kLongBlock), 0, s, a, means);
    if (sums) hipLaunchKernelGGL((norm_long_sums_kernel<T>), dim3(columns, a.blocks), dim3(256), 0, s, a, means);
    hipLaunchKernelGGL((norm_long_apply_kernel<T>), dim3(columns, (uint32_t)std::min<int64_t>(a.rows, 4096)), dim3(256), 0, s, a, means);
  }
  if (rc) return rc;
  if (f.by_column) f.by_column = by_column;
  if (sums) hipLaunchKernelGGL((norm_finish_kernel<T>), dim3((uint32_t)std::min<int64_t>((a.width + 31) / 32, kMostFinishBlocks), 2), dim3(1024), 0, s, f);
  if (f.by_column) hipLaunchKernelGGL((norm_scalar_gate_kernel<T>), dim3(1), dim3(256), 0, s, by_column, a.width, static_cast<T*>(f.gate_gradient));
  note_kernel(fits ? "norm_residual_gradient" : "norm_residual_gradient_long");
  return after_launch(s);
}

// A [rows, width] operand; dimensions of one are a row.
int read_matrix(const char* what, const void* p, const ct_dims* d, int64_t rows, int64_t width, Matrix* out) {
  *out = Matrix{const_cast<void*>(p), 0};
  if (!p) return CT_OK;
  CT_REQUIRE(d && (d->ndim == 1 || d->ndim == 2), "%s: one or two dimensions are taken", what);
  const int last = d->ndim - 1;
  for (int i = 0; i <= last; ++i) CT_REQUIRE(!d->index[i], "%s: no indexed dimension is taken", what);
  CT_REQUIRE((last ? d->shape[0] : 1) == rows && d->shape[last] == width, "%s is [%lld, %lld], [%lld, %lld] is needed", what,
             (long long)(last ? d->shape[0] : 1), (long long)d->shape[last], (long long)rows, (long long)width);
  CT_REQUIRE(width <= 1 || d->strides[last] == 1, "%s: the innermost stride must be 1", what);
  out->ld = last ? d->strides[0] : width;
  if (rows == 1) out->ld = std::max(out->ld, width);
  CT_REQUIRE(out->ld >= width, "%s: column stride %lld below the row's length", what, (long long)out->ld);
  return CT_OK;
}

int read_gate(const char* what, const void* p, const ct_dims* d, int64_t rows, int64_t width, Matrix* out, int* kind) {
  *out = Matrix{const_cast<void*>(p), 0};
  *kind = kNoGate;
  if (!p) return CT_OK;
  CT_REQUIRE(d && (d->ndim == 1 || d->ndim == 2), "%s: one or two dimensions are taken", what);
  const int last = d->ndim - 1;
  for (int i = 0; i <= last; ++i) CT_REQUIRE(!d->index[i], "%s: no indexed dimension is taken", what);
  const int64_t r = last ? d->shape[0] : 1, w = d->shape[last];
  CT_REQUIRE((r == rows || r == 1) && (w == width || w == 1), "%s is [%lld, %lld]: [%lld or 1, %lld or 1] is needed", what, (long long)r,
             (long long)w, (long long)rows, (long long)width);
  // of no rows, [0, ..] is a gate by row too: its gradient has no elements, a column sum would be stored behind it
  const bool by_row = r == rows && rows != 1, by_column = w == width && width > 1;
  CT_REQUIRE(!by_column || d->strides[last] == 1, "%s: the innermost stride must be 1", what);
  *kind = by_row ? (by_column ? kFullGate : kRowGate) : by_column ? kColumnGate : kScalarGate;
  out->ld = by_row ? d->strides[0] : width;
  CT_REQUIRE(!by_row || out->ld >= w, "%s: column stride %lld below the row's length", what, (long long)out->ld);
  return CT_OK;
}

RowRange range_of(const Matrix& m, int64_t rows, int64_t width) { return {m.p, rows, width, m.ld}; }
// Another matrix's elements, other than by being that matrix.
bool meets_other(const Matrix& a, const Matrix& b, int64_t rows, int64_t width, int64_t size) {
  return !(a.p == b.p && (a.ld == b.ld || rows == 1)) && rows_meet(range_of(a, rows, width), range_of(b, rows, width), size);
}
RowRange gate_range(const Matrix& m, int kind, int64_t rows, int64_t width) {
  switch (kind) {
    case kScalarGate: return {m.p, 1, 1, 1};
    case kColumnGate: return {m.p, 1, width, width};
    case kRowGate: return {m.p, rows, 1, m.ld};
    case kFullGate: return {m.p, rows, width, m.ld};
    default: return {nullptr, 0, 0, 1};
  }
}
bool known_norm(int kind) { return kind == CT_NORM_NONE || kind == CT_NORM_RMS || kind == CT_NORM_LAYER; }
constexpr int64_t kMostWidth = (int64_t(1) << 30);

#define CT_TRY(expr) \
  if (int rc__ = (expr)) return rc__

}  // namespace

extern "C" {

int ct_norm_residual(void* stream, void* output, const ct_dims* output_dims, void* normalized, const ct_dims* normalized_dims,
                     void* statistics, const void* input, const ct_dims* input_dims, const void* residual,
                     const ct_dims* residual_dims, const void* gate, const ct_dims* gate_dims, const void* post_scale,
                     const void* post_bias, const void* pre_scale, const void* pre_bias, int post_kind, int pre_kind,
                     double residual_scale, double epsilon, int dtype) {
  CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, "ct_norm_residual: datatype must be float or double");
  CT_REQUIRE(known_norm(post_kind) && known_norm(pre_kind), "ct_norm_residual: unknown kind of norm");
  CT_REQUIRE(epsilon >= 0, "ct_norm_residual: epsilon must not be negative");
  CT_REQUIRE(output_dims && (output_dims->ndim == 1 || output_dims->ndim == 2), "output: one or two dimensions are taken");
  const int64_t rows = output_dims->ndim == 2 ? output_dims->shape[0] : 1, width = output_dims->shape[output_dims->ndim - 1];
  CT_REQUIRE(rows >= 0 && width >= 0 && width <= kMostWidth, "ct_norm_residual: bad extent");
  if (rows == 0 || width == 0) return CT_OK;
  CT_REQUIRE(output && input && (normalized || pre_kind == CT_NORM_NONE), "ct_norm_residual: null buffer");
  NormArgs a{};
  CT_TRY(read_matrix("output", output, output_dims, rows, width, &a.output));
  CT_TRY(read_matrix("input", input, input_dims, rows, width, &a.input));
  CT_TRY(read_matrix("residual", residual, residual_dims, rows, width, &a.residual));
  CT_TRY(read_matrix("normalized", pre_kind == CT_NORM_NONE ? nullptr : normalized, normalized_dims, rows, width, &a.normalized));
  CT_TRY(read_gate("gate", gate, gate_dims, rows, width, &a.gate, &a.gate_kind));
  const int64_t size = dtype_size(dtype);
  const RowRange of_gate = gate_range(a.gate, a.gate_kind, rows, width);
  const Run of_statistics{statistics, 4 * rows * size};
  for (const Matrix* to : {&a.output, &a.normalized}) {
    const RowRange range = range_of(*to, rows, width);
    bool bad = meets_other(*to, a.input, rows, width, size) || meets_other(*to, a.residual, rows, width, size) || rows_meet(range, of_gate, size);
    for (const void* p : {post_scale, post_bias, pre_scale, pre_bias}) bad = bad || run_meets({p, width * size}, range, size);
    bad = bad || run_meets(of_statistics, range, size);
    CT_REQUIRE(!bad, "ct_norm_residual: a result overlaps an operand");
  }
  bool of_operands = run_meets(of_statistics, range_of(a.input, rows, width), size) || run_meets(of_statistics, range_of(a.residual, rows, width), size) ||
                     run_meets(of_statistics, of_gate, size);
  for (const void* p : {post_scale, post_bias, pre_scale, pre_bias}) of_operands = of_operands || runs_meet(of_statistics, {p, width * size});
  CT_REQUIRE(!of_operands, "ct_norm_residual: the statistics overlap an operand");
  CT_REQUIRE(!rows_meet(range_of(a.output, rows, width), range_of(a.normalized, rows, width), size), "ct_norm_residual: the results overlap");
  a.post_scale = post_scale; a.post_bias = post_bias; a.pre_scale = pre_scale; a.pre_bias = pre_bias;
  a.statistics = statistics;
  a.rows = rows; a.width = (uint32_t)width;
  a.post = post_kind; a.pre = pre_kind;
  a.residual_scale = residual_scale; a.epsilon = epsilon;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == CT_F32 ? norm_typed<float>(s, a) : norm_typed<double>(s, a);
}

int ct_norm_residual_gradient(void* stream, void* input_gradient, const ct_dims* input_gradient_dims, void* residual_gradient,
                              const ct_dims* residual_gradient_dims, void* gate_gradient, void* post_scale_gradient,
                              void* post_bias_gradient, void* pre_scale_gradient, void* pre_bias_gradient,
                              const void* output_gradient, const ct_dims* output_gradient_dims, const void* normalized_gradient,
                              const ct_dims* normalized_gradient_dims, const void* input, const ct_dims* input_dims,
                              const void* output, const ct_dims* output_dims, const void* statistics, const void* gate,
                              const ct_dims* gate_dims, const void* post_scale, const void* post_bias, const void* pre_scale,
                              int post_kind, int pre_kind, double residual_scale, int dtype) {
  CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, "ct_norm_residual_gradient: datatype must be float or double");
  CT_REQUIRE(known_norm(post_kind) && known_norm(pre_kind), "ct_norm_residual_gradient: unknown kind of norm");
  CT_REQUIRE(input_dims && (input_dims->ndim == 1 || input_dims->ndim == 2), "input: one or two dimensions are taken");
  const int64_t rows = input_dims->ndim == 2 ? input_dims->shape[0] : 1, width = input_dims->shape[input_dims->ndim - 1];
  CT_REQUIRE(rows >= 0 && width >= 0 && width <= kMostWidth, "ct_norm_residual_gradient: bad extent");
  CT_REQUIRE(!gate_gradient || gate, "ct_norm_residual_gradient: a gradient of no gate");
  if (width == 0) {   // a gate by row or of one value has a gradient all the same: a sum of nothing
    if (!gate_gradient) return CT_OK;
    Matrix of_gate;
    int kind;
    CT_TRY(read_gate("gate", gate, gate_dims, rows, width, &of_gate, &kind));
    return ct_memset(stream, gate_gradient, dtype, 0.0, (gate_dims->ndim == 2 ? gate_dims->shape[0] : 1) * gate_dims->shape[gate_dims->ndim - 1]);
  }
  const bool before = pre_kind != CT_NORM_NONE && normalized_gradient;
  CT_REQUIRE(rows == 0 || (input && (output || !before) && (statistics || (post_kind == CT_NORM_NONE && !before))),
             "ct_norm_residual_gradient: null buffer");
  CT_REQUIRE(post_kind != CT_NORM_NONE || (!post_scale_gradient && !post_bias_gradient), "ct_norm_residual_gradient: gradients of no post norm");
  CT_REQUIRE(pre_kind != CT_NORM_NONE || (!pre_scale_gradient && !pre_bias_gradient), "ct_norm_residual_gradient: gradients of no pre norm");
  NormGradientArgs a{};
  CT_TRY(read_matrix("input", input, input_dims, rows, width, &a.input));
  CT_TRY(read_matrix("output", before ? output : nullptr, output_dims, rows, width, &a.output));
  CT_TRY(read_matrix("output gradient", output_gradient, output_gradient_dims, rows, width, &a.output_gradient));
  CT_TRY(read_matrix("normalized gradient", before ? normalized_gradient : nullptr, normalized_gradient_dims, rows, width, &a.normalized_gradient));
  CT_TRY(read_matrix("input gradient", input_gradient, input_gradient_dims, rows, width, &a.input_gradient));
  CT_TRY(read_matrix("residual gradient", residual_gradient, residual_gradient_dims, rows, width, &a.residual_gradient));
  CT_TRY(read_gate("gate", gate, gate_dims, rows, width, &a.gate, &a.gate_kind));
  // rows of a gate's gradient are packed as the gate's dimensions are
  a.gate_gradient = Matrix{gate_gradient, a.gate_kind == kFullGate ? width : 1};
  const int64_t size = dtype_size(dtype);
  const RowRange of_gate = gate_range(a.gate, a.gate_kind, rows, width), of_gate_gradient = gate_range(a.gate_gradient, a.gate_kind, rows, width);
  // of what is read, and of the gradients that are no matrices
  const RowRange matrices[] = {range_of(a.input, rows, width), range_of(a.output, rows, width), range_of(a.output_gradient, rows, width),
                               range_of(a.normalized_gradient, rows, width), of_gate};
  const Run vectors[] = {{post_kind != CT_NORM_NONE ? post_scale : nullptr, width * size}, {post_kind != CT_NORM_NONE ? post_bias : nullptr, width * size},
                         {before ? pre_scale : nullptr, width * size}, {statistics, 4 * rows * size}};
  const Run gradients[] = {{post_scale_gradient, width * size}, {post_bias_gradient, width * size}, {pre_scale_gradient, width * size},
                           {pre_bias_gradient, width * size}, {gate_gradient, of_gate_gradient.rows * of_gate_gradient.width * size}};
  for (const Matrix* to : {&a.input_gradient, &a.residual_gradient}) {
    const RowRange range = range_of(*to, rows, width);
    bool bad = meets_other(*to, a.output_gradient, rows, width, size) || meets_other(*to, a.normalized_gradient, rows, width, size) ||
               rows_meet(range, matrices[0], size) || rows_meet(range, matrices[1], size) || rows_meet(range, of_gate, size);
    for (const Run& run : vectors) bad = bad || run_meets(run, range, size);
    for (const Run& run : gradients) bad = bad || run_meets(run, range, size);
    CT_REQUIRE(!bad, "ct_norm_residual_gradient: a result overlaps an operand");
  }
  for (int i = 0; i < 5; ++i) {
    bool bad = false, results = false;
    for (const RowRange& m : matrices) bad = bad || run_meets(gradients[i], m, size);
    for (const Run& run : vectors) bad = bad || runs_meet(gradients[i], run);
    for (int j = 0; j < i; ++j) results = results || runs_meet(gradients[i], gradients[j]);
    CT_REQUIRE(!bad, "ct_norm_residual_gradient: %s overlaps an operand", i == 4 ? "the gate's gradient" : "the gradient of a scale or bias");
    CT_REQUIRE(!results, "ct_norm_residual_gradient: the results overlap");
  }
  CT_REQUIRE(!rows_meet(range_of(a.input_gradient, rows, width), range_of(a.residual_gradient, rows, width), size),
             "ct_norm_residual_gradient: the results overlap");
  const bool of_columns = gate_gradient && (a.gate_kind == kColumnGate || a.gate_kind == kScalarGate);
  a.post_scale = post_scale; a.post_bias = post_bias; a.pre_scale = pre_scale;
  a.statistics = statistics;
  a.rows = rows; a.width = (uint32_t)width;
  a.post = post_kind; a.pre = pre_kind;
  a.residual_scale = residual_scale;
  const bool has_bias = post_kind != CT_NORM_NONE && post_bias;
  const bool wanted[4] = {post_scale_gradient || of_columns, post_bias_gradient || (of_columns && has_bias), pre_scale_gradient != nullptr,
                          pre_bias_gradient != nullptr};
  NormFinishArgs f{};
  for (int i = 0, slot = 0; i < 4; ++i) a.slot[i] = f.slot[i] = wanted[i] ? slot++ : -1;
  f.post_scale = post_kind != CT_NORM_NONE ? post_scale : nullptr;
  f.post_bias = has_bias ? post_bias : nullptr;
  f.gate = gate; f.gate_kind = a.gate_kind;
  f.gate_gradient = of_columns ? gate_gradient : nullptr;
  f.post_scale_gradient = post_scale_gradient; f.post_bias_gradient = post_bias_gradient;
  f.pre_scale_gradient = pre_scale_gradient; f.pre_bias_gradient = pre_bias_gradient;
  f.by_column = of_columns && a.gate_kind == kScalarGate ? gate_gradient : nullptr;   // replaced by scratch
  f.width = (uint32_t)width;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == CT_F32 ? norm_gradient_typed<float>(s, a, f) : norm_gradient_typed<double>(s, a, f);
}

}  // extern "C"
