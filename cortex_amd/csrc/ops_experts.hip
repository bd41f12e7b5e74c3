// ops_experts.hip -- the choice of experts, the order of rows by expert, and the sum of a token's rows.
//
// Routing.  A group of lanes holds a token's logits in registers and takes the largest n_chosen times; ties go to the lowest
// index.  Logits are compared as integers that order as they do, NaN above all, -infinity below every one that may be chosen.
// The order of rows is a stable counting sort of the assignments (t, j) by expert: blocks of consecutive tokens count their
// assignments, one wave to an expert adds the blocks' counts up, and each block then knows the place of its own.
//
// Combining reads the rows of a token once and writes its sum; its gradient reads the token's gradient and its rows once and
// writes as many.
#include <algorithm>

#include "elementwise.h"
#include "rows.h"

using namespace cthip;

namespace {

constexpr int kRouteBlock = 256;
constexpr int64_t kCombineCacheBytes = int64_t(256) << 20;   // what the last-level cache holds
constexpr int64_t kMostBlocks = 1 << 20;   // of a launch; blocks take more than one token each beyond
constexpr int kMostExperts = 1024, kMostChosen = 32;

template <class T> struct KeyOf;
template <> struct KeyOf<float> {
  using Key = uint32_t;
  using Bits = int32_t;
};
template <> struct KeyOf<double> {
  using Key = uint64_t;
  using Bits = int64_t;
};

// An unsigned integer that orders as the floats do: -0 and +0 alike, NaN above all, 0 below all.
template <class T> __device__ __forceinline__ typename KeyOf<T>::Key key_of(T x) {
  using Key = typename KeyOf<T>::Key;
  using Bits = typename KeyOf<T>::Bits;
  if (x != x) return ~Key(0);
  const Bits b = __builtin_bit_cast(Bits, x + T(0));
  return b < 0 ? ~Key(b) : Key(b) | (Key(1) << (sizeof(T) * 8 - 1));
}
template <class T> __device__ __forceinline__ T of_key(typename KeyOf<T>::Key k) {
  using Key = typename KeyOf<T>::Key;
  const Key top = Key(1) << (sizeof(T) * 8 - 1);
  return __builtin_bit_cast(T, k & top ? Key(k ^ top) : Key(~k));
}
// Of -infinity: this and all below it are never chosen.
template <class T> __device__ __forceinline__ typename KeyOf<T>::Key closed_key() { return key_of<T>(-__builtin_inf()); }

struct RouteArgs {
  int32_t* experts;
  void* weights;
  int32_t* offsets;
  int32_t* tokens;
  int32_t* slots;
  const void* logits;
  int64_t colstride;
  uint32_t n, n_experts, n_chosen, tokens_per_block, blocks;
  bool renormalize;
  int32_t* counts;   // [blocks][n_experts + 1]; then, in place, of all blocks before
  int32_t* totals;   // [n_experts + 1]
};

// experts and weights of one token by LANES lanes, V logits to each (lane + v * LANES).
template <class T, int LANES, int V>
__device__ __forceinline__ void choose(const RouteArgs& a, uint32_t token, uint32_t lane, uint32_t* counts) {
  using Key = typename KeyOf<T>::Key;
  const T* row = static_cast<const T*>(a.logits) + (int64_t)token * a.colstride;
  T x[V];
  Key key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const uint32_t e = lane + v * LANES;
    x[v] = e < a.n_experts ? row[e] : -__builtin_inf();
    key[v] = key_of<T>(x[v]);
    if (key[v] <= closed_key<T>()) key[v] = 0;
  }
  T top = 0, sum = 0;
  uint32_t found = 0;
  T mine[kMostChosen / LANES + 1];   // value j of the chosen ones, in lane j % LANES
#pragma unroll
  for (auto& m : mine) m = 0;
  const int64_t at = (int64_t)token * a.n_chosen;
  for (uint32_t j = 0; j < a.n_chosen; ++j) {
    Key best = 0;
    uint32_t index = 0xffffffffu;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > best) {
        best = key[v];
        index = lane + v * LANES;
      }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) {
      const Key k = __shfl_xor(best, m);
      const uint32_t i = __shfl_xor(index, m);
      if (k > best || (k == best && i < index)) {
        best = k;
        index = i;
      }
    }
    const bool any = best != 0;
    const T value = of_key<T>(best);
    if (j == 0) top = value;
    const T power = any ? (T)exp(value - top) : T(0);
    sum += power;
    found += any;
#pragma unroll
    for (int q = 0; q < (int)(sizeof(mine) / sizeof(T)); ++q)
      if (j == lane + q * LANES) mine[q] = power;
    if (lane == 0) {
      a.experts[at + j] = any ? (int32_t)index : -1;
      atomicAdd(&counts[any ? index : a.n_experts], 1u);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (index == lane + v * LANES) key[v] = 0;
  }
  if (!a.renormalize) {
    sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += (T)exp(x[v] - top);   // of a row without an open expert: not used
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
  }
  T* weights = static_cast<T*>(a.weights) + at;
#pragma unroll
  for (int q = 0; q < (int)(sizeof(mine) / sizeof(T)); ++q) {
    const uint32_t j = lane + q * LANES;
    if (j < a.n_chosen) weights[j] = j < found ? mine[q] / sum : T(0);
  }
}

template <class T, int LANES, int V>
__global__ void __launch_bounds__(kRouteBlock) route_choose_kernel(const RouteArgs a) {
  __shared__ uint32_t counts[kMostExperts + 1];
  for (uint32_t e = threadIdx.x; e <= a.n_experts; e += kRouteBlock) counts[e] = 0;
  __syncthreads();
  const uint32_t first = blockIdx.x * a.tokens_per_block, end = min(a.n, first + a.tokens_per_block);
  for (uint32_t t = first + threadIdx.x / LANES; t < end; t += kRouteBlock / LANES)
    choose<T, LANES, V>(a, t, threadIdx.x % LANES, counts);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e <= a.n_experts; e += kRouteBlock)
    a.counts[(int64_t)blockIdx.x * (a.n_experts + 1) + e] = counts[e];
}

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(x, d);
    if ((threadIdx.x & 63) >= d) x += y;
  }
  return x;
}

// Block e: the counts of expert e in the blocks before each.
__global__ void __launch_bounds__(64) route_scan_kernel(const RouteArgs a) {
  const uint32_t e = blockIdx.x, pitch = a.n_experts + 1, lane = threadIdx.x;
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < a.blocks; b0 += 64) {
    const uint32_t b = b0 + lane;
    const uint32_t count = b < a.blocks ? a.counts[(int64_t)b * pitch + e] : 0;
    const uint32_t upto = wave_inclusive(count);
    if (b < a.blocks) a.counts[(int64_t)b * pitch + e] = before + upto - count;
    before += __shfl(upto, 63);
  }
  if (lane == 0) a.totals[e] = before;
}

// tokens and slots of a block's assignments, each wave a run of them in its order.
__global__ void __launch_bounds__(kRouteBlock) route_place_kernel(const RouteArgs a) {
  constexpr int kWaves = kRouteBlock / 64;
  __shared__ uint32_t start[kMostExperts + 1];
  __shared__ uint32_t cursor[kWaves][kMostExperts + 1];   // where a wave's next assignment of an expert goes
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, buckets = a.n_experts + 1;
  for (uint32_t e = threadIdx.x; e < kWaves * (kMostExperts + 1); e += kRouteBlock) (&cursor[0][0])[e] = 0;
  if (wave == 0) {
    uint32_t before = 0;
    for (uint32_t e0 = 0; e0 < buckets; e0 += 64) {
      const uint32_t e = e0 + lane, count = e < buckets ? a.totals[e] : 0, upto = wave_inclusive(count);
      if (e < buckets) {
        start[e] = before + upto - count;
        if (blockIdx.x == 0) a.offsets[e] = start[e];
      }
      before += __shfl(upto, 63);
    }
  }
  __syncthreads();
  const uint32_t first = blockIdx.x * a.tokens_per_block * a.n_chosen;
  const uint32_t end = min(a.n, (blockIdx.x + 1) * a.tokens_per_block) * a.n_chosen;
  const uint32_t run = ((end - first + kWaves - 1) / kWaves + 63) / 64 * 64;
  const uint32_t mine = min(end, first + wave * run), mine_end = min(end, mine + run);
  auto bucket_of = [&](uint32_t i) {
    const int32_t e = a.experts[i];
    return e < 0 ? a.n_experts : (uint32_t)e;
  };
  for (uint32_t i = mine + lane; i < mine_end; i += 64) atomicAdd(&cursor[wave][bucket_of(i)], 1u);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < buckets; e += kRouteBlock) {
    uint32_t at = start[e] + a.counts[(int64_t)blockIdx.x * buckets + e];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t count = cursor[w][e];
      cursor[w][e] = at;
      at += count;
    }
  }
  __syncthreads();
  for (uint32_t i0 = mine; i0 < mine_end; i0 += 64) {
    const uint32_t i = i0 + lane;
    const bool in = i < mine_end;
    const uint32_t bucket = in ? bucket_of(i) : 0xffffffffu;
    // the lanes with this bucket
    uint64_t same = __ballot(in);
    for (uint32_t bit = 1; bit < buckets; bit <<= 1) {
      const uint64_t set = __ballot((bucket & bit) != 0);
      same &= bucket & bit ? set : ~set;
    }
    const uint32_t rank = __popcll(same & ((uint64_t(1) << lane) - 1));
    uint32_t at = 0;
    if (in) at = cursor[wave][bucket] + rank;
    __threadfence_block();   // read by all lanes before one of them moves it
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) cursor[wave][bucket] = at + __popcll(same);
    __threadfence_block();
    __builtin_amdgcn_wave_barrier();
    if (in) {
      const bool open = bucket < a.n_experts;
      a.tokens[at] = open ? (int32_t)(i / a.n_chosen) : -1;
      a.slots[i] = open ? (int32_t)at : -1;
    }
  }
}

template <class T, int LANES, int V>
void route_launch(hipStream_t s, const RouteArgs& a) {
  hipLaunchKernelGGL((route_choose_kernel<T, LANES, V>), dim3(a.blocks), dim3(kRouteBlock), 0, s, a);
}

template <class T>
int route_typed(hipStream_t s, RouteArgs a) {
  if (a.n > 0) {
    const uint32_t e = a.n_experts;
    if (e <= 16) route_launch<T, 16, 1>(s, a);
    else if (e <= 32) route_launch<T, 16, 2>(s, a);
    else if (e <= 64) route_launch<T, 16, 4>(s, a);
    else if (e <= 128) route_launch<T, 16, 8>(s, a);
    else if (e <= 256) route_launch<T, 64, 4>(s, a);
    else if (e <= 512) route_launch<T, 64, 8>(s, a);
    else route_launch<T, 64, 16>(s, a);
  }
  hipLaunchKernelGGL(route_scan_kernel, dim3(a.n_experts + 1), dim3(64), 0, s, a);
  hipLaunchKernelGGL(route_place_kernel, dim3(std::max(a.blocks, 1u)), dim3(kRouteBlock), 0, s, a);
  note_kernel("route");
  return after_launch(s);
}

// ------------------------------------------------------------------ gradient of the choice

struct RouteGradientArgs {
  void* logits_gradient;
  const void* weights_gradient;
  const void* weights;
  const int32_t* experts;
  const void* logits;
  int64_t gradient_colstride, colstride;
  uint32_t n, n_experts, n_chosen;
  bool renormalize;
};

// A wave to a token: lane j holds its j-th choice.
template <class T>
__global__ void __launch_bounds__(kRouteBlock) route_gradient_kernel(const RouteGradientArgs a) {
  const uint32_t lane = threadIdx.x & 63, waves = gridDim.x * (kRouteBlock / 64);
  for (uint32_t token = (blockIdx.x * kRouteBlock + threadIdx.x) >> 6; token < a.n; token += waves) {
  const int64_t at = (int64_t)token * a.n_chosen + lane;
  const bool in = lane < a.n_chosen;
  const int32_t expert = in ? a.experts[at] : -1;
  const T weight = in ? static_cast<const T*>(a.weights)[at] : T(0);
  const T dw = in ? static_cast<const T*>(a.weights_gradient)[at] : T(0);
  T common = expert >= 0 ? weight * dw : T(0);
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) common += __shfl_xor(common, m);
  const T taken = a.renormalize ? weight * (dw - common) : weight * dw;
  T* to = static_cast<T*>(a.logits_gradient) + (int64_t)token * a.gradient_colstride;
  const T* row = static_cast<const T*>(a.logits) + (int64_t)token * a.colstride;
  const int32_t first = __shfl(expert, 0);
  const T first_weight = __shfl(weight, 0);
  const bool any = first >= 0 && (uint32_t)first < a.n_experts;
  const T top = any && !a.renormalize ? row[first] : T(0);
  for (uint32_t e0 = 0; e0 < a.n_experts; e0 += 64) {
    const uint32_t e = e0 + lane;
    const bool is = e < a.n_experts;
    T d = 0;
    // the largest logit's weight is one over the sum of all powers
    if (!a.renormalize && any && is) d = -common * (first_weight * (T)exp(row[e] - top));
    for (uint32_t j = 0; j < a.n_chosen; ++j) {
      const int32_t chosen = __shfl(expert, j);
      const T of = __shfl(taken, j);
      if (chosen == (int32_t)e) d += of;
    }
    if (is) to[e] = d;
  }
  }
}

// ------------------------------------------------------------------ combining

struct CombineArgs {
  void* output;               // gradient: of the rows
  void* weights_gradient;
  const void* output_gradient;
  const void* rows;
  const void* weights;
  const int32_t* slots;
  int64_t output_colstride, gradient_colstride, rows_colstride;
  int64_t row_count;
  uint32_t n, n_chosen, width;
};

constexpr int kCombineBlock = 256;
constexpr int kRowsAhead = 4;   // of a token, whose loads are on their way together

// A wave to a part of a token's row: 16 bytes to a lane, kRowsAhead rows of the token at a time.  A lane that would pass the end of the
// row takes its last 16 bytes and stores what lies behind its place.
template <class T, bool kStreaming>
__global__ void __launch_bounds__(kCombineBlock) combine_kernel(const CombineArgs a, uint32_t parts, FastDiv parts_fd) {
  constexpr uint32_t N = Quad<T>::N;
  const uint32_t lane = threadIdx.x & 63, waves = gridDim.x * (kCombineBlock / 64);
  const T* rows = static_cast<const T*>(a.rows);
  const T* weights = static_cast<const T*>(a.weights);
  for (uint64_t unit = (blockIdx.x * kCombineBlock + threadIdx.x) >> 6; unit < (uint64_t)a.n * parts; unit += waves) {
    uint32_t token, part;
    if (parts == 1) token = (uint32_t)unit, part = 0;
    else if (unit < (uint64_t(1) << 31)) parts_fd.divmod((uint32_t)unit, token, part);
    else token = (uint32_t)(unit / parts), part = (uint32_t)(unit % parts);
    const uint32_t place = (part * 64 + lane) * N;
    if (place >= a.width) continue;
    const uint32_t c = a.width >= N ? min(place, a.width - N) : 0, count = min(N, a.width);
    const int64_t first = (int64_t)token * a.n_chosen;
    Quad<T> sum = {};
    for (uint32_t j0 = 0; j0 < a.n_chosen; j0 += kRowsAhead) {
      Quad<T> x[kRowsAhead];
      T w[kRowsAhead];
#pragma unroll
      for (int r = 0; r < kRowsAhead; ++r) {
        const uint32_t j = min(j0 + r, a.n_chosen - 1);
        const int64_t slot = a.slots[first + j];
        const bool in = j0 + r < a.n_chosen && slot >= 0 && slot < a.row_count;
        w[r] = !in ? T(0) : weights ? weights[first + j] : T(1);
        x[r] = Quad<T>{};
        if (!in) continue;
        const T* from = rows + slot * a.rows_colstride + c;
        if (a.width >= N) x[r] = load_quad<kStreaming>(from);
        else
          for (uint32_t e = 0; e < count; ++e) x[r].v[e] = from[e];
      }
#pragma unroll
      for (int r = 0; r < kRowsAhead; ++r)
#pragma unroll
        for (uint32_t e = 0; e < N; ++e) sum.v[e] += w[r] * x[r].v[e];
    }
    T* out = static_cast<T*>(a.output) + (int64_t)token * a.output_colstride;
    if (place + N <= a.width) store_quad<kStreaming>(out + place, sum);
    else {
#pragma unroll
      for (uint32_t e = 0; e < N; ++e)
        if (e < count && c + e >= place) out[c + e] = sum.v[e];
    }
  }
}

// WAVES waves to a token, and its rows kRowsAhead at a time: its gradient is read again from the caches for every such lot.
template <class T, int WAVES, bool kStreaming>
__global__ void __launch_bounds__(kCombineBlock) combine_gradient_kernel(const CombineArgs a) {
  constexpr uint32_t N = Quad<T>::N;
  constexpr int kTokens = kCombineBlock / 64 / WAVES;
  __shared__ T lds[2][kCombineBlock / 64][kRowsAhead];
  int turn = 0;
  const uint32_t wave = threadIdx.x >> 6, of_token = threadIdx.x % (64 * WAVES), stride = 64 * WAVES * N;
  const T* weights = static_cast<const T*>(a.weights);
  // all of a block's waves go on together: a token beyond the last one is the last one, and not stored
  for (uint32_t t0 = blockIdx.x * kTokens; t0 < a.n; t0 += gridDim.x * kTokens) {
    const uint32_t token = min(t0 + wave / WAVES, a.n - 1);
    const bool mine = t0 + wave / WAVES < a.n;
    const int64_t first = (int64_t)token * a.n_chosen;
    const T* dy = static_cast<const T*>(a.output_gradient) + (int64_t)token * a.gradient_colstride;
    for (uint32_t j0 = 0; j0 < a.n_chosen; j0 += kRowsAhead) {
      T dot[kRowsAhead], w[kRowsAhead];
      int64_t slot[kRowsAhead];
#pragma unroll
      for (int r = 0; r < kRowsAhead; ++r) {
        const uint32_t j = min(j0 + r, a.n_chosen - 1);
        slot[r] = a.slots[first + j];
        if (!mine || j0 + r >= a.n_chosen || slot[r] < 0 || slot[r] >= a.row_count) slot[r] = -1;
        w[r] = weights ? weights[first + j] : T(1);
        dot[r] = 0;
      }
      for (uint32_t place = of_token * N; place < a.width; place += stride) {
        const uint32_t c = a.width >= N ? min(place, a.width - N) : 0, count = min(N, a.width);
        Quad<T> g = {}, x[kRowsAhead];
        if (a.width >= N) g = load_quad(dy + c);
        else
          for (uint32_t e = 0; e < count; ++e) g.v[e] = dy[c + e];
#pragma unroll
        for (int r = 0; r < kRowsAhead; ++r) {
          x[r] = Quad<T>{};
          if (slot[r] < 0 || !a.weights_gradient) continue;
          const T* from = static_cast<const T*>(a.rows) + slot[r] * a.rows_colstride + c;
          if (a.width >= N) x[r] = load_quad<kStreaming>(from);
          else
            for (uint32_t e = 0; e < count; ++e) x[r].v[e] = from[e];
        }
        const bool whole = place + N <= a.width;
#pragma unroll
        for (int r = 0; r < kRowsAhead; ++r) {
          if (slot[r] < 0) continue;
          if (a.output) {
            T* to = static_cast<T*>(a.output) + slot[r] * a.output_colstride;
            Quad<T> q;
#pragma unroll
            for (uint32_t e = 0; e < N; ++e) q.v[e] = w[r] * g.v[e];
            if (whole) store_quad<kStreaming>(to + place, q);
            else {
#pragma unroll
              for (uint32_t e = 0; e < N; ++e)
                if (e < count && c + e >= place) to[c + e] = q.v[e];
            }
          }
#pragma unroll
          for (uint32_t e = 0; e < N; ++e) dot[r] += c + e >= place ? g.v[e] * x[r].v[e] : T(0);
        }
      }
      if (!a.weights_gradient) continue;
#pragma unroll
      for (int m = 32; m > 0; m >>= 1)
#pragma unroll
        for (int r = 0; r < kRowsAhead; ++r) dot[r] += __shfl_xor(dot[r], m);
      T* to = static_cast<T*>(a.weights_gradient) + first + j0;
      const uint32_t j = threadIdx.x & 63;
      if constexpr (WAVES == 1) {
#pragma unroll
        for (int r = 0; r < kRowsAhead; ++r)
          if (mine && j == (uint32_t)r && j0 + r < a.n_chosen) to[r] = dot[r];
      } else {
        if (j == 0) {
#pragma unroll
          for (int r = 0; r < kRowsAhead; ++r) lds[turn][wave][r] = dot[r];
        }
        __syncthreads();
        if (mine && wave % WAVES == 0 && j < kRowsAhead && j0 + j < a.n_chosen) {
          T sum = lds[turn][wave][j];
#pragma unroll
          for (int v = 1; v < WAVES; ++v) sum += lds[turn][wave + v][j];
          to[j] = sum;
        }
        turn ^= 1;   // written again only after another barrier
      }
    }
  }
}

template <class T>
void combine_launch(hipStream_t s, const CombineArgs& a) {
  constexpr int64_t kWaves = kCombineBlock / 64;
  const uint32_t parts = (a.width + 64 * Quad<T>::N - 1) / (64 * Quad<T>::N);
  const int64_t blocks = std::min<int64_t>(((int64_t)a.n * parts + kWaves - 1) / kWaves, kMostBlocks);
  const bool past = (int64_t)a.n * (a.n_chosen + 1) * a.width * (int64_t)sizeof(T) > kCombineCacheBytes;
  if (past) hipLaunchKernelGGL((combine_kernel<T, true>), dim3((uint32_t)blocks), dim3(kCombineBlock), 0, s, a, parts, FastDiv(parts));
  else hipLaunchKernelGGL((combine_kernel<T, false>), dim3((uint32_t)blocks), dim3(kCombineBlock), 0, s, a, parts, FastDiv(parts));
}

template <class T>
void combine_gradient_launch(hipStream_t s, const CombineArgs& a) {
  const bool past = (int64_t)a.n * (2 * a.n_chosen + 1) * a.width * (int64_t)sizeof(T) > kCombineCacheBytes;
  // a wave to a token, four where that leaves compute units without work
  const bool few = a.n < 4096 && a.width > 256;
  const int64_t blocks = std::min<int64_t>(few ? a.n : (a.n + 3) / 4, kMostBlocks);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kCombineBlock), 0, s, a); };
  if (few && past) launch(combine_gradient_kernel<T, 4, true>);
  else if (few) launch(combine_gradient_kernel<T, 4, false>);
  else if (past) launch(combine_gradient_kernel<T, 1, true>);
  else launch(combine_gradient_kernel<T, 1, false>);
}

constexpr int64_t kMostRows = (int64_t(1) << 31) - 1;

}  // namespace

#define CT_FLOATING(name) CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, name ": datatype must be float or double")

extern "C" {

int ct_route_experts(void* stream, int32_t* experts, void* weights, int32_t* offsets, int32_t* tokens, int32_t* slots,
                     const void* logits, int64_t logits_colstride, int64_t n, int64_t n_experts, int64_t n_chosen,
                     int renormalize, int dtype) {
  CT_FLOATING("ct_route_experts");
  CT_REQUIRE(n >= 0, "ct_route_experts: negative count");
  CT_REQUIRE(n_experts >= 1 && n_experts <= kMostExperts, "ct_route_experts: %lld experts, 1 to %d are taken", (long long)n_experts,
             kMostExperts);
  CT_REQUIRE(n_chosen >= 1 && n_chosen <= std::min<int64_t>(n_experts, kMostChosen),
             "ct_route_experts: %lld chosen of %lld experts, 1 to %d are taken", (long long)n_chosen, (long long)n_experts, kMostChosen);
  CT_REQUIRE(n <= kMostRows / n_chosen, "ct_route_experts: %lld tokens", (long long)n);
  CT_REQUIRE(offsets && (n == 0 || (experts && weights && tokens && slots && logits)), "ct_route_experts: null buffer");
  CT_REQUIRE(logits_colstride >= n_experts, "ct_route_experts: column stride %lld below the row's length", (long long)logits_colstride);
  hipStream_t s = static_cast<hipStream_t>(stream);
  RouteArgs a{};
  a.experts = experts; a.weights = weights; a.offsets = offsets; a.tokens = tokens; a.slots = slots; a.logits = logits;
  a.colstride = logits_colstride;
  a.n = (uint32_t)n; a.n_experts = (uint32_t)n_experts; a.n_chosen = (uint32_t)n_chosen;
  a.renormalize = renormalize != 0;
  // 64 tokens to a block, more where the blocks' counts would take more than 8 MiB
  const int64_t most_blocks = std::max<int64_t>(1, (int64_t(2) << 20) / (n_experts + 1));
  a.tokens_per_block = (uint32_t)std::max<int64_t>(64, (n + most_blocks - 1) / most_blocks);
  a.blocks = (uint32_t)((n + a.tokens_per_block - 1) / a.tokens_per_block);
  void* scratch = nullptr;
  if (int rc = stream_scratch(s, ((size_t)a.blocks + 1) * (n_experts + 1) * sizeof(int32_t), &scratch)) return rc;
  a.totals = static_cast<int32_t*>(scratch);
  a.counts = a.totals + n_experts + 1;
  return dtype == CT_F32 ? route_typed<float>(s, a) : route_typed<double>(s, a);
}

int ct_route_experts_gradient(void* stream, void* logits_gradient, int64_t logits_gradient_colstride,
                              const void* weights_gradient, const void* weights, const int32_t* experts, const void* logits,
                              int64_t logits_colstride, int64_t n, int64_t n_experts, int64_t n_chosen, int renormalize,
                              int dtype) {
  CT_FLOATING("ct_route_experts_gradient");
  CT_REQUIRE(n >= 0, "ct_route_experts_gradient: negative count");
  CT_REQUIRE(n_experts >= 1 && n_experts <= kMostExperts && n_chosen >= 1 && n_chosen <= std::min<int64_t>(n_experts, kMostChosen),
             "ct_route_experts_gradient: %lld chosen of %lld experts", (long long)n_chosen, (long long)n_experts);
  CT_REQUIRE(n <= kMostRows / n_chosen, "ct_route_experts_gradient: %lld tokens", (long long)n);
  if (n == 0) return CT_OK;
  CT_REQUIRE(logits_gradient && weights_gradient && weights && experts && (renormalize || logits),
             "ct_route_experts_gradient: null buffer");
  CT_REQUIRE(logits_gradient_colstride >= n_experts && (renormalize || logits_colstride >= n_experts),
             "ct_route_experts_gradient: a column stride below the row's length");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const RouteGradientArgs a{logits_gradient, weights_gradient, weights, experts, logits, logits_gradient_colstride,
                            logits_colstride, (uint32_t)n, (uint32_t)n_experts, (uint32_t)n_chosen, renormalize != 0};
  const dim3 grid((uint32_t)std::min<int64_t>((n + kRouteBlock / 64 - 1) / (kRouteBlock / 64), kMostBlocks));
  if (dtype == CT_F32) hipLaunchKernelGGL((route_gradient_kernel<float>), grid, dim3(kRouteBlock), 0, s, a);
  else hipLaunchKernelGGL((route_gradient_kernel<double>), grid, dim3(kRouteBlock), 0, s, a);
  note_kernel("route_gradient");
  return after_launch(s);
}

int ct_combine_experts(void* stream, void* output, int64_t output_colstride, const void* rows, int64_t row_count,
                       int64_t rows_colstride, const void* weights, const int32_t* slots, int64_t n, int64_t n_chosen,
                       int64_t width, int dtype) {
  CT_FLOATING("ct_combine_experts");
  CT_REQUIRE(n >= 0 && width >= 0 && row_count >= 0 && row_count <= kMostRows && width <= kMostRows, "ct_combine_experts: bad extent");
  CT_REQUIRE(n_chosen >= 1 && n_chosen <= kMostChosen, "ct_combine_experts: %lld chosen, 1 to %d are taken", (long long)n_chosen, kMostChosen);
  CT_REQUIRE(n <= kMostRows / n_chosen, "ct_combine_experts: %lld tokens", (long long)n);
  if (n == 0 || width == 0) return CT_OK;
  CT_REQUIRE(output && slots && (rows || row_count == 0), "ct_combine_experts: null buffer");
  CT_REQUIRE(output_colstride >= width && rows_colstride >= width, "ct_combine_experts: a column stride below the row's length");
  CT_REQUIRE(!rows_meet({output, n, width, output_colstride}, {rows, row_count, width, rows_colstride}, dtype_size(dtype)),
             "ct_combine_experts: output and rows overlap");
  hipStream_t s = static_cast<hipStream_t>(stream);
  CombineArgs a{};
  a.output = output; a.rows = rows; a.weights = weights; a.slots = slots;
  a.output_colstride = output_colstride; a.rows_colstride = rows_colstride; a.row_count = row_count;
  a.n = (uint32_t)n; a.n_chosen = (uint32_t)n_chosen; a.width = (uint32_t)width;
  if (dtype == CT_F32) combine_launch<float>(s, a);
  else combine_launch<double>(s, a);
  note_kernel("combine");
  return after_launch(s);
}

int ct_combine_experts_gradient(void* stream, void* rows_gradient, int64_t rows_gradient_colstride, void* weights_gradient,
                                const void* output_gradient, int64_t output_gradient_colstride, const void* rows,
                                int64_t row_count, int64_t rows_colstride, const void* weights, const int32_t* slots,
                                int64_t n, int64_t n_chosen, int64_t width, int dtype) {
  CT_FLOATING("ct_combine_experts_gradient");
  CT_REQUIRE(n >= 0 && width >= 0 && row_count >= 0 && row_count <= kMostRows && width <= kMostRows,
             "ct_combine_experts_gradient: bad extent");
  CT_REQUIRE(n_chosen >= 1 && n_chosen <= kMostChosen, "ct_combine_experts_gradient: %lld chosen, 1 to %d are taken",
             (long long)n_chosen, kMostChosen);
  CT_REQUIRE(n <= kMostRows / n_chosen, "ct_combine_experts_gradient: %lld tokens", (long long)n);
  if (n == 0 || (!rows_gradient && !weights_gradient)) return CT_OK;
  CT_REQUIRE(slots && (width == 0 || (output_gradient && (!weights_gradient || rows || row_count == 0))),
             "ct_combine_experts_gradient: null buffer");
  CT_REQUIRE(output_gradient_colstride >= width && (!rows_gradient || rows_gradient_colstride >= width) &&
                 (!weights_gradient || rows_colstride >= width),
             "ct_combine_experts_gradient: a column stride below the row's length");
  const RowRange result{rows_gradient, row_count, width, rows_gradient_colstride};
  CT_REQUIRE(!rows_meet(result, {output_gradient, n, width, output_gradient_colstride}, dtype_size(dtype)) &&
                 !rows_meet(result, {weights_gradient ? rows : nullptr, row_count, width, rows_colstride}, dtype_size(dtype)),
             "ct_combine_experts_gradient: rows_gradient overlaps an operand");
  hipStream_t s = static_cast<hipStream_t>(stream);
  CombineArgs a{};
  a.output = rows_gradient; a.weights_gradient = weights_gradient; a.output_gradient = output_gradient; a.rows = rows;
  a.weights = weights; a.slots = slots;
  a.output_colstride = rows_gradient_colstride; a.gradient_colstride = output_gradient_colstride; a.rows_colstride = rows_colstride;
  a.row_count = row_count;
  a.n = (uint32_t)n; a.n_chosen = (uint32_t)n_chosen; a.width = (uint32_t)width;
  if (dtype == CT_F32) combine_gradient_launch<float>(s, a);
  else combine_gradient_launch<double>(s, a);
  note_kernel("combine_gradient");
  return after_launch(s);
}

}  // extern "C"
