// ops_experts.hip -- the choice of experts, the order of rows by expert, and the sum of a token's rows.
//
// Routing.  A group of lanes holds a token's logits in registers and takes the largest n_chosen times; ties go to the lowest
// index.  Logits are compared as integers that order as they do, NaN above all, -infinity below every one that may be chosen.
// The order of rows is a stable counting sort of the assignments (t, j) by expert: blocks of consecutive tokens count their
// assignments, one block to an expert adds the blocks' counts up, and each block then knows the place of its own.  The choice is bound by its
// instructions, some hundred to a choice of a wave's four tokens: 65536 tokens, 8 of 128 experts, 28 us of 41 (57 in double); 14 for the gradient, which is
// bound by memory.
//
// Combining reads the rows of a token once and writes its sum; its gradient reads each row once, the token's gradient once for each of
// them, out of the caches from the second time on, and writes as many rows.  Memory bounds both: 16384 tokens of 4 rows of 1000 floats 69 us
// (4.8 TB/s) and 109 to 118 (5.0 to 5.4).
#include <algorithm>

#include "elementwise.h"
#include "rows.h"

using namespace cthip;

namespace {

constexpr int kRouteBlock = 256, kFewBlock = 1024;
constexpr uint32_t kFewBlocks = 64;   // whose counts each adds up itself, rather than a launch between (1024 tokens of 128 experts: 9.7 us, were 12.5)
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

// ------------------------------------------------------------------ reductions over the lanes of a token

// The value `step` lanes further on in a row of 16, around its end: no trip through LDS.
template <int step> __device__ __forceinline__ uint32_t rotated(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + step, 0xf, 0xf, true);
}
template <int step> __device__ __forceinline__ uint64_t rotated(uint64_t x) {
  return (uint64_t)rotated<step>((uint32_t)x) | (uint64_t)rotated<step>((uint32_t)(x >> 32)) << 32;
}
template <int step> __device__ __forceinline__ float rotated(float x) { return __builtin_bit_cast(float, rotated<step>(__builtin_bit_cast(uint32_t, x))); }
template <int step> __device__ __forceinline__ double rotated(double x) { return __builtin_bit_cast(double, rotated<step>(__builtin_bit_cast(uint64_t, x))); }

// f over the LANES (16 or 64) lanes of a token, in all of them.
template <int LANES, class X, class F>
__device__ __forceinline__ X over_lanes(X x, F f) {
  x = f(x, rotated<8>(x));
  x = f(x, rotated<4>(x));
  x = f(x, rotated<2>(x));
  x = f(x, rotated<1>(x));
  if constexpr (LANES == 64) {
    x = f(x, __shfl_xor(x, 16));
    x = f(x, __shfl_xor(x, 32));
  }
  return x;
}

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
  int32_t* counts;   // [n_experts + 1][blocks]; then, in place, of all blocks before
  int32_t* totals;   // [n_experts + 1]
};

// experts and weights of one token by LANES lanes, V logits to each (lane + v * LANES).
template <class T, int LANES, int V>
__device__ __forceinline__ void choose(const RouteArgs& a, uint32_t token, uint32_t lane, uint32_t* counts) {
  using Key = typename KeyOf<T>::Key;
  constexpr int kMine = kMostChosen / LANES + (kMostChosen % LANES > 0);   // choices that a lane keeps: j % LANES is its own
  const T* row = static_cast<const T*>(a.logits) + (int64_t)token * a.colstride;
  T x[V];
  Key key[V];
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = row[min(lane + v * LANES, a.n_experts - 1)];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (lane + v * LANES >= a.n_experts) x[v] = -__builtin_inf();
    key[v] = key_of<T>(x[v]);
    if (key[v] <= closed_key<T>()) key[v] = 0;
  }
  T top = 0, sum = 0;
  uint32_t found = 0;
  T power_of[kMine] = {};
  int32_t expert_of[kMine];
#pragma unroll
  for (int q = 0; q < kMine; ++q) expert_of[q] = -1;
  for (uint32_t j = 0; j < a.n_chosen; ++j) {
    Key best = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) best = max(best, key[v]);
    best = over_lanes<LANES>(best, [](Key x, Key y) { return x > y ? x : y; });
    uint32_t index = 0xffffffffu;   // the lowest that has it
#pragma unroll
    for (int v = V - 1; v >= 0; --v) index = key[v] == best ? lane + v * LANES : index;
    index = over_lanes<LANES>(index, [](uint32_t x, uint32_t y) { return min(x, y); });
    const bool any = best != 0;
    const T value = of_key<T>(best);
    if (j == 0) top = value;
    const T power = any ? (T)exp(value - top) : T(0);
    sum += power;
    found += any;
#pragma unroll
    for (int q = 0; q < kMine; ++q)
      if (j == lane + q * LANES) {
        power_of[q] = power;
        expert_of[q] = any ? (int32_t)index : -1;
      }
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = index == lane + v * LANES ? Key(0) : key[v];
  }
  if (!a.renormalize) {
    sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) sum += (T)exp(x[v] - top);   // of a row without an open expert: not used
    sum = over_lanes<LANES>(sum, [](T x, T y) { return x + y; });
  }
  const int64_t at = (int64_t)token * a.n_chosen;
#pragma unroll
  for (int q = 0; q < kMine; ++q) {
    const uint32_t j = lane + q * LANES;
    if (j >= a.n_chosen) continue;
    a.experts[at + j] = expert_of[q];
    static_cast<T*>(a.weights)[at + j] = j < found ? power_of[q] / sum : T(0);
    atomicAdd(&counts[expert_of[q] < 0 ? a.n_experts : (uint32_t)expert_of[q]], 1u);
  }
}

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t x) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(x, d);
    if ((threadIdx.x & 63) >= d) x += y;
  }
  return x;
}

constexpr int kRouteWaves = kRouteBlock / 64;

// What a block keeps in LDS to place its assignments: where each expert's begin, and where a wave's next one of each goes.
struct PlaceLds {
  uint32_t start[kMostExperts + 1];
  uint32_t cursor[kRouteWaves][kMostExperts + 1];
};

// The assignments of each expert begin where those of the ones before end.  By the first wave; `offsets` where they are stored.
template <class Total>
__device__ __forceinline__ void begin_experts(const RouteArgs& a, PlaceLds& lds, Total total, bool store) {
  const uint32_t lane = threadIdx.x & 63, buckets = a.n_experts + 1;
  if (threadIdx.x >= 64) return;
  uint32_t before = 0;
  for (uint32_t e0 = 0; e0 < buckets; e0 += 64) {
    const uint32_t e = e0 + lane, count = e < buckets ? total(e) : 0, upto = wave_inclusive(count);
    if (e < buckets) {
      lds.start[e] = before + upto - count;
      if (store) a.offsets[e] = (int32_t)lds.start[e];
    }
    before += __shfl(upto, 63);
  }
}

// tokens and slots of assignments first .. end - 1, each wave a run of them in its order; before(e): those of expert e ahead of
// `first`.
template <int kThreads, class Before>
__device__ __forceinline__ void place(const RouteArgs& a, PlaceLds& lds, uint32_t first, uint32_t end, Before before) {
  const uint32_t lane = threadIdx.x & 63, wave = min(threadIdx.x >> 6, (uint32_t)kRouteWaves), buckets = a.n_experts + 1;   // later waves: no run
  for (uint32_t e = threadIdx.x; e < buckets; e += kThreads)
#pragma unroll
    for (int w = 0; w < kRouteWaves; ++w) lds.cursor[w][e] = 0;
  __syncthreads();
  const uint32_t run = ((end - first + kRouteWaves - 1) / kRouteWaves + 63) / 64 * 64;
  const uint32_t mine = min(end, first + wave * run), mine_end = wave < kRouteWaves ? min(end, mine + run) : mine;
  auto bucket_of = [&](uint32_t i) {
    const int32_t e = a.experts[i];
    return e < 0 ? a.n_experts : (uint32_t)e;
  };
  for (uint32_t i = mine + lane; i < mine_end; i += 64) atomicAdd(&lds.cursor[wave][bucket_of(i)], 1u);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < buckets; e += kThreads) {
    uint32_t at = lds.start[e] + before(e);
#pragma unroll
    for (int w = 0; w < kRouteWaves; ++w) {
      const uint32_t count = lds.cursor[w][e];
      lds.cursor[w][e] = at;
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
    if (in) at = lds.cursor[wave][bucket] + rank;
    __threadfence_block();   // read by all lanes before one of them moves it
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) lds.cursor[wave][bucket] = at + __popcll(same);
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
__global__ void __launch_bounds__(kRouteBlock) route_choose_kernel(const RouteArgs a) {
  __shared__ uint32_t counts[kMostExperts + 1];
  for (uint32_t e = threadIdx.x; e <= a.n_experts; e += kRouteBlock) counts[e] = 0;
  __syncthreads();
  const uint32_t first = blockIdx.x * a.tokens_per_block, end = min(a.n, first + a.tokens_per_block);
  for (uint32_t t = first + threadIdx.x / LANES; t < end; t += kRouteBlock / LANES)
    choose<T, LANES, V>(a, t, threadIdx.x % LANES, counts);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e <= a.n_experts; e += kRouteBlock) a.counts[(int64_t)e * a.blocks + blockIdx.x] = counts[e];
}

// Block e: the counts of expert e in the blocks before each.
__global__ void __launch_bounds__(kRouteBlock) route_scan_kernel(const RouteArgs a) {
  __shared__ uint32_t of_waves[kRouteWaves];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t* counts = a.counts + (int64_t)blockIdx.x * a.blocks;
  constexpr uint32_t kEach = 4;
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < a.blocks; b0 += kRouteBlock * kEach) {
    const uint32_t b = b0 + threadIdx.x * kEach;
    uint32_t count[kEach], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      count[i] = b + i < a.blocks ? counts[b + i] : 0;
      sum += count[i];
    }
    const uint32_t upto = wave_inclusive(sum);
    __syncthreads();
    if (lane == 63) of_waves[wave] = upto;
    __syncthreads();
    uint32_t at = before + upto - sum;
#pragma unroll
    for (uint32_t w = 0; w < kRouteWaves; ++w) {
      if (w < wave) at += of_waves[w];
      before += of_waves[w];
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      if (b + i < a.blocks) counts[b + i] = (int32_t)at;
      at += count[i];
    }
  }
  if (threadIdx.x == 0) a.totals[blockIdx.x] = (int32_t)before;
}

// kScan: a block adds up the counts of all blocks itself, and of those before it.
template <bool kScan>
__global__ void __launch_bounds__(kRouteBlock) route_place_kernel(const RouteArgs a) {
  __shared__ PlaceLds lds;
  __shared__ uint32_t totals[kScan ? kMostExperts + 1 : 1], befores[kScan ? kMostExperts + 1 : 1];
  if constexpr (kScan) {
    for (uint32_t e = threadIdx.x; e <= a.n_experts; e += kRouteBlock) {
      const int32_t* counts = a.counts + (int64_t)e * a.blocks;
      uint32_t total = 0, before = 0;
#pragma unroll 8
      for (uint32_t b = 0; b < a.blocks; ++b) {
        const uint32_t count = (uint32_t)counts[b];
        total += count;
        before += b < blockIdx.x ? count : 0;
      }
      totals[e] = total;
      befores[e] = before;
    }
    __syncthreads();
  }
  begin_experts(a, lds, [&](uint32_t e) { return kScan ? totals[e] : (uint32_t)a.totals[e]; }, blockIdx.x == 0);
  const uint32_t first = blockIdx.x * a.tokens_per_block * a.n_chosen;
  const uint32_t end = min(a.n, (blockIdx.x + 1) * a.tokens_per_block) * a.n_chosen;
  place<kRouteBlock>(a, lds, first, end, [&](uint32_t e) { return kScan ? befores[e] : (uint32_t)a.counts[(int64_t)e * a.blocks + blockIdx.x]; });
}

// A few tokens: all of it in one block.
template <class T, int LANES, int V>
__global__ void __launch_bounds__(kFewBlock) route_few_kernel(const RouteArgs a) {
  __shared__ uint32_t counts[kMostExperts + 1];
  __shared__ PlaceLds lds;
  for (uint32_t e = threadIdx.x; e <= a.n_experts; e += kFewBlock) counts[e] = 0;
  __syncthreads();
  for (uint32_t t = threadIdx.x / LANES; t < a.n; t += kFewBlock / LANES) choose<T, LANES, V>(a, t, threadIdx.x % LANES, counts);
  __threadfence_block();   // the experts are read again by other lanes
  __syncthreads();
  begin_experts(a, lds, [&](uint32_t e) { return counts[e]; }, true);
  place<kFewBlock>(a, lds, 0, a.n * a.n_chosen, [](uint32_t) { return 0u; });
}

// What one block does in less time than two launches take.  Us of one block, and of two launches: 32 tokens, 8 of 128 experts, 6.3 and
// 8.0; 64 tokens, 8 of 128, 9.2 and 8.3; 8 tokens, 8 of 506, 8.3 and 12.7; 32 tokens, 8 of 506, 16.0 and 14.0.
bool is_few(int64_t n, int64_t n_experts, int64_t n_chosen, int64_t size) {
  return n_experts <= (size == 8 ? 128 : 256) ? n <= 64 && n * n_chosen <= 256 : n <= 32 && n * n_chosen <= 64;
}

template <class T, int LANES, int V>
void route_launch(hipStream_t s, const RouteArgs& a, bool few) {
  if (few) hipLaunchKernelGGL((route_few_kernel<T, LANES, V>), dim3(1), dim3(kFewBlock), 0, s, a);
  else hipLaunchKernelGGL((route_choose_kernel<T, LANES, V>), dim3(a.blocks), dim3(kRouteBlock), 0, s, a);
}

// The lanes of a token: 16, so that a wave works on four, as long as they have registers for its logits; a block of 1024 has fewer.
// (65536 tokens, 8 of 256: 48 us, with 64 lanes 88; 4096 tokens 16 and 57.)
template <class T>
int route_typed(hipStream_t s, RouteArgs a) {
  const uint32_t e = a.n_experts;
  const bool few = is_few(a.n, e, a.n_chosen, sizeof(T));
  if (e <= 16) route_launch<T, 16, 1>(s, a, few);
  else if (e <= 32) route_launch<T, 16, 2>(s, a, few);
  else if (e <= 64) route_launch<T, 16, 4>(s, a, few);
  else if (e <= 128) route_launch<T, 16, 8>(s, a, few);
  else if (e <= 256 && few && sizeof(T) == 8) hipLaunchKernelGGL((route_few_kernel<T, 64, 4>), dim3(1), dim3(kFewBlock), 0, s, a);
  else if (e <= 256) route_launch<T, 16, 16>(s, a, few);
  else if (e <= 512 && few) hipLaunchKernelGGL((route_few_kernel<T, 64, 8>), dim3(1), dim3(kFewBlock), 0, s, a);
  else if (e <= 512) hipLaunchKernelGGL((route_choose_kernel<T, 16, 32>), dim3(a.blocks), dim3(kRouteBlock), 0, s, a);
  else route_launch<T, 64, 16>(s, a, few);
  if (!few && a.blocks <= kFewBlocks) {
    hipLaunchKernelGGL(route_place_kernel<true>, dim3(a.blocks), dim3(kRouteBlock), 0, s, a);
  } else if (!few) {
    hipLaunchKernelGGL(route_scan_kernel, dim3(a.n_experts + 1), dim3(kRouteBlock), 0, s, a);
    hipLaunchKernelGGL(route_place_kernel<false>, dim3(a.blocks), dim3(kRouteBlock), 0, s, a);
  }
  note_kernel(few ? "route_few" : "route");
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

// 16 bytes of a row to a lane: the ones at its place, or the row's last ones if those would pass its end; rows shorter than
// that element by element.
template <class T>
struct RowPart {
  static constexpr uint32_t N = Quad<T>::N;
  uint32_t place, start, width;
  __device__ __forceinline__ RowPart(uint32_t place, uint32_t width) : place(place), start(width >= N ? min(place, width - N) : 0), width(width) {}
  __device__ __forceinline__ bool owns(uint32_t e) const { return start + e >= place && (width >= N || e < width); }
  template <bool kStreaming> __device__ __forceinline__ Quad<T> load(const T* row) const {
    if (width >= N) return load_quad<kStreaming>(row + start);
    Quad<T> q;
#pragma unroll
    for (uint32_t e = 0; e < N; ++e) q.v[e] = row[min(e, width - 1)];
    return q;
  }
  template <bool kStreaming> __device__ __forceinline__ void store(T* row, const Quad<T>& q) const {
    if (place + N <= width) {
      store_quad<kStreaming>(row + place, q);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < N; ++e)
        if (owns(e)) row[start + e] = q.v[e];
    }
  }
};

// LANES lanes to a token, as many as it has choices or more; lane j holds its j-th choice.  The chosen ones' gradients reach the lanes
// that store them through a row in LDS, zeros elsewhere.
template <class T, int LANES>
__global__ void __launch_bounds__(kRouteBlock) route_gradient_kernel(const RouteGradientArgs a) {
  extern __shared__ __attribute__((aligned(16))) char row_lds[];
  const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES, groups = kRouteBlock / LANES;
  T* taken_of = reinterpret_cast<T*>(row_lds) + group * a.n_experts;
  for (uint32_t e = lane; e < a.n_experts; e += LANES) taken_of[e] = 0;
  const uint32_t rounds = (a.n + gridDim.x * groups - 1) / (gridDim.x * groups);
  for (uint32_t i = 0; i < rounds; ++i) {
    const uint32_t unit = (i * gridDim.x + blockIdx.x) * groups + group, token = min(unit, a.n - 1);   // beyond the last one: not stored
    const int64_t at = (int64_t)token * a.n_chosen + min(lane, a.n_chosen - 1);
    const int32_t expert = a.experts[at];
    const bool in = lane < a.n_chosen && expert >= 0 && (uint32_t)expert < a.n_experts;
    const T weight = static_cast<const T*>(a.weights)[at];
    const T dw = static_cast<const T*>(a.weights_gradient)[at];
    T common = in ? weight * dw : T(0);
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) common += __shfl_xor(common, m);
    if (in) taken_of[expert] = a.renormalize ? weight * (dw - common) : weight * dw;
    __threadfence_block();
    __builtin_amdgcn_wave_barrier();   // a token's lanes are one wave's
    const int32_t first = __shfl(expert, 0, LANES);
    const T first_weight = __shfl(weight, 0, LANES);
    const bool any = first >= 0 && (uint32_t)first < a.n_experts;
    const T* row = static_cast<const T*>(a.logits) + (int64_t)token * a.colstride;
    const T top = any && !a.renormalize ? row[first] : T(0);
    T* to = static_cast<T*>(a.logits_gradient) + (int64_t)token * a.gradient_colstride;
    for (uint32_t place = lane * Quad<T>::N; place < a.n_experts; place += LANES * Quad<T>::N) {
      const RowPart<T> part(place, a.n_experts);
      Quad<T> q;
#pragma unroll
      for (uint32_t e = 0; e < Quad<T>::N; ++e) q.v[e] = taken_of[min(part.start + e, a.n_experts - 1)];
      if (!a.renormalize && any) {
        const Quad<T> x = part.template load<false>(row);
        // the largest logit's weight is one over the sum of all powers
#pragma unroll
        for (uint32_t e = 0; e < Quad<T>::N; ++e) q.v[e] -= common * (first_weight * (T)exp(x.v[e] - top));
      }
      if (unit < a.n) part.template store<false>(to, q);
    }
    __threadfence_block();
    __builtin_amdgcn_wave_barrier();
    if (in) taken_of[expert] = 0;
  }
}

template <class T>
void route_gradient_launch(hipStream_t s, const RouteGradientArgs& a) {
  constexpr uint32_t N = Quad<T>::N;
  const uint32_t lanes = std::max((a.n_experts + N - 1) / N, a.n_chosen);
  auto launch = [&](auto of_lanes) {
    constexpr uint32_t L = decltype(of_lanes)::value, kGroups = kRouteBlock / L;
    const uint32_t blocks = (uint32_t)std::min<int64_t>((a.n + kGroups - 1) / kGroups, 2048);
    hipLaunchKernelGGL((route_gradient_kernel<T, L>), dim3(blocks), dim3(kRouteBlock), kGroups * a.n_experts * sizeof(T), s, a);
  };
  if (lanes <= 8) launch(std::integral_constant<uint32_t, 8>());
  else if (lanes <= 16) launch(std::integral_constant<uint32_t, 16>());
  else if (lanes <= 32) launch(std::integral_constant<uint32_t, 32>());
  else launch(std::integral_constant<uint32_t, 64>());
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

template <class T> __device__ __forceinline__ T from_lane(T x, uint32_t lane) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
  } else {
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    const uint64_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, lane);
    return __builtin_bit_cast(T, low | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane) << 32);
  }
}

// A wave to a run of tokens and 64 x 16 bytes of their rows.  The slots and weights of up to 64 assignments are one load of the
// wave's, and the rows of kRowsAhead assignments are on their way together, whichever tokens they are of: waves that took a
// token each spent their time on two loads, one behind the other (65536 tokens of one row of 1 KiB 42 us).
constexpr int kRowsAhead = 8;

template <class T, bool kStreaming>
__global__ void __launch_bounds__(kCombineBlock) combine_kernel(const CombineArgs a, uint32_t parts, uint32_t run, uint32_t units) {
  const uint32_t lane = threadIdx.x & 63, unit = __builtin_amdgcn_readfirstlane((blockIdx.x * kCombineBlock + threadIdx.x) >> 6);
  if (unit >= units) return;
  const uint32_t runs = unit / parts, part = unit - runs * parts, k = a.n_chosen;
  const RowPart<T> at((part * 64 + lane) * Quad<T>::N, a.width);
  const T* rows = static_cast<const T*>(a.rows);
  T* out = static_cast<T*>(a.output);
  const uint64_t begin = (uint64_t)runs * run;
  const uint32_t tokens = (uint32_t)min((uint64_t)run, a.n - begin);
  Quad<T> sum = {};
  for (uint32_t t0 = 0; t0 < tokens;) {
    const uint32_t now = min(64 / k, tokens - t0), count = now * k;   // tokens, assignments
    const int64_t first = (int64_t)(begin + t0) * k;
    const int64_t mine = first + min(lane, count - 1);
    const int32_t slot = a.slots[mine];
    const T weight = a.weights ? static_cast<const T*>(a.weights)[mine] : T(1);
    uint32_t left = k, token = t0;
    for (uint32_t i0 = 0; i0 < count; i0 += kRowsAhead) {
      Quad<T> x[kRowsAhead];
      bool in[kRowsAhead];
#pragma unroll
      for (uint32_t r = 0; r < kRowsAhead; ++r) {
        const int32_t of = __builtin_amdgcn_readlane(slot, min(i0 + r, count - 1));
        in[r] = i0 + r < count && of >= 0 && of < a.row_count;
        if (in[r]) x[r] = at.template load<kStreaming>(rows + (int64_t)of * a.rows_colstride);
      }
#pragma unroll
      for (uint32_t r = 0; r < kRowsAhead; ++r) {
        if (i0 + r >= count) break;
        if (in[r]) {
          const T w = from_lane(weight, i0 + r);
#pragma unroll
          for (uint32_t e = 0; e < Quad<T>::N; ++e) sum.v[e] += w * x[r].v[e];
        }
        if (--left == 0) {
          if (at.place < a.width) at.template store<kStreaming>(out + (int64_t)(begin + token) * a.output_colstride, sum);
          sum = Quad<T>{};
          left = k;
          ++token;
        }
      }
    }
    t0 += now;
  }
}

constexpr int64_t kWavesOfTheChip = 256 * 32;

template <class T>
void combine_launch(hipStream_t s, const CombineArgs& a) {
  const int64_t parts = (a.width + 64 * Quad<T>::N - 1) / (64 * Quad<T>::N);
  // tokens to a wave: no more than leave a wave to every place there is for one, unless there are more waves than a launch takes
  int64_t run = std::max<int64_t>(1, std::min<int64_t>((int64_t)a.n * parts / kWavesOfTheChip, 64 / a.n_chosen));
  run = std::max(run, ((int64_t)a.n * parts + kMostBlocks - 1) / kMostBlocks);
  const int64_t units = (a.n + run - 1) / run * parts;
  const dim3 grid((uint32_t)((units + kCombineBlock / 64 - 1) / (kCombineBlock / 64)));
  const bool past = (int64_t)a.n * (a.n_chosen + 1) * a.width * (int64_t)sizeof(T) > kCombineCacheBytes;
  if (past) hipLaunchKernelGGL((combine_kernel<T, true>), grid, dim3(kCombineBlock), 0, s, a, (uint32_t)parts, (uint32_t)run, (uint32_t)units);
  else hipLaunchKernelGGL((combine_kernel<T, false>), grid, dim3(kCombineBlock), 0, s, a, (uint32_t)parts, (uint32_t)run, (uint32_t)units);
}

// LANES lanes to an assignment, each by itself: its row's gradient, and the product of its row with the token's gradient.  That is read
// again for each of its rows, out of the caches, and nothing waits for another row.  (A wave to a token, two or four rows at a time with the
// next ones on their way, was as fast for 16384 tokens of 4 rows of 1000 floats, 125 us, and slower elsewhere: 60000 tokens of 8 rows of 64
// floats 113 us and 48 so; one token of 8 rows of 4096 doubles 19 and 6.)
template <class T, int LANES, bool kStreaming>
__global__ void __launch_bounds__(kCombineBlock) combine_gradient_kernel(const CombineArgs a, uint32_t assignments, FastDiv k_fd) {
  constexpr uint32_t N = Quad<T>::N, kGroups = kCombineBlock / LANES;
  __shared__ T lds[2][kCombineBlock / 64];
  int turn = 0;
  const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const bool dots = a.weights_gradient != nullptr;
  for (uint32_t unit0 = blockIdx.x * kGroups; unit0 < assignments; unit0 += gridDim.x * kGroups) {
    const uint32_t unit = min(unit0 + group, assignments - 1);
    const int32_t slot = a.slots[unit];
    const bool in = slot >= 0 && slot < a.row_count;
    const T weight = a.weights ? static_cast<const T*>(a.weights)[unit] : T(1);
    const T* dy = static_cast<const T*>(a.output_gradient) + (int64_t)k_fd.div(unit) * a.gradient_colstride;
    const T* row = in && dots ? static_cast<const T*>(a.rows) + (int64_t)slot * a.rows_colstride : dy;
    T* to = static_cast<T*>(a.output) + (int64_t)(in ? slot : 0) * a.output_colstride;
    T dot = 0;
#pragma unroll 4
    for (uint32_t place = lane * N; place < a.width; place += LANES * N) {
      const RowPart<T> at(place, a.width);
      Quad<T> g = at.template load<false>(dy);
      const Quad<T> x = at.template load<kStreaming>(row);
#pragma unroll
      for (uint32_t e = 0; e < N; ++e) {
        dot += at.owns(e) ? g.v[e] * x.v[e] : T(0);
        g.v[e] *= weight;
      }
      if (a.output && in && unit0 + group < assignments) at.template store<kStreaming>(to, g);
    }
    if (!dots) continue;
#pragma unroll
    for (int m = (LANES < 64 ? LANES : 64) / 2; m > 0; m >>= 1) dot += __shfl_xor(dot, m);
    if constexpr (LANES > 64) {
      T* mine = lds[turn];
      turn ^= 1;
      if (threadIdx.x % 64 == 0) mine[threadIdx.x / 64] = dot;
      __syncthreads();
      dot = mine[0];
#pragma unroll
      for (int w = 1; w < LANES / 64; ++w) dot += mine[w];
    }
    if (lane == 0 && unit0 + group < assignments) static_cast<T*>(a.weights_gradient)[unit] = in ? dot : T(0);
  }
}

template <class T>
void combine_gradient_launch(hipStream_t s, const CombineArgs& a) {
  const bool past = (int64_t)a.n * (2 * a.n_chosen + 1) * a.width * (int64_t)sizeof(T) > kCombineCacheBytes;
  const int64_t assignments = (int64_t)a.n * a.n_chosen, pieces = (a.width + Quad<T>::N - 1) / Quad<T>::N;
  // Lanes by the length of a row, and all of a block where there are too few rows for the chip, or where the caches do not hold long ones.  Us with
  // 16, 64 and 256: 60000 tokens of 4 rows of 64 floats 25, 67 and 222; 2000 of 4 of 1024 15.5, 14.0 and 19.3; 500 of one of 4096 38, 11.8 and
  // 6.0; 8192 of 4 of 2048 160, 156 and 123.
  const int lanes = pieces <= 64 ? 16 : assignments <= 1024 || (past && pieces >= 512 && a.n_chosen > 2) ? 256 : 64;
  const int64_t groups = kCombineBlock / lanes;
  const dim3 grid((uint32_t)std::min((assignments + groups - 1) / groups, kMostBlocks));
  const FastDiv k_fd(a.n_chosen);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kCombineBlock), 0, s, a, (uint32_t)assignments, k_fd); };
  if (lanes == 16 && past) launch(combine_gradient_kernel<T, 16, true>);
  else if (lanes == 16) launch(combine_gradient_kernel<T, 16, false>);
  else if (lanes == 64 && past) launch(combine_gradient_kernel<T, 64, true>);
  else if (lanes == 64) launch(combine_gradient_kernel<T, 64, false>);
  else if (past) launch(combine_gradient_kernel<T, 256, true>);
  else launch(combine_gradient_kernel<T, 256, false>);
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
  const int64_t size = dtype_size(dtype), choices = n * n_chosen;
  const Run results[] = {{experts, choices * 4}, {weights, choices * size}, {offsets, (n_experts + 1) * 4}, {tokens, choices * 4}, {slots, choices * 4}};
  for (int i = 0; i < 5; ++i) {
    CT_REQUIRE(!run_meets(results[i], {logits, n, n_experts, logits_colstride}, size), "ct_route_experts: a result overlaps the logits");
    for (int j = 0; j < i; ++j) CT_REQUIRE(!runs_meet(results[i], results[j]), "ct_route_experts: the results overlap");
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  RouteArgs a{};
  a.experts = experts; a.weights = weights; a.offsets = offsets; a.tokens = tokens; a.slots = slots; a.logits = logits;
  a.colstride = logits_colstride;
  a.n = (uint32_t)n; a.n_experts = (uint32_t)n_experts; a.n_chosen = (uint32_t)n_chosen;
  a.renormalize = renormalize != 0;
  if (!is_few(n, n_experts, n_chosen, size)) {
    // 16 tokens to a block, 64 where there are blocks enough, more where the blocks' counts and their totals would take more than 8 MiB
    const int64_t most_blocks = (int64_t(2) << 20) / (n_experts + 1) - 1;
    a.tokens_per_block = (uint32_t)std::max<int64_t>(n <= 8192 ? 16 : 64, (n + most_blocks - 1) / most_blocks);
    a.blocks = (uint32_t)((n + a.tokens_per_block - 1) / a.tokens_per_block);
    void* scratch = nullptr;
    if (int rc = stream_scratch(s, ((size_t)a.blocks + 1) * (n_experts + 1) * sizeof(int32_t), &scratch)) return rc;
    a.totals = static_cast<int32_t*>(scratch);
    a.counts = a.totals + n_experts + 1;
  }
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
  const int64_t size = dtype_size(dtype), choices = n * n_chosen;
  const RowRange result{logits_gradient, n, n_experts, logits_gradient_colstride};
  const bool in_place = logits_gradient == logits && (logits_gradient_colstride == logits_colstride || n == 1);   // a token's lanes read its row piece by piece ahead of storing it
  CT_REQUIRE(!run_meets({weights_gradient, choices * size}, result, size) && !run_meets({weights, choices * size}, result, size) &&
                 !run_meets({experts, choices * 4}, result, size) &&
                 (renormalize || in_place || !rows_meet(result, {logits, n, n_experts, logits_colstride}, size)),
             "ct_route_experts_gradient: logits_gradient overlaps an operand");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const RouteGradientArgs a{logits_gradient, weights_gradient, weights, experts, logits, logits_gradient_colstride,
                            logits_colstride, (uint32_t)n, (uint32_t)n_experts, (uint32_t)n_chosen, renormalize != 0};
  if (dtype == CT_F32) route_gradient_launch<float>(s, a);
  else route_gradient_launch<double>(s, a);
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
  const int64_t size = dtype_size(dtype);
  const RowRange result{output, n, width, output_colstride};
  CT_REQUIRE(!rows_meet(result, {rows, row_count, width, rows_colstride}, size), "ct_combine_experts: output and rows overlap");
  CT_REQUIRE(!run_meets({weights, n * n_chosen * size}, result, size) && !run_meets({slots, n * n_chosen * 4}, result, size),
             "ct_combine_experts: output overlaps the weights or the slots");
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
  const int64_t size = dtype_size(dtype);
  const RowRange of_output{output_gradient, n, width, output_gradient_colstride}, of_rows{weights_gradient ? rows : nullptr, row_count, width, rows_colstride};
  const Run of_weights{weights, n * n_chosen * size}, of_slots{slots, n * n_chosen * 4}, to_weights{weights_gradient, n * n_chosen * size};
  CT_REQUIRE(!rows_meet(result, of_output, size) && !rows_meet(result, of_rows, size) && !run_meets(of_weights, result, size) &&
                 !run_meets(of_slots, result, size),
             "ct_combine_experts_gradient: rows_gradient overlaps an operand");
  // a weight is read by the lanes that store its gradient, ahead of that
  CT_REQUIRE(!run_meets(to_weights, of_output, size) && !run_meets(to_weights, of_rows, size) && !runs_meet(to_weights, of_slots) &&
                 (weights_gradient == weights || !runs_meet(to_weights, of_weights)),
             "ct_combine_experts_gradient: weights_gradient overlaps an operand");
  CT_REQUIRE(!run_meets(to_weights, result, size), "ct_combine_experts_gradient: the results overlap");
  if (width == 0) return weights_gradient ? ct_memset(stream, weights_gradient, dtype, 0.0, n * n_chosen) : (int)CT_OK;
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
