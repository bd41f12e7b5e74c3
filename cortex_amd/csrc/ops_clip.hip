// ops_clip.hip -- the norm over many gradients and their clipping (ct_clip_gradients).
//
// norm = sqrt(sum over all tensors of g^2), factor = max_norm / max(norm, max_norm), out = g * factor.  Squares are formed and
// summed in double: a float's square is exact there and no sum of floats overflows.
//
// The tensors are cut into pieces; a launch's blocks take every so manieth piece, form one sum of squares each, and the norm is
// the sum of those in their order.  A few sums are added by every block that needs the factor, more by a launch of their own.
// Multiplying takes the launches' tables last to first, and each tensor's pieces last to first, but the tensors of a table in their
// order (the table holds them in reverse, and is gone through from its end): of what was read last, and is still in the last-level
// cache, the last table's comes first.  Memory bounds it: 171 million floats in 300 tensors 377 us, two reads and a write at 5.5 TB/s.
// The tensors travel in the launch's arguments, kTensors to a launch: a table in device memory would have to be copied there
// by every call.
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "elementwise.h"
#include "rows.h"

using namespace cthip;

namespace {

constexpr int kClipBlock = 256;
constexpr int kTensors = 120;
constexpr int64_t kMostClipBlocks = 2048;   // of a launch: what the chip holds
constexpr int64_t kFewSums = 2048;          // which every block adds by itself (19 tensors, 4.9 million floats: 15.9 us, with a launch for them 18.5)
constexpr int64_t kLeastPiece = 4 << 10, kMostPiece = 64 << 10;   // bytes
constexpr int64_t kClipCacheBytes = int64_t(256) << 20;

struct ClipTable {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t count[kTensors];
  uint32_t first[kTensors + 1];   // piece of the launch that begins a tensor; all of them
  uint32_t tensors;
};
static_assert(sizeof(ClipTable) <= 3600, "with the other arguments within 4 KiB");

template <class T> struct Piece {
  const T* in;
  T* out;
  uint32_t n;
};

// The tensor that a piece belongs to is the last one that begins at or before it: a wave looks at 64 at a time.
template <class T>
__device__ __forceinline__ Piece<T> piece_of(const ClipTable& t, uint32_t piece, uint32_t piece_shift) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t i = 0;
#pragma unroll
  for (uint32_t i0 = 0; i0 < kTensors; i0 += 64) {
    const uint32_t at = min(i0 + lane, (uint32_t)kTensors);
    i += __popcll(__ballot(i0 + lane < t.tensors && t.first[at] <= piece));
  }
  i = __builtin_amdgcn_readfirstlane(i) - 1;
  const int64_t begin = (int64_t)(piece - t.first[i]) << piece_shift;
  return {static_cast<const T*>(t.in[i]) + begin, static_cast<T*>(t.out[i]) + begin,
          (uint32_t)min(int64_t(1) << piece_shift, t.count[i] - begin)};
}

__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
  const int wave = threadIdx.x >> 6, waves = kClipBlock >> 6;
  if ((threadIdx.x & 63) == 0) lds[wave] = x;
  __syncthreads();
  double sum = lds[0];
  for (int w = 1; w < waves; ++w) sum += lds[w];
  return sum;
}

constexpr int kQuads = 4;   // of a lane, whose loads are on their way together

// Calls f(at, quad) for the quads of n elements, and g(at, element) for what is left.
template <bool kStreaming, class T, class F, class G>
__device__ __forceinline__ void for_piece(const T* in, uint32_t n, F f, G g) {
  constexpr uint32_t N = Quad<T>::N, kStep = kClipBlock * N;
  uint32_t at = threadIdx.x * N, done = 0;
  for (; done + kQuads * kStep <= n; done += kQuads * kStep, at += kQuads * kStep) {
    Quad<T> q[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) q[i] = load_quad<kStreaming>(in + at + i * kStep);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) f(at + i * kStep, q[i]);
  }
  for (; at < n; at += kStep) {
    if (at + N <= n) f(at, load_quad<kStreaming>(in + at));
    else
      for (uint32_t e = at; e < n; ++e) g(e, in[e]);
  }
}

template <class T>
__global__ void __launch_bounds__(kClipBlock) clip_squares_kernel(const ClipTable t, uint32_t pieces, uint32_t piece_shift, double* partial) {
  __shared__ double lds[kClipBlock / 64];
  double sum = 0;
  for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
    const Piece<T> piece = piece_of<T>(t, p, piece_shift);
    for_piece<false>(
        piece.in, piece.n,
        [&](uint32_t, const Quad<T>& q) {
#pragma unroll
          for (int e = 0; e < Quad<T>::N; ++e) sum = fma((double)q.v[e], (double)q.v[e], sum);
        },
        [&](uint32_t, T x) { sum = fma((double)x, (double)x, sum); });
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// By the lanes of a block of kClipBlock, in every kernel: the same bits.
template <class T>
__device__ __forceinline__ T factor_of(const double* partial, uint32_t n, double max_norm, T* norm_and_factor, double* lds) {
  double sum = 0;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n; i += kClipBlock) sum += partial[i];
  const double norm = sqrt(block_sum(sum, lds));
  const T factor = (T)(norm <= max_norm ? 1.0 : max_norm / norm);   // NaN where the norm is
  if (norm_and_factor && threadIdx.x == 0) {
    norm_and_factor[0] = (T)norm;
    norm_and_factor[1] = factor;
  }
  return factor;
}

template <class T>
__global__ void __launch_bounds__(kClipBlock) clip_norm_kernel(const double* partial, uint32_t n, double max_norm, T* norm_and_factor) {
  __shared__ double lds[kClipBlock / 64];
  factor_of(partial, n, max_norm, norm_and_factor, lds);
}

// `sums` != 0: the factor is found from as many sums, and stored by the first block if `norm_and_factor` is to be; else read there.
template <class T, bool kStreaming>
__global__ void __launch_bounds__(kClipBlock) clip_scale_kernel(const ClipTable t, uint32_t pieces, uint32_t piece_shift, const double* partial,
                                                                uint32_t sums, double max_norm, T* norm_and_factor, bool store) {
  __shared__ double lds[kClipBlock / 64];
  const T factor = sums ? factor_of(partial, sums, max_norm, store && blockIdx.x == 0 ? norm_and_factor : nullptr, lds) : norm_and_factor[1];
  for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
    const Piece<T> piece = piece_of<T>(t, pieces - 1 - p, piece_shift);
    if (piece.in == piece.out && factor == (T)1) continue;
    T* const out = piece.out;
    for_piece<kStreaming>(
        piece.in, piece.n,
        [&](uint32_t at, Quad<T> q) {
#pragma unroll
          for (int e = 0; e < Quad<T>::N; ++e) q.v[e] *= factor;
          store_quad<kStreaming>(out + at, q);
        },
        [&](uint32_t at, T x) { out[at] = x * factor; });
  }
}

// Calls `launch(table, pieces, blocks)` for tables that together hold every piece, of the tensors in their order or in the other.
template <class F>
void for_tables(const void* const* in, void* const* out, const int64_t* counts, int64_t count, uint32_t piece_shift, bool last_first, F launch) {
  ClipTable t;
  t.tensors = 0;
  uint32_t pieces = 0;
  auto flush = [&] {
    t.first[t.tensors] = pieces;
    if (t.tensors) launch(t, pieces, (uint32_t)std::min<int64_t>(pieces, kMostClipBlocks));
    pieces = t.tensors = 0;
  };
  for (int64_t k = 0; k < count; ++k) {
    const int64_t i = last_first ? count - 1 - k : k;
    if (counts[i] == 0) continue;
    const int64_t of_this = ((counts[i] - 1) >> piece_shift) + 1;
    if (t.tensors == kTensors || pieces + of_this > INT32_MAX) flush();
    t.in[t.tensors] = in[i];
    t.out[t.tensors] = out ? out[i] : nullptr;
    t.count[t.tensors] = counts[i];
    t.first[t.tensors++] = pieces;
    pieces += (uint32_t)of_this;
  }
  flush();
}

template <class T>
int clip_typed(hipStream_t s, const void* const* in, void* const* out, const int64_t* counts, int64_t count, double max_norm,
               T* norm_and_factor) {
  int64_t values = 0;
  for (int64_t i = 0; i < count; ++i) values += counts[i];
  // pieces small enough to give every block one
  int64_t bytes = kLeastPiece;
  while (bytes < kMostPiece && values * (int64_t)sizeof(T) > bytes * kMostClipBlocks) bytes *= 2;
  uint32_t piece_shift = 0;
  while ((int64_t(1) << piece_shift) * (int64_t)sizeof(T) < bytes) ++piece_shift;
  int64_t sums = 0;
  for_tables(in, out, counts, count, piece_shift, false, [&](const ClipTable&, uint32_t, uint32_t blocks) { sums += blocks; });
  CT_REQUIRE(sums < INT32_MAX, "ct_clip_gradients: %lld tensors", (long long)count);
  void* scratch = nullptr;
  if (int rc = stream_scratch(s, std::max<int64_t>(sums, 1) * sizeof(double), &scratch)) return rc;
  double* const partial = static_cast<double*>(scratch);
  double* to = partial;
  for_tables(in, out, counts, count, piece_shift, false, [&](const ClipTable& t, uint32_t pieces, uint32_t blocks) {
    hipLaunchKernelGGL((clip_squares_kernel<T>), dim3(blocks), dim3(kClipBlock), 0, s, t, pieces, piece_shift, to);
    to += blocks;
  });
  const bool few = out && sums > 0 && sums <= kFewSums;
  if (!few) hipLaunchKernelGGL((clip_norm_kernel<T>), dim3(1), dim3(kClipBlock), 0, s, partial, (uint32_t)sums, max_norm, norm_and_factor);
  if (out) {
    const bool past = 2 * values * (int64_t)sizeof(T) > kClipCacheBytes;
    bool store = few;
    for_tables(in, out, counts, count, piece_shift, true, [&](const ClipTable& t, uint32_t pieces, uint32_t blocks) {
      auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kClipBlock), 0, s, t, pieces, piece_shift, partial, few ? (uint32_t)sums : 0u, max_norm,
                           norm_and_factor, store);
      };
      if (past) launch(clip_scale_kernel<T, true>);
      else launch(clip_scale_kernel<T, false>);
      store = false;
    });
  }
  note_kernel("clip");
  return after_launch(s);
}

// The memory of a tensor that has elements.
struct Extent {
  uintptr_t begin, end;
  int64_t tensor;
};

// Whether no output meets another one or another tensor's gradient; `by_place` has room for all outputs.
bool outputs_apart(const void* const* in, void* const* out, const int64_t* counts, int64_t count, int64_t size, Extent* by_place, int64_t* bad) {
  int64_t n = 0;
  bool in_order = true, in_place = true;
  for (int64_t i = 0; i < count; ++i) {
    if (counts[i] == 0) continue;
    const uintptr_t at = (uintptr_t)out[i];
    in_order = in_order && (n == 0 || by_place[n - 1].begin <= at);
    in_place = in_place && out[i] == in[i];
    by_place[n++] = {at, at + (uintptr_t)(counts[i] * size), i};
  }
  if (!in_order) std::sort(by_place, by_place + n, [](const Extent& a, const Extent& b) { return a.begin < b.begin; });
  for (int64_t k = 1; k < n; ++k)
    if (by_place[k].begin < by_place[k - 1].end) return *bad = by_place[k].tensor, false;
  if (in_place) return true;
  for (int64_t i = 0; i < count; ++i) {
    if (counts[i] == 0) continue;
    const uintptr_t begin = (uintptr_t)in[i], end = begin + (uintptr_t)(counts[i] * size);
    const Extent* const o = std::upper_bound(by_place, by_place + n, begin, [](uintptr_t at, const Extent& e) { return at < e.end; });
    if (o != by_place + n && o->begin < end && !(o->tensor == i && out[i] == in[i])) return *bad = o->tensor, false;
  }
  return true;
}

}  // namespace

extern "C" int ct_clip_gradients(void* stream, const void* const* gradients, void* const* outputs, const int64_t* counts,
                                 int64_t count, double max_norm, void* norm_and_factor, int dtype) {
  CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, "ct_clip_gradients: datatype must be float or double");
  CT_REQUIRE(count >= 0, "ct_clip_gradients: negative count");
  CT_REQUIRE(max_norm > 0, "ct_clip_gradients: max_norm must be positive");
  CT_REQUIRE(norm_and_factor && (count == 0 || (gradients && counts)), "ct_clip_gradients: null argument");
  const int64_t size = dtype_size(dtype), most = int64_t(1) << 40;
  const Run of_norm{norm_and_factor, 2 * size};
  for (int64_t i = 0; i < count; ++i) {
    CT_REQUIRE(counts[i] >= 0 && counts[i] <= most, "ct_clip_gradients: tensor %lld has %lld values", (long long)i, (long long)counts[i]);
    if (counts[i] == 0) continue;
    CT_REQUIRE(gradients[i] && (!outputs || outputs[i]), "ct_clip_gradients: null buffer");
    CT_REQUIRE(!runs_meet(of_norm, {gradients[i], counts[i] * size}) && !(outputs && runs_meet(of_norm, {outputs[i], counts[i] * size})),
               "ct_clip_gradients: the norm and the factor overlap tensor %lld", (long long)i);
    if (outputs && outputs[i] != gradients[i]) {
      const uintptr_t a = (uintptr_t)gradients[i], b = (uintptr_t)outputs[i], bytes = (uintptr_t)(counts[i] * size);
      CT_REQUIRE(a + bytes <= b || b + bytes <= a, "ct_clip_gradients: output %lld overlaps its gradient", (long long)i);
    }
  }
  if (outputs) {
    Extent few[kTensors];
    const std::unique_ptr<Extent[]> many(count > kTensors ? new (std::nothrow) Extent[count] : nullptr);
    CT_REQUIRE(count <= kTensors || many, "ct_clip_gradients: no memory for a list of %lld tensors", (long long)count);
    int64_t bad = 0;
    CT_REQUIRE(outputs_apart(gradients, outputs, counts, count, size, many ? many.get() : few, &bad),
               "ct_clip_gradients: output %lld overlaps another tensor", (long long)bad);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == CT_F32) return clip_typed<float>(s, gradients, outputs, counts, count, max_norm, static_cast<float*>(norm_and_factor));
  return clip_typed<double>(s, gradients, outputs, counts, count, max_norm, static_cast<double*>(norm_and_factor));
}
