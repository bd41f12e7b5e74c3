// ops_clip.hip -- the norm over many gradients and their clipping (ct_clip_gradients).
//
// norm = sqrt(sum over all tensors of g^2), factor = max_norm / max(norm, max_norm), out = g * factor.  Squares are formed and
// summed in double: a float's square is exact there and no sum of floats overflows.
//
// Three launches: pieces of kPiece values sum their squares, one block adds the pieces' sums in their order, the pieces are
// multiplied by the factor.  The tensors travel in the launch's arguments, kTensors to a launch: a table in device memory
// would have to be copied there by every call.
#include <algorithm>
#include <cmath>

#include "elementwise.h"
#include "rows.h"

using namespace cthip;

namespace {

constexpr int kClipBlock = 256;
constexpr int kPieceBytes = 64 << 10;
constexpr int kTensors = 120;

struct ClipTable {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t count[kTensors];
  uint32_t first[kTensors];   // piece of the launch that begins a tensor
  uint32_t tensors;
};
static_assert(sizeof(ClipTable) <= 3600, "with the other arguments within 4 KiB");

// The tensor that a piece belongs to: the last one that begins at or before it.
__device__ __forceinline__ uint32_t tensor_of(const ClipTable& t, uint32_t piece) {
  uint32_t low = 0, high = t.tensors;
  while (high - low > 1) {
    const uint32_t mid = (low + high) / 2;
    if (t.first[mid] <= piece) low = mid; else high = mid;
  }
  return low;
}

__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) lds[wave] = x;
  __syncthreads();
  double sum = lds[0];
  for (int w = 1; w < waves; ++w) sum += lds[w];
  return sum;
}

template <class T>
__global__ void __launch_bounds__(kClipBlock) clip_squares_kernel(const ClipTable t, double* partial) {
  constexpr int N = Quad<T>::N, kPiece = kPieceBytes / sizeof(T);
  __shared__ double lds[kClipBlock / 64];
  const uint32_t i = tensor_of(t, blockIdx.x);
  const int64_t first = (int64_t)(blockIdx.x - t.first[i]) * kPiece;
  const uint32_t n = (uint32_t)min((int64_t)kPiece, t.count[i] - first);
  const T* in = static_cast<const T*>(t.in[i]) + first;
  double sum = 0;
  for (uint32_t at = threadIdx.x * N; at < n; at += kClipBlock * N) {
    if (at + N <= n) {
      const Quad<T> q = load_quad(in + at);
#pragma unroll
      for (int e = 0; e < N; ++e) sum += (double)q.v[e] * (double)q.v[e];
    } else {
      for (uint32_t e = at; e < n; ++e) sum += (double)in[e] * (double)in[e];
    }
  }
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <class T>
__global__ void __launch_bounds__(1024) clip_norm_kernel(const double* partial, uint32_t n, double max_norm, T* norm_and_factor) {
  __shared__ double lds[16];
  double sum = 0;
  for (uint32_t i = threadIdx.x; i < n; i += 1024) sum += partial[i];
  sum = block_sum(sum, lds);
  if (threadIdx.x == 0) {
    const double norm = sqrt(sum);
    norm_and_factor[0] = (T)norm;
    norm_and_factor[1] = (T)(norm <= max_norm ? 1.0 : max_norm / norm);   // NaN where the norm is
  }
}

template <class T>
__global__ void __launch_bounds__(kClipBlock) clip_scale_kernel(const ClipTable t, const T* norm_and_factor) {
  constexpr int N = Quad<T>::N, kPiece = kPieceBytes / sizeof(T);
  const T factor = norm_and_factor[1];
  const uint32_t i = tensor_of(t, blockIdx.x);
  if (t.in[i] == t.out[i] && factor == (T)1) return;
  const int64_t first = (int64_t)(blockIdx.x - t.first[i]) * kPiece;
  const uint32_t n = (uint32_t)min((int64_t)kPiece, t.count[i] - first);
  const T* in = static_cast<const T*>(t.in[i]) + first;
  T* out = static_cast<T*>(t.out[i]) + first;
  for (uint32_t at = threadIdx.x * N; at < n; at += kClipBlock * N) {
    if (at + N <= n) {
      Quad<T> q = load_quad(in + at);
#pragma unroll
      for (int e = 0; e < N; ++e) q.v[e] *= factor;
      store_quad(out + at, q);
    } else {
      for (uint32_t e = at; e < n; ++e) out[e] = in[e] * factor;
    }
  }
}

// Calls `launch(table, pieces of the launch, pieces before it)` for tables that together hold every piece.
template <class F>
void for_tables(const void* const* in, void* const* out, const int64_t* counts, int64_t count, int64_t piece, F launch) {
  ClipTable t;
  t.tensors = 0;
  uint32_t pieces = 0;
  int64_t before = 0;
  auto flush = [&] {
    if (t.tensors) launch(t, pieces, before);
    before += pieces;
    pieces = t.tensors = 0;
  };
  for (int64_t i = 0; i < count; ++i) {
    if (counts[i] == 0) continue;
    const int64_t of_this = (counts[i] + piece - 1) / piece;
    if (t.tensors == kTensors || pieces + of_this > INT32_MAX / kClipBlock) flush();
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
  constexpr int64_t kPiece = kPieceBytes / sizeof(T);
  int64_t pieces = 0;
  for (int64_t i = 0; i < count; ++i) pieces += (counts[i] + kPiece - 1) / kPiece;
  CT_REQUIRE(pieces < INT32_MAX, "ct_clip_gradients: %lld pieces", (long long)pieces);
  void* scratch = nullptr;
  if (int rc = stream_scratch(s, std::max<int64_t>(pieces, 1) * sizeof(double), &scratch)) return rc;
  double* partial = static_cast<double*>(scratch);
  for_tables(in, out, counts, count, kPiece, [&](const ClipTable& t, uint32_t n, int64_t before) {
    hipLaunchKernelGGL((clip_squares_kernel<T>), dim3(n), dim3(kClipBlock), 0, s, t, partial + before);
  });
  hipLaunchKernelGGL((clip_norm_kernel<T>), dim3(1), dim3(1024), 0, s, partial, (uint32_t)pieces, max_norm, norm_and_factor);
  if (out)
    for_tables(in, out, counts, count, kPiece, [&](const ClipTable& t, uint32_t n, int64_t) {
      hipLaunchKernelGGL((clip_scale_kernel<T>), dim3(n), dim3(kClipBlock), 0, s, t, norm_and_factor);
    });
  note_kernel("clip");
  return after_launch(s);
}

}  // namespace

extern "C" int ct_clip_gradients(void* stream, const void* const* gradients, void* const* outputs, const int64_t* counts,
                                 int64_t count, double max_norm, void* norm_and_factor, int dtype) {
  CT_REQUIRE(dtype == CT_F32 || dtype == CT_F64, "ct_clip_gradients: datatype must be float or double");
  CT_REQUIRE(count >= 0, "ct_clip_gradients: negative count");
  CT_REQUIRE(max_norm > 0, "ct_clip_gradients: max_norm must be positive");
  CT_REQUIRE(norm_and_factor && (count == 0 || (gradients && counts)), "ct_clip_gradients: null argument");
  const int64_t size = dtype_size(dtype), most = int64_t(1) << 40;
  for (int64_t i = 0; i < count; ++i) {
    CT_REQUIRE(counts[i] >= 0 && counts[i] <= most, "ct_clip_gradients: tensor %lld has %lld values", (long long)i, (long long)counts[i]);
    if (counts[i] == 0) continue;
    CT_REQUIRE(gradients[i] && (!outputs || outputs[i]), "ct_clip_gradients: null buffer");
    if (outputs && outputs[i] != gradients[i]) {
      const uintptr_t a = (uintptr_t)gradients[i], b = (uintptr_t)outputs[i], bytes = (uintptr_t)(counts[i] * size);
      CT_REQUIRE(a + bytes <= b || b + bytes <= a, "ct_clip_gradients: output %lld overlaps its gradient", (long long)i);
    }
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == CT_F32) return clip_typed<float>(s, gradients, outputs, counts, count, max_norm, static_cast<float*>(norm_and_factor));
  return clip_typed<double>(s, gradients, outputs, counts, count, max_norm, static_cast<double*>(norm_and_factor));
}
