// ortho.h -- what the kernels that make matrices orthogonal have in common (ops_ortho.hip; ops_ortho_few.hip for few rows).
#pragma once

#include "common.h"

namespace cthip {

// What a step begins with: of ct_orthogonalize a matrix x; of ct_muon_step the momentum x, which takes up the gradient.
struct StartArgs {
  const void* x;
  const void* gradient;      // of a step, else null
  void* momentum;            // x itself, of a step
  double* partial;           // [matrix][kParts]
  int64_t ld, stride;
  uint32_t rows, columns;
  double gradient_alpha, decay, epsilon;   // decay: of the momentum
  bool nesterov;
  void move(int64_t bytes) {
    x = static_cast<const char*>(x) + bytes;
    if (gradient) gradient = static_cast<const char*>(gradient) + bytes;
    if (momentum) momentum = static_cast<char*>(momentum) + bytes;
  }
};

// What is made orthogonal: the matrix, the momentum, or what it will be after another such gradient.
template <class T>
__device__ __forceinline__ T start_value(const StartArgs& a, int64_t at) {
  const T x = static_cast<const T*>(a.x)[at];
  if (!a.gradient || !a.nesterov) return x;
  return (T)a.gradient_alpha * static_cast<const T*>(a.gradient)[at] + (T)a.decay * x;
}

// Float matrices whose shorter side is at most this are ortho_few's, where the steps make what X X^T is off by, 2^-53 of its largest
// value or a few times that, at most this many times as large: a float's half step is not reached.  It is 2^19 after five of the
// usual steps, and six are taken.  After twenty a row that is there twice, a singular value of 0, would have become -1 in X X^T, and the
// next steps infinite.
constexpr int64_t kMostFew = 64;
constexpr double kMostFewChange = 0x1p24;

struct FewMatrices {
  StartArgs start;
  char* workspace;             // workspace_stride bytes to a matrix, few_bytes() at least
  int64_t workspace_stride;
  float* out;
  int64_t ldo, out_stride;
  float alpha, beta;
  const double* coefficients;  // of the host
  int steps;
};
int64_t few_bytes(int64_t shorter, int64_t longer);
// Three launches.
void ortho_few(hipStream_t s, const FewMatrices& f, int64_t count);

}  // namespace cthip
