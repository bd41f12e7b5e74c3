// rows.h -- matrices of rows: where they lie in memory, and accesses of 16 bytes at any element.
#pragma once

#include "common.h"

namespace cthip {

// rows x width elements, a leading dimension of ld.
struct RowRange {
  const void* p;
  int64_t rows, width, ld;
};

// Whether two of them have an element in common.  Column blocks of one wider matrix do not; where the leading dimensions
// differ, ranges of bytes decide.
inline bool rows_meet(const RowRange& a, const RowRange& b, int64_t size) {
  if (!a.p || !b.p || a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1) return false;
  const int64_t x = (int64_t)(uintptr_t)a.p, y = (int64_t)(uintptr_t)b.p;
  if (y >= x + ((a.rows - 1) * a.ld + a.width) * size || x >= y + ((b.rows - 1) * b.ld + b.width) * size) return false;
  if (a.ld != b.ld || (y - x) % size) return true;
  const int64_t off = ((y - x) / size % a.ld + a.ld) % a.ld;   // of b's columns from a's
  return off < a.width || off + b.width > a.ld;
}

// 16 bytes that begin at any element: the hardware takes them from any multiple of four bytes.
template <class T> struct Quad {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};
template <class T> __device__ __forceinline__ Quad<T> load_quad(const T* p) {
  Quad<T> q;
  __builtin_memcpy(&q, p, 16);
  return q;
}
template <class T> __device__ __forceinline__ void store_quad(T* p, const Quad<T>& q) { __builtin_memcpy(p, &q, 16); }

}  // namespace cthip
