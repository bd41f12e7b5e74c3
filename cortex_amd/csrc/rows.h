// rows.h -- matrices of rows: where they lie in memory, and accesses of 16 bytes at any element.
#pragma once

#include "common.h"

namespace cthip {

// rows x width elements, a leading dimension of ld.
struct RowRange {
  const void* p;
  int64_t rows, width, ld;
};

// Bytes one behind the other.
struct Run {
  const void* p;
  int64_t bytes;
};

inline bool runs_meet(const Run& a, const Run& b) {
  const int64_t x = (int64_t)(uintptr_t)a.p, y = (int64_t)(uintptr_t)b.p;
  return a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}

// Whether a run has a byte of one of the rows; what lies between rows is none.
inline bool run_meets(const Run& run, const RowRange& m, int64_t size) {
  if (m.rows < 1 || m.width < 1 || !runs_meet(run, {m.p, ((m.rows - 1) * m.ld + m.width) * size})) return false;
  const int64_t off = (int64_t)(uintptr_t)run.p - (int64_t)(uintptr_t)m.p;
  return off < 0 || off % (m.ld * size) < m.width * size || off % (m.ld * size) + run.bytes > m.ld * size;
}

// Whether two of them have an element in common.  Column blocks of one wider matrix do not, nor does a single row, or one of rows
// without gaps, that lies between the other's; else, where the leading dimensions differ, ranges of bytes decide.
inline bool rows_meet(const RowRange& a, const RowRange& b, int64_t size) {
  if (!a.p || !b.p || a.rows < 1 || b.rows < 1 || a.width < 1 || b.width < 1) return false;
  if (a.rows == 1 || a.ld == a.width) return run_meets({a.p, a.rows * a.width * size}, b, size);
  if (b.rows == 1 || b.ld == b.width) return run_meets({b.p, b.rows * b.width * size}, a, size);
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
template <class T> struct QuadBits {
  typedef T Aligned __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef Aligned AtElement __attribute__((aligned(sizeof(T))));
};
// kStreaming: past the caches, for what is used once and does not fit them
template <bool kStreaming = false, class T> __device__ __forceinline__ Quad<T> load_quad(const T* p) {
  using Bits = QuadBits<T>;
  const typename Bits::AtElement* from = reinterpret_cast<const typename Bits::AtElement*>(p);
  typename Bits::Aligned v;
  if constexpr (kStreaming) v = __builtin_nontemporal_load(from);
  else v = *from;
  return __builtin_bit_cast(Quad<T>, v);
}
template <bool kStreaming = false, class T> __device__ __forceinline__ void store_quad(T* p, const Quad<T>& q) {
  using Bits = QuadBits<T>;
  typename Bits::AtElement* to = reinterpret_cast<typename Bits::AtElement*>(p);
  const typename Bits::Aligned v = __builtin_bit_cast(typename Bits::Aligned, q);
  if constexpr (kStreaming) __builtin_nontemporal_store(v, to);
  else *to = v;
}

}  // namespace cthip
