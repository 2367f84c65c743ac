// Device helpers of the kernels that rotate heads by their tokens' positions.
//
// A thread owns 16 channels of a head, as two groups of 8 that are each other's
// partners in the rotation: no exchange between lanes, 16-byte loads and stores in
// 16-bit types.
#pragma once
#include "dn_common.h"

namespace dn {

template <class T> __device__ __forceinline__ void ld8(const T* p, float* o) {
  typedef T V __attribute__((ext_vector_type(8)));
  const V a = *reinterpret_cast<const V*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
}
template <class T, bool PAST = false> __device__ __forceinline__ void st8(T* p, const float* v) {
  typedef T V __attribute__((ext_vector_type(8)));
  V a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
  if constexpr (PAST) __builtin_nontemporal_store(a, reinterpret_cast<V*>(p));
  else *reinterpret_cast<V*>(p) = a;
}

// The 16 channels of item `it` of a head row: groups of 8 starting at a and b.
// Items below R/16 are rotated, the others copied.
struct Item {
  int a, b, row;   // row: offset of the cosines in the table's row, -1 for a copy
};
__device__ __forceinline__ Item item_of(int it, int R, bool inter) {
  const int nr = R >> 4;
  if (it >= nr) return {R + (it - nr) * 16, R + (it - nr) * 16 + 8, -1};
  if (inter) return {it * 16, it * 16 + 8, it * 8};
  return {it * 8, (R >> 1) + it * 8, it * 8};
}

// (x, y) -> (x c - y s, y c + x s) for the 8 pairs of an item
__device__ __forceinline__ void turn8(float* x, float* y, const float* c, const float* s, bool inter) {
  if (inter) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1], d = y[2 * i], e = y[2 * i + 1];
      x[2 * i] = a * c[i] - b * s[i];
      x[2 * i + 1] = b * c[i] + a * s[i];
      y[2 * i] = d * c[4 + i] - e * s[4 + i];
      y[2 * i + 1] = e * c[4 + i] + d * s[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[i], b = y[i];
      x[i] = a * c[i] - b * s[i];
      y[i] = b * c[i] + a * s[i];
    }
  }
}

__device__ __forceinline__ void angles8(const float* table, int64_t pos, int rows, int R, int at, float sign, float* c, float* s) {
  if (pos < 0 || pos >= rows) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
    return;
  }
  const float* r = table + pos * R + at;
  ld8<float>(r, c);
  ld8<float>(r + (R >> 1), s);
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] *= sign;
}


// One pair, or one channel that is not rotated, per thread: any sizes and strides.
__device__ __forceinline__ void pair_of(int i, int R, bool inter, int& a, int& b) {
  const int half = R >> 1;
  if (i >= half) { a = R + (i - half); b = -1; }
  else if (inter) { a = 2 * i; b = a + 1; }
  else { a = i; b = i + half; }
}

}  // namespace dn
