// Shared device helpers of the softmax-attention kernels.
//
// Layout of every product here
// ----------------------------
// Products are 16x16 tiles over 32-deep slabs (one v_mfma_f32_16x16x32 for
// 16-bit types, eight v_mfma_f32_16x16x4_f32 for float32), with r = lane & 15
// and q = lane >> 4.  A product over channels takes 8 neighbouring channels
// 8q .. 8q+7 of a slab per lane, as rows lie in memory.  Scores are formed
// transposed, S^T = K Q^T: the accumulator's column r is a query row and its
// rows 4q .. 4q+3 are keys, so a query's maximum and sum stay in one lane but
// for two exchanges over q, and two stacked tiles of probabilities ARE the
// B operand of the next product O^T = V^T P^T, over keys in the order
// {4q .. 4q+3, 16+4q .. 16+4q+3}.  Its A operand, V^T in that order, comes out
// of row-major LDS by two transposing reads.
//
// LDS tiles are rows of D elements whose 16-byte pieces are permuted within
// each 128 bytes by the row number: the row reads of a slab, the transposing
// reads of 4 rows, and the direct loads that fill the tile all spread over the
// banks.
#pragma once
#include "dn_common.h"

namespace dn {

template <class T> struct At;

template <> struct At<bf16> {
  typedef bf16 F __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExp = 0x7f807f80u, kOne = 0x00800080u, kTop = 0x80008000u;
  static __device__ __forceinline__ void mma(f32x4& c, const F& a, const F& b) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct At<f16> {
  typedef f16 F __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExp = 0x7c007c00u, kOne = 0x04000400u, kTop = 0x80008000u;
  static __device__ __forceinline__ void mma(f32x4& c, const F& a, const F& b) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct At<float> {
  typedef float F __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExp = 0x7f800000u, kOne = 0x00800000u, kTop = 0x80000000u;
  static __device__ __forceinline__ void mma(f32x4& c, const F& a, const F& b) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  }
};

// 8 floats as an operand: the one rounding of probabilities and score
// gradients to a 16-bit input type, as the matrix instruction needs it
template <class T> __device__ __forceinline__ typename At<T>::F frag8(const f32x4& a, const f32x4& b) {
  typedef float f8 __attribute__((ext_vector_type(8)));
  return __builtin_convertvector((f8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}), typename At<T>::F);
}

// A value and the one of the lane N (32, 16) lanes away, in either order.
template <int N> __device__ __forceinline__ void both(float x, float& a, float& b) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  unsigned s0, s1;   // (a vector's element does not go through bit_cast by itself)
  if constexpr (N == 32) {
    const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    s0 = s[0], s1 = s[1];
  } else {
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    s0 = s[0], s1 = s[1];
  }
  a = __builtin_bit_cast(float, s0);
  b = __builtin_bit_cast(float, s1);
}
// maximum and sum over the four lanes that share r
__device__ __forceinline__ float max_q(float x) {
  float a, b;
  both<32>(x, a, b);
  both<16>(fmaxf(a, b), a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float sum_q(float x) {
  float a, b;
  both<32>(x, a, b);
  both<16>(a + b, a, b);
  return a + b;
}

// Waits for this wave's direct loads into LDS, then for everyone's.  (A barrier
// alone does not cover them.)
__device__ __forceinline__ void loads_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A tile of rows of D elements in LDS.
template <class T, int D> struct Tile {
  using F = typename At<T>::F;
  static constexpr int kPer = 16 / sizeof(T);       // elements of a 16-byte piece
  static constexpr int kPieces = D / kPer;          // pieces of a row
  static __device__ __forceinline__ int swz(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

  // channels 32 s + 8q .. + 7 of a row
  static __device__ __forceinline__ F row8(const T* t, int row, int s, int q) {
    const T* p = t + row * D;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const F*>(p + (((4 * s + q) ^ swz(row)) * 8));
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p + ((8 * s + 2 * q) ^ swz(row)) * 4);
      const f32x4 b = *reinterpret_cast<const f32x4*>(p + ((8 * s + 2 * q + 1) ^ swz(row)) * 4);
      return F{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }

  // channel c0 + r of rows row0 + {4q .. 4q+3, 16+4q .. 16+4q+3}
  static __device__ __forceinline__ F col8(const T* t, int row0, int c0, int r, int q) {
    if constexpr (sizeof(T) == 2) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef short s8 __attribute__((ext_vector_type(8)));
      const int row = row0 + 4 * q + (r >> 2);   // (row0 is a multiple of 16: both halves have the row's permutation)
      const T* p = t + row * D + (((c0 >> 3) + ((r & 3) >> 1)) ^ swz(row)) * 8 + (r & 1) * 4;
      const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
      const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 16 * D));
      return __builtin_bit_cast(F, (s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}));
    } else {
      F f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = at(t, row0 + pi_k(q, e), c0 + r);
      return f;
    }
  }

  static __device__ __forceinline__ T at(const T* t, int row, int c) {
    return t[row * D + ((c / kPer) ^ swz(row)) * kPer + c % kPer];
  }

  // Whether any of 32 rows has an infinity or a NaN.
  static __device__ __forceinline__ bool odd32(const T* t) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    uint32_t bad = 0;
    const u4* p = reinterpret_cast<const u4*>(t);
#pragma unroll 4
    for (int i = lane_id(); i < 32 * kPieces; i += 64) {
      const u4 x = p[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) bad |= (x[e] & At<T>::kExp) + At<T>::kOne;
    }
    return __any((bad & At<T>::kTop) != 0);
  }

  // Starts the loads of ROWS rows into t by NT threads; at(row) is a row's
  // first channel in memory.  A wave's load fills 1 KB of LDS in lane order,
  // each lane from its own address.
  template <int ROWS, int NT, class At_> static __device__ __forceinline__ void load(T* t, int tid, At_ at) {
    constexpr int n = ROWS * kPieces / NT;
    static_assert(n * NT == ROWS * kPieces, "whole loads");
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int c = i * NT + tid, row = c / kPieces, piece = (c % kPieces) ^ swz(row);
      const T* s = at(row) + piece * kPer;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)s,
                                       (__attribute__((address_space(3))) void*)(t + (i * NT + (tid & ~63)) * kPer), 16, 0, 0);
    }
  }
};

// An operand with its infinities and NaNs replaced by zero.  Rows of a tile that
// some query must not see may hold them, and the matrix instruction would make
// NaN of them even times a probability of 0: such a tile's operand goes through
// here, and what the queries that do see those elements get of them is added at
// the end (`odd`).
template <class T> __device__ __forceinline__ typename At<T>::F finite8(const typename At<T>::F& a) {
  typename At<T>::F f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __builtin_isfinite((float)a[e]) ? a[e] : (T)0.f;
  return f;
}

}  // namespace dn
