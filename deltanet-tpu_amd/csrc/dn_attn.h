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
// LDS tiles are slabs of 32 channels, each ROWS rows of them: the 16 rows of an
// operand are 1 KB in a row, which a wave reads without a bank conflict, and
// slabs, tiles of 16 rows and steps of 32 are constant offsets from one address.
// The halves of a row change places in every other four rows, for the
// transposing reads' sake: they take half a row of 4 rows at a time.
// (Rows of all D channels with permuted 16-byte pieces read as fast, but each
// slab needs an address register of its own: 37 spilled registers at D = 128.)
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

// What that rounding cut off, itself rounded.
template <class T> __device__ __forceinline__ typename At<T>::F rest8(const f32x4& a, const f32x4& b, const typename At<T>::F& f) {
  f32x4 x, y;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = a[e] - (float)f[e], y[e] = b[e] - (float)f[4 + e];
  return frag8<T>(x, y);
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

// A use of a loaded value in front of a loop: the wait for it lands here.  Left to
// its first use inside the loop, the wait is for every load in flight there, in
// every trip, the next tile's just started ones included.
template <class V> __device__ __forceinline__ void settle(V& x) { asm volatile("" : "+v"(x)); }

// Waits for this wave's direct loads into LDS, then for everyone's.  (A barrier
// alone does not cover them.)
__device__ __forceinline__ void loads_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// N batches of operands out of LDS: read(b), then use(b).  AHEAD: each batch is
// read while the products of the one before it run, the order held against the
// compiler, which elsewhere reads an operand, waits for it (130 clocks) and uses
// it, one after another.  It takes registers for two batches; where those are not
// there the compiler's order is the better one.
template <int N, bool AHEAD, class Read, class Use> __device__ __forceinline__ void batches(Read read, Use use) {
  if (AHEAD) read(0);
#pragma unroll
  for (int b = 0; b < N; ++b) {
    if (!AHEAD) read(b);
    if (AHEAD && b + 1 < N) read(b + 1);
    if (AHEAD) __builtin_amdgcn_sched_barrier(0);
    use(b);
    if (AHEAD) __builtin_amdgcn_sched_barrier(0);
  }
}

// A tile of ROWS rows of D elements in LDS, a multiple of 32 rows.
template <class T, int D, int ROWS> struct Tile {
  using F = typename At<T>::F;
  static constexpr int kPer = 16 / sizeof(T);     // elements of a 16-byte piece
  static constexpr int kPieces = 32 / kPer;       // pieces of a row of a slab
  static constexpr int kLoad = 64 / kPieces;      // rows that a wave's load fills
  static constexpr int kSlab = ROWS * 32;
  static __device__ __forceinline__ int piece(int row, int x) { return x ^ (((row >> 2) & 1) * (kPieces / 2)); }
  static __device__ __forceinline__ int at(int row, int x) { return row * 32 + piece(row, x) * kPer; }   // piece x of a slab's row

  // channels 32 s + 8q .. + 7 of a row
  static __device__ __forceinline__ F row8(const T* t, int row, int s, int q) {
    const T* p = t + s * kSlab;
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const F*>(p + at(row, q));
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p + at(row, 2 * q));
      const f32x4 b = *reinterpret_cast<const f32x4*>(p + at(row, 2 * q) + 4);
      return F{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }

  // channel 16 c + r of rows {4q .. 4q+3, 16+4q .. 16+4q+3}
  static __device__ __forceinline__ F col8(const T* t, int c, int r, int q) {
    const T* p = t + (c >> 1) * kSlab;
    if constexpr (sizeof(T) == 2) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef short s8 __attribute__((ext_vector_type(8)));
      const int row = 4 * q + (r >> 2);
      p += at(row, 2 * (c & 1) + ((r & 3) >> 1)) + (r & 1) * 4;
      const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p);
      const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 16 * 32));
      return __builtin_bit_cast(F, (s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}));
    } else {
      F f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = pi_k(q, e), ch = 16 * (c & 1) + r;
        f[e] = p[at(row, ch / kPer) + ch % kPer];
      }
      return f;
    }
  }

  // Whether any of 32 rows has an infinity or a NaN.
  static __device__ __forceinline__ bool odd32(const T* t) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    uint32_t bad = 0;
#pragma unroll 1
    for (int s = 0; s < D / 32; ++s) {
      const u4* p = reinterpret_cast<const u4*>(t + s * kSlab);
#pragma unroll
      for (int i = 0; i < 32 * kPieces / 64; ++i) {
        const u4 x = p[i * 64 + lane_id()];
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (x[e] & At<T>::kExp) + At<T>::kOne;
      }
    }
    return __any((bad & At<T>::kTop) != 0);
  }

  // Starts wave w's part (of NW) of the loads of all rows into t; at(row) is a
  // row's first channel in memory.  A load fills 1 KB of LDS in lane order, each
  // lane from its own address; a lane has the same row in all of them.
  template <int NW, class Row> static __device__ __forceinline__ void load(T* t, int w, Row at) {
    constexpr int groups = ROWS / kLoad;
    static_assert(groups * (D / 32) % NW == 0 && (NW % groups == 0 || groups % NW == 0), "whole loads");
    if constexpr (NW % groups == 0) {
      load_part<NW, 0, 1>(t, w, source<NW>(w, at));
    } else {
      const int l = lane_id();
#pragma unroll
      for (int j = 0; j < groups / NW; ++j) {
        const int g = w + j * NW, row = g * kLoad + l / kPieces;
        const T* s = at(row) + piece(row, l % kPieces) * kPer;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) copy(s + i * 32, t + i * kSlab + g * kLoad * 32);
      }
    }
  }
  // The same in parts, for NW a multiple of the groups of rows: where the lane
  // reads, and part PART of PARTS of the wave's loads.
  template <int NW, class Row> static __device__ __forceinline__ const T* source(int w, Row at) {
    const int row = w % (ROWS / kLoad) * kLoad + lane_id() / kPieces;
    return at(row) + piece(row, lane_id() % kPieces) * kPer;
  }
  template <int NW, int PART, int PARTS> static __device__ __forceinline__ void load_part(T* t, int w, const T* s) {
    constexpr int groups = ROWS / kLoad, n = groups * (D / 32) / NW;
    static_assert(NW % groups == 0 && n * NW == groups * (D / 32), "whole loads");
#pragma unroll
    for (int i = n * PART / PARTS; i < n * (PART + 1) / PARTS; ++i) {
      const int slab = w / groups + i * (NW / groups);
      copy(s + slab * 32, t + slab * kSlab + w % groups * kLoad * 32);
    }
  }
  // 64 lanes x 16 bytes from s (each lane's own) to the 1 KB of LDS at d.  Written
  // out because the compiler takes any LDS read after its builtin for a read of
  // what that writes and waits for it, the next tile's loads in front of this
  // tile's products; here loads_barrier() is the wait.  No register is written,
  // and the compiler's own counts of loads in flight only err to the safe side.
  static __device__ __forceinline__ void copy(const T* s, T* d) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)d);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(s) : "m0");
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

// an operand with its signs changed
template <class T> __device__ __forceinline__ typename At<T>::F minus8(const typename At<T>::F& a) {
  typedef uint32_t U __attribute__((ext_vector_type(2 * sizeof(T))));
  U u = __builtin_bit_cast(U, a);
#pragma unroll
  for (int i = 0; i < 2 * (int)sizeof(T); ++i) u[i] ^= At<T>::kTop;
  return __builtin_bit_cast(typename At<T>::F, u);
}

}  // namespace dn
