// Forward softmax attention: kernel parameters and the many-row kernel, shared
// by the contiguous (training) and the paged (serving) entry.
#pragma once
#include "dn_attn.h"
#include "dn_host.h"

namespace dn {

// Kernel parameters, strides in elements.
struct AF {
  int B, N, T;               // sequences; new tokens in all; per sequence (0: cu)
  int Hkv, G;                // query heads = Hkv * G, query head h reads key head h / G
  int window;                // keys that a query sees, itself the last; 0: all
  int shift, pages, max_pages;
  float sc;                  // scale * log2(e)
  const void *q, *k, *v;
  void* out;                 // dense (tokens, Hkv G, D)
  float* lse;                // NULL or (tokens, Hkv G)
  const int32_t *cu, *lens, *pt;
  const int32_t* start;      // contiguous: NULL or the first token of each token's document (B, T)
  int64_t qs[3], ks[3], vs[3];   // batch or page, token, head
  int64_t pts;
};

// Rows of K or V in memory: contiguous, or through a page table.
template <class T, bool PAGED> struct Rows {
  const T* base;       // the head's first channel of token 0 (of page 0)
  int64_t token, page;
  const int32_t* pt;
  int shift, pages, last;   // last: the last token that may be read
  __device__ __forceinline__ const T* operator()(int t) const {
    t = min(t, last);
    if constexpr (!PAGED) return base + t * token;
    const int pg = min(max(pt[t >> shift], 0), pages - 1);
    return base + pg * page + (t & ((1 << shift) - 1)) * token;
  }
};

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLazy = 8.f;   // a running maximum may lag behind by a factor 2^8

// The sequence b that owns row tile `tile` (tiles of BM rows (token, head of the
// group), whole per sequence), by all threads of a wave together; false past the
// last tile.  c0: b's first token among the new ones, n: its new tokens.
struct Seq { int b, c0, n, m; };
__device__ __forceinline__ bool find_tile(const AF& p, int tile, int BM, Seq& s) {
  if (p.cu == nullptr) {
    const int M = (p.T * p.G + BM - 1) / BM;
    s.b = tile / M;
    s.m = tile - s.b * M;
    s.n = p.T;
    s.c0 = s.b * p.T;
    return s.b < p.B;
  }
  const int l = lane_id();
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int b = b0 + l;
    int c0 = 0, n = 0;
    if (b < p.B) {
      c0 = min(max(p.cu[b], 0), p.N);
      n = min(max(p.cu[b + 1], c0), p.N) - c0;
    }
    const int mine = (int)(((int64_t)n * p.G + BM - 1) / BM);
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(sum, o);
      if (l >= o) sum += x;
    }
    const unsigned long long hit = __ballot(before + sum > tile);
    if (hit) {
      const int w = __builtin_ctzll(hit);
      s.b = b0 + w;
      s.c0 = __shfl(c0, w);
      s.n = __shfl(n, w);
      s.m = tile - before - __shfl(sum - mine, w);
      return true;
    }
    before += __shfl(sum, 63);
  }
  return false;
}

// Attention over many rows per sequence (training, prompts): head dimension and
// type checked by the caller.
hipError_t attn_many(const AF& p, int D, int dtype, bool paged, hipStream_t st);

// The gradient (contiguous rows): p with out, lse and start of the forward, d_out
// dense, the three gradients dense, delta (tokens, Hkv G) floats of scratch.
struct AB {
  AF f;
  float scale;
  const void* d_out;
  void *dq, *dk, *dv;
  float* delta;
};
hipError_t attn_backward(const AB& p, int D, int dtype, hipStream_t st);

}  // namespace dn
