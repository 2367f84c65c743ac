// Forward softmax attention over many rows: training and prompts.
#include "dn_attn_fwd.h"

namespace dn {
namespace {

// One workgroup: NW waves of 16 NQ query rows each over one head's keys.
template <class T, int D, int NQ, int NW, int BN, bool PAGED>
__global__ __launch_bounds__(64 * NW) void k_attn(const AF p) {
  using TL = Tile<T, D>;
  using F = typename At<T>::F;
  constexpr int BM = 16 * NQ * NW, NS = D / 32, NC = D / 16, NT = 64 * NW;
  __shared__ __align__(16) T lds[4 * BN * D];   // [2][K, V][BN][D]

  const int l = lane_id(), r = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // head innermost, then the tiles of all sequences, the last (longest) first
  const int nt = gridDim.x / p.Hkv;
  const int h = blockIdx.x % p.Hkv;
  Seq s;
  if (!find_tile(p, nt - 1 - (int)(blockIdx.x / p.Hkv), BM, s)) return;
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  s.c0 = __builtin_amdgcn_readfirstlane(s.c0);
  s.n = __builtin_amdgcn_readfirstlane(s.n);
  s.m = __builtin_amdgcn_readfirstlane(s.m);
  int len = s.n;
  if (PAGED) len = min(max(p.lens[s.b], 0), p.max_pages << p.shift);
  const int off = len - s.n;                       // position of the first new token
  const int rows = s.n * p.G, row0 = s.m * BM;
  const int row1 = min(row0 + BM, rows);           // the tile's rows
  const int p0 = off + row0 / p.G, p1 = off + (row1 - 1) / p.G;   // their positions

  // queries: row -> token row / G, head h G + row % G
  F qf[NQ][NS];
  int pos[NQ], low[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = min(row0 + (w * NQ + i) * 16 + r, rows - 1);
    const int t = row / p.G, g = row - t * p.G;
    const T* qp = (const T*)p.q + (p.cu ? (int64_t)(s.c0 + t) * p.qs[1] : s.b * p.qs[0] + t * p.qs[1]) + (h * p.G + g) * p.qs[2];
#pragma unroll
    for (int c = 0; c < NS; ++c) qf[i][c] = *reinterpret_cast<const F*>(qp + 32 * c + 8 * q);
    pos[i] = off + t;
    low[i] = p.window ? pos[i] - p.window + 1 : 0;
    if (!PAGED && p.start) low[i] = max(low[i], p.start[s.b * p.T + t]);
  }
  int lo0 = p.window ? max(p0 - p.window + 1, 0) : 0, lo1 = p.window ? p1 - p.window + 1 : 0;   // first keys of the first and last row
  if (!PAGED && p.start) {
    lo0 = max(lo0, p.start[s.b * p.T + p0]);
    lo1 = max(lo1, p.start[s.b * p.T + p1]);
  }
  const int j0 = lo0 / BN, j1 = p1 < 0 ? 0 : p1 / BN + 1;

  Rows<T, PAGED> kr, vr;
  kr.base = (const T*)p.k + (PAGED ? 0 : s.b * p.ks[0]) + h * p.ks[2];
  vr.base = (const T*)p.v + (PAGED ? 0 : s.b * p.vs[0]) + h * p.vs[2];
  kr.token = p.ks[1]; vr.token = p.vs[1];
  kr.page = p.ks[0]; vr.page = p.vs[0];
  kr.pt = vr.pt = PAGED ? p.pt + s.b * p.pts : nullptr;
  kr.shift = vr.shift = p.shift;
  kr.pages = vr.pages = p.pages;
  kr.last = vr.last = max(p1, 0);   // rows past it repeat it: finite unless a query that sees it is not

  f32x4 o[NQ][NC];
  float mx[NQ], sum[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    mx[i] = -INFINITY;
    sum[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[i][c] = zero4();
  }

  auto fetch = [&](int j) {
    T* t = lds + (j & 1) * 2 * BN * D;
    TL::template load<BN, NT>(t, threadIdx.x, [&](int x) { return kr(j * BN + x); });
    TL::template load<BN, NT>(t + BN * D, threadIdx.x, [&](int x) { return vr(j * BN + x); });
  };
  if (j0 < j1) fetch(j0);
  bool odd = false;   // infinities or NaNs in a masked tile were left out
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    loads_barrier();   // tile j is there, tile j - 1 is no longer read
    if (j + 1 < j1) fetch(j + 1);
    const T* kt = lds + (j & 1) * 2 * BN * D;
    const T* vt = kt + BN * D;
    const bool masked = j * BN + BN - 1 > p0 || j * BN < lo1;
#pragma unroll 1
    for (int u = 0; u < BN; u += 32) {
      f32x4 sc[NQ][2];
#pragma unroll
      for (int i = 0; i < NQ; ++i) sc[i][0] = sc[i][1] = zero4();
#pragma unroll
      for (int c = 0; c < NS; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const F kf = TL::row8(kt, u + 16 * e + r, c, q);
#pragma unroll
          for (int i = 0; i < NQ; ++i) At<T>::mma(sc[i][e], kf, qf[i][c]);
        }
      F pf[NQ];
      bool grow = false;
      float mt[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (masked) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int key = j * BN + u + 16 * e + 4 * q + x;
              sc[i][e][x] = key <= pos[i] && key >= low[i] ? sc[i][e][x] : -INFINITY;
            }
        }
        float m = fmaxf(fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3])),
                        fmaxf(fmaxf(sc[i][1][0], sc[i][1][1]), fmaxf(sc[i][1][2], sc[i][1][3])));
        mt[i] = max_q(m) * p.sc;
        grow |= mt[i] > mx[i] + kLazy;
      }
      if (__any(grow)) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          const float m = fmaxf(mx[i], mt[i]);
          const float f = m == -INFINITY ? 1.f : fast_exp2(mx[i] - m);
          mx[i] = m;
          sum[i] *= f;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            o[i][c] *= f;
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const float m = mx[i] == -INFINITY ? 0.f : mx[i];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            sc[i][e][x] = fast_exp2(__builtin_fmaf(sc[i][e][x], p.sc, -m));
            sum[i] += sc[i][e][x];
          }
        pf[i] = frag8<T>(sc[i][0], sc[i][1]);
      }
      const bool bad = masked && TL::odd32(vt + u * D);
      odd |= bad;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        F vf = TL::col8(vt, u, 16 * c, r, q);
        if (bad) vf = finite8<T>(vf);
#pragma unroll
        for (int i = 0; i < NQ; ++i) At<T>::mma(o[i][c], vf, pf[i]);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = row0 + (w * NQ + i) * 16 + r;
    const float z = sum_q(sum[i]);
    if (row >= rows) continue;
    const int t = row / p.G, g = row - t * p.G;
    const int64_t at = (int64_t)(s.c0 + t) * p.Hkv * p.G + h * p.G + g;
    const float f = z == 0.f ? 0.f : 1.f / z;
    T* op = (T*)p.out + at * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float x[4] = {o[i][c][0] * f, o[i][c][1] * f, o[i][c][2] * f, o[i][c][3] * f};
      if (odd) {
#pragma unroll 1
        for (int key = j0 * BN; key < j1 * BN; ++key) {
          if (key >= max(low[i], 0) && key <= pos[i] && (key / BN * BN + BN - 1 > p0 || key / BN * BN < lo1)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = (float)vr(key)[16 * c + 4 * q + e];
              if (!__builtin_isfinite(y)) x[e] += y;
            }
          }
        }
      }
      st4<T>(op + 16 * c + 4 * q, x);
    }
    if (p.lse && q == 0) p.lse[at] = z == 0.f ? -INFINITY : kLn2 * (mx[i] + __log2f(z));
  }
}

template <class T, int D, bool PAGED> hipError_t run(const AF& p, hipStream_t st) {
  constexpr int NQ = sizeof(T) == 4 ? 2 : 2, NW = 4, BN = sizeof(T) == 4 ? 32 : 64;
  constexpr int BM = 16 * NQ * NW;
  // rows are whole tiles per sequence: at most one more tile each
  const int64_t tiles = p.cu ? (int64_t)p.N * p.G / BM + p.B : (int64_t)p.B * (((int64_t)p.T * p.G + BM - 1) / BM);
  hipLaunchKernelGGL((k_attn<T, D, NQ, NW, BN, PAGED>), dim3((unsigned)(tiles * p.Hkv)), dim3(64 * NW), 0, st, p);
  return hipGetLastError();
}

}  // namespace

hipError_t attn_many(const AF& p, int D, int dtype, bool paged, hipStream_t st) {
  auto go = [&](auto z) {
    using T = decltype(z);
    if (paged) return D == 64 ? run<T, 64, true>(p, st) : D == 128 ? run<T, 128, true>(p, st) : run<T, 256, true>(p, st);
    return D == 64 ? run<T, 64, false>(p, st) : D == 128 ? run<T, 128, false>(p, st) : run<T, 256, false>(p, st);
  };
  return dtype == DN_BF16 ? go((bf16)0.f) : dtype == DN_F16 ? go((f16)0.f) : go(0.f);
}

}  // namespace dn
