// Attention over a paged cache with the keys split over the workgroups: the partial
// results and their join, shared by the kernels of few rows and of drafted trees.
#pragma once
#include "dn_attn_fwd.h"

namespace dn {
namespace {

// A partial result: BM rows of D sums, then BM maxima, then BM sums of exponentials.
template <int D, int BM> constexpr int64_t slot_floats() { return (int64_t)BM * (D + 2); }

// the first unit of workgroup w of W
__device__ __forceinline__ int first_unit(int w, int W, int C) { return (int)((int64_t)w * C / W); }

// Joins the parts of a query row if more than one workgroup had some: D/4 threads
// per part, 1024/D parts at a time.
template <class T, int D, int BM, int UNIT, bool TREE>
__global__ __launch_bounds__(256) void k_attn_join(const AF p, int groups) {
  constexpr int NP = 1024 / D;
  __shared__ float ps[NP][D + 4];
  Task t;
  int row;
  const int Hq = p.Hkv * p.G, i = blockIdx.x / Hq, hq = blockIdx.x - i * Hq;
  const PlanOf<TREE> plan(p, BM, UNIT);
  const int W = min(groups, plan.C);
  if (!plan.of_row(i, hq, t, row)) return;
  // the workgroup that has unit u: the last w with w C / W <= u
  auto owner = [&](int u) { return (int)((((int64_t)u + 1) * W + plan.C - 1) / plan.C) - 1; };
  const int w0 = owner(t.first), w1 = owner(t.first + t.units - 1);
  if (w0 == w1) return;
  row -= t.m * BM;
  const int ch = threadIdx.x % (D / 4), part = threadIdx.x / (D / 4);
  f32x4 a = zero4();
  float m = -INFINITY, z = 0.f;
#pragma unroll 4
  for (int w = w0 + part; w <= w1; w += NP) {
    const float* s = p.part + (2 * (int64_t)w + (w == w0 ? 1 : 0)) * slot_floats<D, BM>();
    const f32x4 y = *reinterpret_cast<const f32x4*>(s + row * D + 4 * ch);
    const float mw = s[BM * D + row], zw = s[BM * D + BM + row];
    const float n = fmaxf(m, mw);
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - n), g = mw == -INFINITY ? 0.f : fast_exp2(mw - n);
    if (f != 1.f) a *= f;
    if (g != 0.f) a += g * y;
    z = z * f + g * zw;
    m = n;
  }
  *reinterpret_cast<f32x4*>(&ps[part][4 * ch]) = a;
  if (ch == 0) {
    ps[part][D] = m;
    ps[part][D + 1] = z;
  }
  __syncthreads();
  if (part) return;
#pragma unroll
  for (int k = 1; k < NP; ++k) {
    const float mw = ps[k][D], n = fmaxf(m, mw);
    const float f = m == -INFINITY ? 0.f : fast_exp2(m - n), g = mw == -INFINITY ? 0.f : fast_exp2(mw - n);
    const f32x4 y = *reinterpret_cast<const f32x4*>(&ps[k][4 * ch]);
    if (f != 1.f) a *= f;
    if (g != 0.f) a += g * y;
    z = z * f + g * ps[k][D + 1];
    m = n;
  }
  const bool none = TREE ? tree_empty(p, i, t.s) : t.s.len - t.s.n + i - t.s.c0 < 0;
  const float f = none ? 0.f : 1.f / z;   // (a sum of 0 over keys that are seen is no number)
  const float y[4] = {a[0] * f, a[1] * f, a[2] * f, a[3] * f};
  st4<T>((T*)p.out + (int64_t)blockIdx.x * D + 4 * ch, y);
  if (p.lse && ch == 0) p.lse[blockIdx.x] = z == 0.f ? -INFINITY : kLn2 * (m + __log2f(z));
}

}  // namespace
}  // namespace dn
