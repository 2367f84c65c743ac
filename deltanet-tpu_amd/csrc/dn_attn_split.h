// Attention over a paged cache with the keys split over the workgroups: the partial
// results, shared by the kernels of few rows and of drafted trees, and the trees' join.
#pragma once
#include "dn_attn_fwd.h"

namespace dn {
namespace {

// A partial result: BM rows of D sums, then BM maxima, then BM sums of exponentials.
// Workgroup w writes the one of a task that begins with it to slot 2 w + 1, of one that
// began before to slot 2 w.
template <int D, int BM> constexpr int64_t slot_floats() { return (int64_t)BM * (D + 2); }

// the first unit of workgroup w of W
__device__ __forceinline__ int first_unit(int w, int W, int C) { return (int)((int64_t)w * C / W); }

// Workgroups that share C units, UNITS or more each: what a part costs to write and to
// join is more than one unit of its keys.
template <int UNITS> __device__ __forceinline__ int shares(int groups, int C) { return max(min(groups, C / UNITS), 1); }

// Joins the parts of the tasks that several workgroups share, in the order of their
// keys.  x: the tasks, or, where there are fewer of those, the borders between
// workgroups, of which the first inside a task joins it.  A row takes D / 4 threads,
// once or, where there are many parts, up to 1024 / D times; y shares the rows.
template <class T, int D, int BM, int UNIT, int UNITS, bool TASKS>
__global__ __launch_bounds__(256) void k_tree_join(const AF p, int groups) {
  constexpr int NP = 1024 / D;
  __shared__ __align__(16) float ps[NP][D + 4];
  const PlanOf<true> plan(p, BM, UNIT);
  const int W = shares<UNITS>(groups, plan.C);
  // the workgroup that has unit u: the last w with w C / W <= u
  auto owner = [&](int u) { return (int)((((int64_t)u + 1) * W + plan.C - 1) / plan.C) - 1; };
  Task t;
  if constexpr (TASKS) {
    if (!plan.of_task(blockIdx.x, t)) return;
  } else {
    const int w = blockIdx.x;
    if (w + 1 >= W) return;
    const int u = first_unit(w + 1, W, plan.C);
    if (!plan.of_unit(u, t) || t.first == u || first_unit(w, W, plan.C) > t.first) return;
  }
  const int w0 = owner(t.first), w1 = owner(t.first + t.units - 1);
  if (w0 == w1) return;
  int per = 1;   // threads' groups for a row: four parts or more each
  while (per < NP && 4 * per <= w1 - w0) per *= 2;
  const int row0 = t.m * BM, n = min(BM, t.s.n * p.G - row0), ch = threadIdx.x % (D / 4), in = threadIdx.x / (D / 4), k = in % per;
  const int step = gridDim.y * (NP / per);
#pragma unroll 1
  for (int base = blockIdx.y * (NP / per); base < n; base += step) {
    const int row = base + in / per;
    const bool live = row < n;
    f32x4 a = zero4();
    float m = -INFINITY, z = 0.f;
    if (live) {
#pragma unroll 1
      for (int w = w0 + k; w <= w1; w += 4 * per) {   // four parts at a time, all on their way at once
        f32x4 y[4];
        float mw[4], zw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int v = min(w + e * per, w1);
          const float* s = p.part + (2 * (int64_t)v + (v == w0 ? 1 : 0)) * slot_floats<D, BM>();
          y[e] = *reinterpret_cast<const f32x4*>(s + row * D + 4 * ch);
          mw[e] = s[BM * D + row];
          zw[e] = s[BM * D + BM + row];
        }
        __builtin_amdgcn_sched_barrier(0);   // (the compiler would load each where it is used)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (w + e * per > w1) mw[e] = -INFINITY, zw[e] = 0.f;
          const float x = fmaxf(m, mw[e]);
          const float f = m == -INFINITY ? 0.f : fast_exp2(m - x), g = mw[e] == -INFINITY ? 0.f : fast_exp2(mw[e] - x);
          if (f != 1.f) a *= f;
          if (g != 0.f) a += g * y[e];
          z = z * f + g * zw[e];
          m = x;
        }
      }
    }
    if (per > 1) {
      __syncthreads();   // (the last rows have been read)
      *reinterpret_cast<f32x4*>(&ps[in][4 * ch]) = a;
      if (ch == 0) {
        ps[in][D] = m;
        ps[in][D + 1] = z;
      }
      __syncthreads();
      if (k == 0) {
        for (int i = 1; i < per; ++i) {
          const float mw = ps[in + i][D], x = fmaxf(m, mw);
          const float f = m == -INFINITY ? 0.f : fast_exp2(m - x), g = mw == -INFINITY ? 0.f : fast_exp2(mw - x);
          const f32x4 y = *reinterpret_cast<const f32x4*>(&ps[in + i][4 * ch]);
          if (f != 1.f) a *= f;
          if (g != 0.f) a += g * y;
          z = z * f + g * ps[in + i][D + 1];
          m = x;
        }
      }
    }
    if (!live || k) continue;
    const int tk = over_g(p, row0 + row), g = row0 + row - tk * p.G;
    const int64_t at = (int64_t)(t.s.c0 + tk) * p.Hkv * p.G + t.h * p.G + g;
    const float f = tree_empty(p, t.s.c0 + tk, t.s) ? 0.f : 1.f / z;   // (a sum of 0 over keys that are seen is no number)
    const float y[4] = {a[0] * f, a[1] * f, a[2] * f, a[3] * f};
    st4<T>((T*)p.out + at * D + 4 * ch, y);
    if (p.lse && ch == 0) p.lse[at] = z == 0.f ? -INFINITY : kLn2 * (m + __log2f(z));
  }
}
template <class T, int D, int BM, int UNIT, int UNITS> void launch_tree_join(const AF& p, unsigned W, int64_t tasks, hipStream_t st) {
  if (W <= 1) return;
  const unsigned x = (unsigned)std::min<int64_t>(W - 1, tasks), y = std::min<unsigned>(BM, (2048 + x - 1) / x);
  if (tasks < W) hipLaunchKernelGGL((k_tree_join<T, D, BM, UNIT, UNITS, true>), dim3(x, y), dim3(256), 0, st, p, (int)W);
  else hipLaunchKernelGGL((k_tree_join<T, D, BM, UNIT, UNITS, false>), dim3(x, y), dim3(256), 0, st, p, (int)W);
}

}  // namespace
}  // namespace dn
