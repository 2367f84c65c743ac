// Attention of drafted trees over a paged cache: many rows per key head (new tokens
// times the heads of a group) over long contexts, the keys split over the card.
//
// A tile of query rows stays in a workgroup's registers, keys and values come through
// LDS a tile ahead by direct loads, and a workgroup takes an even share of all
// sequences' keys, wherever tiles of rows begin and end in it; what several hold parts
// of is joined by a second launch.  Only the last keys, the trees' own, are masked.
#include <type_traits>

#include "dn_attn_split.h"

namespace dn {
namespace {

// NW waves of 16 NQ rows, tiles of BN keys.
template <class T, int D, int NQ, int NW, int BN>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 2 : 1) void k_attn_tree(const AF p) {
  using TL = Tile<T, D, BN>;
  using F = typename At<T>::F;
  constexpr float kLift = std::is_same<T, f16>::value ? 7.f : 0.f;   // (as in the kernel of few rows)
  constexpr int BM = 16 * NQ * NW, NS = D / 32, NC = D / 16;
  __shared__ __align__(16) T lds[4 * BN * D];   // [2][K, V][BN][D]
  const int l = lane_id(), r = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const float scale = exponent_scale(p);
  const Rest rest(p);
  const PlanOf<true> plan(p, BM, BN);
  rest.clear<T, D>(p);
  const int W = min((int)gridDim.x, plan.C);
  if ((int)blockIdx.x >= W) return;
  int u = first_unit(blockIdx.x, W, plan.C);
  const int uend = first_unit(blockIdx.x + 1, W, plan.C);
#pragma unroll 1
  while (u < uend) {
    Task t;
    if (!plan.of_unit(u, t)) break;
    const int rows = t.s.n * p.G, row0 = t.m * BM, off = t.s.len - t.s.n, last = max(t.s.len - 1, 0);
    int k0, k1;
    units_of<true>(p, t.s, 0, 1, BN, k0, k1);
    const int skip = u - t.first, take = min(t.units - skip, uend - u);
    const int j0 = k0 + skip, j1 = j0 + take;
    const int lo1 = p.window ? max(off + min(t.s.n, 64 * p.words) - p.window, 0) : 0;   // no row's first key is later

    F qf[NQ][NS];
    int token[NQ], low[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int row = min(row0 + (w * NQ + i) * 16 + r, rows - 1);
      const int tk = over_g(p, row), g = row - tk * p.G;
      const T* qp = (const T*)p.q + (p.cu ? (int64_t)(t.s.c0 + tk) * p.qs[1] : t.b * p.qs[0] + tk * p.qs[1]) + (t.h * p.G + g) * p.qs[2];
#pragma unroll
      for (int c = 0; c < NS; ++c) qf[i][c] = *reinterpret_cast<const F*>(qp + 32 * c + 8 * q);
      if (p.sc < 0.f)
#pragma unroll
        for (int c = 0; c < NS; ++c) qf[i][c] = minus8<T>(qf[i][c]);
      token[i] = t.s.c0 + tk;
      low[i] = tree_low(p, tree_words(p, token[i]), off, t.s.n);
    }
    Rows<T, true> kr, vr;
    kr.base = (const T*)p.k + t.h * p.ks[2];
    vr.base = (const T*)p.v + t.h * p.vs[2];
    kr.token = p.ks[1]; vr.token = p.vs[1];
    kr.page = p.ks[0]; vr.page = p.vs[0];
    kr.pt = vr.pt = p.pt + t.b * p.pts;
    kr.shift = vr.shift = p.shift;
    kr.pages = vr.pages = p.pages;
    kr.last = vr.last = last;
    auto fetch = [&](int j) {
      T* to = lds + (j - j0 & 1) * 2 * BN * D;
      TL::template load<NW>(to, w, [&](int x) { return kr(j * BN + x); });
      TL::template load<NW>(to + BN * D, w, [&](int x) { return vr(j * BN + x); });
    };
    f32x4 o[NQ][NC];
    float mx[NQ], sum[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      mx[i] = -INFINITY;
      sum[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c] = zero4();
    }
    bool odd = false;
    auto step = [&](auto masked, const T* kt, const T* vt, int key0) {
      constexpr bool MASKED = decltype(masked)::value;
      f32x4 sc[NQ][2];
#pragma unroll
      for (int i = 0; i < NQ; ++i) sc[i][0] = sc[i][1] = zero4();
#pragma unroll
      for (int c = 0; c < NS; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const F kf = TL::row8(kt, 16 * e + r, c, q);
#pragma unroll
          for (int i = 0; i < NQ; ++i) At<T>::mma(sc[i][e], kf, qf[i][c]);
        }
      float mt[NQ];
      bool grow = false;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (MASKED) {
          const uint32_t bits = tree_bits(p, tree_words(p, token[i]), off, t.s.len, low[i], key0) >> (4 * q);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[i][e][x] = bits >> (16 * e + x) & 1 ? sc[i][e][x] : -INFINITY;
        }
        const float m = fmaxf(fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3])),
                              fmaxf(fmaxf(sc[i][1][0], sc[i][1][1]), fmaxf(sc[i][1][2], sc[i][1][3])));
        mt[i] = max_q(m) * scale - kLift;
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
          for (int c = 0; c < NC; ++c) o[i][c] *= f;
        }
      }
      F pf[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const float m = mx[i] == -INFINITY ? 0.f : mx[i];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            sc[i][e][x] = fast_exp2(__builtin_fmaf(sc[i][e][x], scale, -m));
            sum[i] += sc[i][e][x];
          }
        pf[i] = frag8<T>(sc[i][0], sc[i][1]);
      }
      const bool bad = MASKED && TL::odd32(vt);
      if (MASKED) odd |= bad;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        F vf = TL::col8(vt, c, r, q);
        if (MASKED && bad) vf = finite8<T>(vf);
#pragma unroll
        for (int i = 0; i < NQ; ++i) At<T>::mma(o[i][c], vf, pf[i]);
      }
    };
    auto masked_step = [&](int key0) { return key0 + 31 >= off || key0 < lo1; };
    fetch(j0);
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
      loads_barrier();   // the tiles are there, those before them no longer read
      if (j + 1 < j1) fetch(j + 1);
      const T* kt = lds + (j - j0 & 1) * 2 * BN * D;
      const T* vt = kt + BN * D;
      if (masked_step(j * BN) || masked_step(j * BN + BN - 32)) {
#pragma unroll 1
        for (int x = 0; x < BN; x += 32) step(std::true_type{}, kt + x * 32, vt + x * 32, j * BN + x);
      } else {
#pragma unroll
        for (int x = 0; x < BN; x += 32) step(std::false_type{}, kt + x * 32, vt + x * 32, j * BN + x);
      }
    }
    if (odd) {   // infinities and NaNs that some row must not see: to those that do
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll 1
          for (int j = j0; j < j1; ++j) {
            if (!(masked_step(j * BN) || masked_step(j * BN + BN - 32))) continue;
#pragma unroll 1
            for (int key = j * BN; key < min((j + 1) * BN, t.s.len); ++key) {
              if (!(tree_bits(p, tree_words(p, token[i]), off, t.s.len, low[i], key & ~31) >> (key & 31) & 1)) continue;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float y = (float)vr(key)[16 * c + 4 * q + e];
                if (!__builtin_isfinite(y)) o[i][c][e] += y;
              }
            }
          }
        }
    }
    const bool whole = take == t.units;
    float* slot = p.part + (2 * (int64_t)blockIdx.x + (skip == 0 ? 1 : 0)) * slot_floats<D, BM>();
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const float z = sum_q(sum[i]);
      const int in = (w * NQ + i) * 16 + r, row = row0 + in;
      if (row >= rows) continue;
      if (whole) {
        const int tk = over_g(p, row), g = row - tk * p.G;
        const int64_t at = (int64_t)(t.s.c0 + tk) * p.Hkv * p.G + t.h * p.G + g;
        const float f = tree_empty(p, token[i], t.s) ? 0.f : 1.f / z;   // (a sum of 0 over keys that are seen is no number)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float y[4] = {o[i][c][0] * f, o[i][c][1] * f, o[i][c][2] * f, o[i][c][3] * f};
          st4<T>((T*)p.out + at * D + 16 * c + 4 * q, y);
        }
        if (p.lse && q == 0) p.lse[at] = z == 0.f ? -INFINITY : kLn2 * (mx[i] + __log2f(z));
      } else {
#pragma unroll
        for (int c = 0; c < NC; ++c) *reinterpret_cast<f32x4*>(slot + in * D + 16 * c + 4 * q) = o[i][c];
        if (q == 0) {
          slot[BM * D + in] = mx[i];
          slot[BM * D + BM + in] = z;
        }
      }
    }
    __syncthreads();   // the next piece's tiles go where these are read
    u += take;
  }
}

// Workgroups: as many as the card holds at once, and no more than there can be units.
int64_t most_tasks(const AF& p, int BM) {
  return (p.cu ? (int64_t)p.N * p.G / BM + p.B : (int64_t)p.B * (((int64_t)p.T * p.G + BM - 1) / BM)) * p.Hkv;
}
template <class T, int D> struct Form {
  static constexpr int NQ = sizeof(T) == 4 || D < 256 ? 2 : 1, NW = sizeof(T) == 4 || D < 256 ? 4 : 8, BN = sizeof(T) == 4 ? 32 : 64;
  static constexpr int BM = 16 * NQ * NW;
  static constexpr int per_cu = 4 * BN * D * (int)sizeof(T) <= 80 * 1024 && sizeof(T) == 2 ? 2 : 1;
  static int64_t groups(const AF& p) {
    return std::min<int64_t>(256 * per_cu, most_tasks(p, BM) * ((((int64_t)p.max_pages << p.shift) + BN - 1) / BN));
  }
  static size_t bytes(const AF& p) { return (size_t)groups(p) * 2 * BM * (D + 2) * sizeof(float); }
  static hipError_t run(const AF& p, hipStream_t st) {
    const unsigned W = (unsigned)groups(p), rows = (unsigned)p.N * p.Hkv * p.G;
    hipLaunchKernelGGL((k_attn_tree<T, D, NQ, NW, BN>), dim3(W), dim3(64 * NW), 0, st, p);
    if (W > 1) hipLaunchKernelGGL((k_attn_join<T, D, BM, BN, true>), dim3(rows), dim3(256), 0, st, p, (int)W);
    return hipGetLastError();
  }
};

template <class G> auto by_form(int D, int dtype, G g) {
  auto go = [&](auto z) {
    using T = decltype(z);
    return D == 64 ? g(Form<T, 64>{}) : D == 128 ? g(Form<T, 128>{}) : g(Form<T, 256>{});
  };
  return dtype == DN_BF16 ? go((bf16)0.f) : dtype == DN_F16 ? go((f16)0.f) : go(0.f);
}

// Rows that fill a tile of the kernel of few rows; pages of 16 tokens at least there.
bool few(const AF& p) { return p.shift >= 4 && (int64_t)p.N * p.G <= (int64_t)32 * p.B; }

}  // namespace

size_t attn_tree_bytes(const AF& p, int D, int dtype) {
  if (few(p)) return attn_few_bytes(p, D);
  return by_form(D, dtype, [&](auto f) { return decltype(f)::bytes(p); });
}

hipError_t attn_tree(const AF& p, int D, int dtype, hipStream_t st) {
  if (few(p)) return attn_few(p, D, dtype, st);
  return by_form(D, dtype, [&](auto f) { return decltype(f)::run(p, st); });
}

}  // namespace dn
