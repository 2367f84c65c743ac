// Gradient of causal softmax attention.
//
// With P = exp(scale S - lse) and delta = rowsum(dO O):
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q.
// Probabilities are recomputed from lse.  Two kernels, so that every sum runs in
// one place in a fixed order: by keys (dK, dV; a workgroup walks over the query
// rows of all heads of its group, which is the sum over them too) and by query
// rows (dQ).  That is seven products for the five of a single pass, whose third
// output would have to be added up in memory.
//
// Bound as the forward is, by the matrix units and the waits on LDS and barriers.
// 2 x 8192 tokens, D = 128, in us and share of the matrix units' time: by keys 1344
// to 1440, 38 % (half of its reads miss the L2s); by rows 740 to 790, 52 %; delta 30,
// 201 MB at 6.6 TB/s.  2048 tokens in documents, D = 256: 117 + 12, 80, delta 9.
#include <type_traits>

#include "dn_attn_fwd.h"

namespace dn {
namespace {

// float16 holds 2^-14 to 2^15 with all of its bits; probabilities of long rows and
// score gradients of small cotangents lie below.  Probabilities carry 2^14
// (kProb16, in the exponent that makes them).  Score gradients carry a power of two
// per query (dQ) or key (dK): their largest so far is 2^7 to 2^15 with it, and when
// one gets larger the power is lowered, and the sums made with it are too.
// 2 x 8192 tokens, D = 128: 2310 us for the whole gradient, 2070 without (the check
// splits what the compiler would interleave; the power in dQ's exponents and delta
// in dP's accumulators, which saves as many instructions as this adds, spills: 2400).
constexpr float kProb16 = 14.f, kFirst16 = 0x1p100f;
template <int N, int NC> __device__ __forceinline__ void fit16(f32x4 (&d)[N][2], f32x4 (&acc)[N][NC], float (&power)[N]) {
  float top[N];
  bool over = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    top[i] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int z = 0; z < 4; ++z) top[i] = fmaxf(top[i], fabsf(d[i][e][z]));
    over |= top[i] * power[i] > 0x1p15f;
  }
  if (__any(over)) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float m = max_q(top[i]);
      const bool lower = m * power[i] > 0x1p15f && m < INFINITY;
      const float next = lower ? __builtin_ldexpf(1.f, 8 - __builtin_amdgcn_frexp_expf(m)) : power[i];
      const float f = next / power[i];
      power[i] = next;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[i][c] *= f;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) d[i][e] *= power[i];
}

// delta = sum of d_out * (out + out_low) over a row's channels: D/8 lanes per row
template <class T, int D>
__global__ __launch_bounds__(256) void k_attn_delta(const AB p, int64_t rows) {
  constexpr int per = D / 8;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / per;
  float s = 0.f;
  if (row < rows) {
    typedef T V __attribute__((ext_vector_type(8)));
    const V a = reinterpret_cast<const V*>(p.d_out)[id], b = reinterpret_cast<const V*>(p.f.out)[id];
#pragma unroll
    for (int e = 0; e < 8; ++e) s += (float)a[e] * (float)b[e];
    if (p.f.low) {
      const V c = reinterpret_cast<const V*>(p.f.low)[id];
#pragma unroll
      for (int e = 0; e < 8; ++e) s += (float)a[e] * (float)c[e];
    }
  }
#pragma unroll
  for (int o = 1; o < per; o <<= 1) s += __shfl_xor(s, o);
  if (row < rows && id % per == 0) p.delta[row] = s;
}

// Query rows are (token, head of the group), token first.
template <class T> struct QRows {
  const T *q, *g;       // q and d_out of the sequence and key head
  int64_t qt, qh, gt, gh;
  int G, last;
  const AF* f;
  __device__ __forceinline__ const T* query(int row) const {
    row = min(row, last);
    const int t = over_g(*f, row);
    return q + t * qt + (row - t * G) * qh;
  }
  __device__ __forceinline__ const T* grad(int row) const {
    row = min(row, last);
    const int t = over_g(*f, row);
    return g + t * gt + (row - t * G) * gh;
  }
};

// The last token whose document starts at or before key k1 (starts is
// nondecreasing and starts[k1] <= k1), by all lanes of a wave.
__device__ __forceinline__ int last_token(const int32_t* starts, int T, int k1) {
  int lo = k1, hi = T;   // starts[lo] <= k1, hi: T or the first known above
  while (hi - lo > 1) {
    const int step = (hi - lo + 64) / 65;
    const int t = lo + (lane_id() + 1) * step;
    const unsigned long long in = __ballot(t < hi && starts[min(t, T - 1)] <= k1);
    const int n = __popcll(in);
    const int nlo = lo + n * step;
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  return lo;
}

// dK and dV of 64 NK keys of one key head: every S-th tile of query rows from the
// blockIdx.y-th on, of S = gridDim.y.  (From the last tile down, all workgroups of a
// head reading the same rows at a time, is slower: 1658 against 1542 us at 2 x 8192,
// though fewer reads go past L2.)  With S > 1 the sums go to p.part, as
// floats, and are added up by k_attn_dkv_sum.
//
// 16 NK keys belong to two waves of one SIMD: one forms S and P and sums up dV,
// the other dP and dS, for which it takes P from the first through LDS, and dK.
// Each holds half of the operands and sums that one wave would (two waves fit on
// a SIMD) and reads half of the tiles' LDS: against one wave for all of it 116 and
// 137 us at D = 256 (2048 tokens).
template <class T, int D, int NK, int BQ>
__global__ __launch_bounds__(512, sizeof(T) == 2 ? 2 : 1) void k_attn_dkv(const AB p) {
  using TL = Tile<T, D, BQ>;
  using F = typename At<T>::F;
  constexpr int NW = 8, BN = 64 * NK, NS = D / 32, NC = D / 16, RS = 32, NE = RS / 16;   // RS: query rows of a step
  constexpr bool F16 = std::is_same<T, f16>::value;
  __shared__ __align__(16) T lds[4 * BQ * D];    // [2][q, d_out][BQ][D]
  __shared__ __align__(16) f32x4 px[2][4][NK * NE * 64];  // P of a step, by its parity and the pair, as accumulators
  __shared__ __align__(16) float ls[2][BQ], de[2][BQ];   // lse * log2(e) and delta per row
  __shared__ __align__(16) int tk[2][BQ], lw[2][BQ];     // token and first visible key per row
  const AF& f = p.f;

  const int l = lane_id(), r = l & 15, q = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pair = wave & 3;
  const bool first = wave < 4;   // S, P, dV; the others dP, dS, dK
  // batch row and head innermost; the first keys, which most queries see, first
  const int groups = f.B * f.Hkv, gi = blockIdx.x % groups;
  const int b = gi / f.Hkv, h = gi % f.Hkv, k0 = (int)(blockIdx.x / groups) * BN;
  const int k1 = min(k0 + BN, f.T) - 1;
  const int32_t* starts = f.start ? f.start + (int64_t)b * f.T : nullptr;

  int t1 = f.T - 1;   // the last token that sees one of the keys
  if (f.window) t1 = (int)min((int64_t)t1, (int64_t)k1 + f.window - 1);
  if (starts) t1 = min(t1, __builtin_amdgcn_readfirstlane(last_token(starts, f.T, k1)));

  const int key = k0 + pair * NK * 16 + r;
  F own[NK][NS];   // K or V
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int64_t t = min(key + 16 * i, f.T - 1);
    const T* s = first ? (const T*)f.k + b * f.ks[0] + t * f.ks[1] + h * f.ks[2] : (const T*)f.v + b * f.vs[0] + t * f.vs[1] + h * f.vs[2];
#pragma unroll
    for (int c = 0; c < NS; ++c) own[i][c] = *reinterpret_cast<const F*>(s + 32 * c + 8 * q);
  }

  const int Hq = f.Hkv * f.G;
  QRows<T> rows;
  rows.q = (const T*)f.q + b * f.qs[0] + (int64_t)h * f.G * f.qs[2];
  rows.qt = f.qs[1]; rows.qh = f.qs[2];
  rows.g = (const T*)p.d_out + ((int64_t)b * f.T * Hq + h * f.G) * D;
  rows.gt = (int64_t)Hq * D; rows.gh = D;
  rows.G = f.G; rows.last = f.T * f.G - 1; rows.f = &f;
  const int S = gridDim.y;
  const int r0 = k0 * f.G / BQ + blockIdx.y, r1 = (t1 * f.G + f.G - 1) / BQ + 1;   // tiles of query rows, by S

  f32x4 acc[NK][NC];   // dV or dK, transposed
#pragma unroll
  for (int i = 0; i < NK; ++i)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[i][c] = zero4();

#pragma unroll
  for (int i = 0; i < NK; ++i)
#pragma unroll
    for (int c = 0; c < NS; ++c) settle(own[i][c]);
  float m_ls = 0.f, m_de = 0.f;
  int m_tk = 0, m_lw = 0, m_hi = 0;   // m_hi: first visible key of the tile's last row
  auto fetch = [&](int j, int buf) {
    T* t = lds + buf * 2 * BQ * D;
    TL::template load<NW>(t, wave, [&](int x) { return rows.query(j * BQ + x); });
    TL::template load<NW>(t + BQ * D, wave, [&](int x) { return rows.grad(j * BQ + x); });
    auto low = [&](int t) {
      int x = f.window ? max(t - f.window + 1, 0) : 0;
      return starts ? max(x, starts[t]) : x;
    };
    if (threadIdx.x < BQ) {
      const int row = j * BQ + threadIdx.x, c = min(row, rows.last), tok = over_g(f, c);
      const int64_t at = ((int64_t)b * f.T + tok) * Hq + h * f.G + (c - tok * f.G);
      m_ls = f.lse[at] * kLog2e - (F16 ? kProb16 : 0.f);
      m_de = p.delta[at];
      m_tk = row <= rows.last ? tok : -1;   // a row past the last one sees no key
      m_lw = low(tok);
    }
    m_hi = low(over_g(f, min(j * BQ + BQ - 1, rows.last)));
  };
  bool odd = false;
  float power[NK];   // of the keys' score gradients (F16)
#pragma unroll
  for (int i = 0; i < NK; ++i) power[i] = kFirst16;
  // The parts of a step of RS query rows.  Both waves multiply rows x by their own
  // operand (forward) and rows y, transposed, by the result (back).
  using Acc = f32x4[NK][NE];
  auto forward = [&](Acc& s, const T* x) {
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
      for (int e = 0; e < NE; ++e) s[i][e] = zero4();
    constexpr int B = NS < 4 ? NS : 4;   // slabs of a batch
    F xf[2][B][NE];
    batches<NS / B, true>([&](int b) {
#pragma unroll
      for (int c = 0; c < B; ++c)
#pragma unroll
        for (int e = 0; e < NE; ++e) xf[b & 1][c][e] = TL::row8(x, 16 * e + r, b * B + c, q);
    }, [&](int b) {
#pragma unroll
      for (int c = 0; c < B; ++c)
#pragma unroll
        for (int e = 0; e < NE; ++e)
#pragma unroll
          for (int i = 0; i < NK; ++i) At<T>::mma(s[i][e], xf[b & 1][c][e], own[i][b * B + c]);
    });
  };
  // S to P, and to the other wave; MASKED: some of the rows must not see some key
  auto probabilities = [&](auto mask, Acc& s, int buf, int u) {
    constexpr bool MASKED = decltype(mask)::value;
    f32x4* ex = px[u / RS & 1][pair] + l;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const int at = u + 16 * e + 4 * q;
      const f32x4 lse = *reinterpret_cast<const f32x4*>(&ls[buf][at]);
#pragma unroll
      for (int i = 0; i < NK; ++i) {
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          s[i][e][z] = fast_exp2(__builtin_fmaf(s[i][e][z], f.sc, -lse[z]));
          if (MASKED) s[i][e][z] = key + 16 * i <= tk[buf][at + z] && key + 16 * i >= lw[buf][at + z] ? s[i][e][z] : 0.f;
        }
        ex[(i * NE + e) * 64] = s[i][e];
      }
    }
  };
  auto take = [&](Acc& pr, int u) {
    const f32x4* ex = px[u / RS & 1][pair] + l;
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int i = 0; i < NK; ++i) pr[i][e] = ex[(i * NE + e) * 64];
  };
  // dP to dS
  auto differences = [&](auto mask, Acc& s, const Acc& pr, int buf, int u) {
    constexpr bool MASKED = decltype(mask)::value;
#pragma unroll
    for (int e = 0; e < NE; ++e) {
      const f32x4 del = *reinterpret_cast<const f32x4*>(&de[buf][u + 16 * e + 4 * q]);
#pragma unroll
      for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float d = pr[i][e][z] * (s[i][e][z] - del[z]);
          s[i][e][z] = MASKED && pr[i][e][z] == 0.f ? 0.f : d;   // (hidden rows of d_out may hold anything)
        }
    }
    if constexpr (F16) fit16(s, acc, power);
  };
  auto back = [&](auto mask, const Acc& s, const T* y) {
    constexpr bool MASKED = decltype(mask)::value;
    F sf[NK], yc[2][4];
#pragma unroll
    for (int i = 0; i < NK; ++i) sf[i] = frag8<T>(s[i][0], s[i][1]);
    const bool bad = MASKED && TL::odd32(y);
    if (MASKED) odd |= bad;
    batches<NC / 4, true>([&](int b) {
#pragma unroll
      for (int c = 0; c < 4; ++c) yc[b & 1][c] = TL::col8(y, b * 4 + c, r, q);
    }, [&](int b) {
      if (MASKED && bad) {
#pragma unroll
        for (int c = 0; c < 4; ++c) yc[b & 1][c] = finite8<T>(yc[b & 1][c]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NK; ++i) At<T>::mma(acc[i][b * 4 + c], yc[b & 1][c], sf[i]);
    });
  };
  auto step = [&](auto mask, const T* x, const T* y, int buf, int u) {
    Acc s, pr;
    forward(s, x);
    if (first) probabilities(mask, s, buf, u);
    lds_barrier();
    if (!first) {
      take(pr, u);
      differences(mask, s, pr, buf, u);
    }
    back(mask, s, y);
  };
  if (r0 < r1) fetch(r0, 0);
  int buf = 0;
#pragma unroll 1
  for (int j = r0; j < r1; j += S, buf ^= 1) {
    if (threadIdx.x < BQ) {
      ls[buf][threadIdx.x] = m_ls;
      de[buf][threadIdx.x] = m_de;
      tk[buf][threadIdx.x] = m_tk;
      lw[buf][threadIdx.x] = m_lw;
    }
    const bool masked = over_g(f, j * BQ) < k1 || m_hi > k0 || j * BQ + BQ - 1 > rows.last;
    loads_barrier();
    if (j + S < r1) fetch(j + S, buf ^ 1);
    const T* x = lds + buf * 2 * BQ * D + (first ? 0 : BQ * D);
    const T* y = lds + buf * 2 * BQ * D + (first ? BQ * D : 0);
    if (masked) {
#pragma unroll 1
      for (int u = 0; u < BQ; u += RS) step(std::true_type{}, x + u * 32, y + u * 32, buf, u);
    } else {
#pragma unroll
      for (int u = 0; u < BQ; u += RS) step(std::false_type{}, x + u * 32, y + u * 32, buf, u);
    }
  }

  const int64_t n = (int64_t)f.N * f.Hkv * D;
  T* const dst = (T*)(first ? p.dv : p.dk);
  float* const part = p.part + ((int64_t)blockIdx.y * 2 + (first ? 1 : 0)) * n;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int t = key + 16 * i;
    if (t >= f.T) continue;
    const int64_t at = (((int64_t)b * f.T + t) * f.Hkv + h) * D;
    const float back16 = first ? 0x1p-14f : 0x1p-14f / power[i];   // 2^-kProb16
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if constexpr (F16) acc[i][c] *= back16;
      float x[4] = {acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]};
      if (first && odd) {   // what the queries that see this key had left out of dV (dK of such a query is NaN by its scores)
#pragma unroll 1
        for (int row = r0 * BQ; row <= min(r1 * BQ - 1, rows.last); ++row) {
          const int tok = over_g(f, row);
          if ((row / BQ - r0) % S || tok < t) continue;
          int lo = f.window ? max(tok - f.window + 1, 0) : 0;
          if (starts) lo = max(lo, starts[tok]);
          const int j = row / BQ, tl = over_g(f, min(j * BQ + BQ - 1, rows.last));
          int hi = f.window ? max(tl - f.window + 1, 0) : 0;
          if (starts) hi = max(hi, starts[tl]);
          if (t < lo || !(over_g(f, j * BQ) < k1 || hi > k0 || j * BQ + BQ - 1 > rows.last)) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float z = (float)rows.grad(row)[16 * c + 4 * q + e];
            if (!__builtin_isfinite(z)) x[e] += z;
          }
        }
      }
      if (S == 1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = first ? x[e] : x[e] * p.scale;
        st4<T>(dst + at + 16 * c + 4 * q, x);
      } else {
        st4<float>(part + at + 16 * c + 4 * q, x);
      }
    }
  }
}

// dK and dV from S parts of each, in their order: 4 elements per thread.
template <class T>
__global__ __launch_bounds__(256) void k_attn_dkv_sum(const AB p, int64_t n, int S) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= 2 * n) return;
  f32x4 a = *reinterpret_cast<const f32x4*>(p.part + i);
#pragma unroll 4
  for (int s = 1; s < S; ++s) a += *reinterpret_cast<const f32x4*>(p.part + s * 2 * n + i);
  const float f = i < n ? p.scale : 1.f;
  const float x[4] = {a[0] * f, a[1] * f, a[2] * f, a[3] * f};
  st4<T>((i < n ? (T*)p.dk + i : (T*)p.dv + (i - n)), x);
}

// dQ of 16 NQ NW query rows: the forward's walk over the keys.
template <class T, int D, int NQ, int NW, int BN>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 2 : 1) void k_attn_dq(const AB p) {
  using TL = Tile<T, D, BN>;
  using F = typename At<T>::F;
  constexpr int BM = 16 * NQ * NW, NS = D / 32, NC = D / 16;
  constexpr bool F16 = std::is_same<T, f16>::value;
  __shared__ __align__(16) T lds[4 * BN * D];   // [2][K, V][BN][D]
  const AF& f = p.f;

  const int l = lane_id(), r = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = f.B * f.Hkv, gi = blockIdx.x % groups, tiles = gridDim.x / groups;
  const int b = gi / f.Hkv, h = gi % f.Hkv, row0 = (tiles - 1 - (int)(blockIdx.x / groups)) * BM;
  const int nrow = f.T * f.G, row1 = min(row0 + BM, nrow);
  const int p0 = over_g(f, row0), p1 = over_g(f, row1 - 1);
  const int32_t* starts = f.start ? f.start + (int64_t)b * f.T : nullptr;
  const int Hq = f.Hkv * f.G;

  F qf[NQ][NS], gf[NQ][NS];
  int pos[NQ], low[NQ];
  float ls[NQ], de[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = min(row0 + (w * NQ + i) * 16 + r, nrow - 1);
    const int t = over_g(f, row), g = row - t * f.G;
    const int64_t at = ((int64_t)b * f.T + t) * Hq + h * f.G + g;
    const T* qp = (const T*)f.q + b * f.qs[0] + t * f.qs[1] + (h * f.G + g) * f.qs[2];
    const T* gp = (const T*)p.d_out + at * D;
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      qf[i][c] = *reinterpret_cast<const F*>(qp + 32 * c + 8 * q);
      gf[i][c] = *reinterpret_cast<const F*>(gp + 32 * c + 8 * q);
    }
    ls[i] = f.lse[at] * kLog2e;
    de[i] = p.delta[at];
    pos[i] = t;
    low[i] = f.window ? t - f.window + 1 : 0;
    if (starts) low[i] = max(low[i], starts[t]);
  }
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      settle(qf[i][c]);
      settle(gf[i][c]);
    }
    settle(ls[i]);
    settle(de[i]);
    settle(low[i]);
  }
  int lo0 = f.window ? max(p0 - f.window + 1, 0) : 0, lo1 = f.window ? p1 - f.window + 1 : 0;
  if (starts) {
    lo0 = max(lo0, starts[p0]);
    lo1 = max(lo1, starts[p1]);
  }
  const int j0 = lo0 / BN, j1 = p1 / BN + 1;

  Rows<T, false> kr{}, vr{};
  kr.base = (const T*)f.k + b * f.ks[0] + h * f.ks[2];
  vr.base = (const T*)f.v + b * f.vs[0] + h * f.vs[2];
  kr.token = f.ks[1]; vr.token = f.vs[1];
  kr.last = vr.last = p1;

  f32x4 dq[NQ][NC];
  float power[NQ];   // of the rows' score gradients (F16)
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    power[i] = kFirst16;
#pragma unroll
    for (int c = 0; c < NC; ++c) dq[i][c] = zero4();
  }

  auto fetch = [&](int j) {
    T* t = lds + (j & 1) * 2 * BN * D;
    TL::template load<NW>(t, w, [&](int x) { return kr(j * BN + x); });
    TL::template load<NW>(t + BN * D, w, [&](int x) { return vr(j * BN + x); });
  };
  // 32 keys of a tile; MASKED: some query must not see some of them
  auto step = [&](auto mask, const T* kt, const T* vt, int key0) {
    constexpr bool MASKED = decltype(mask)::value;
    f32x4 s[NQ][2], dp[NQ][2];
#pragma unroll
    for (int i = 0; i < NQ; ++i) s[i][0] = s[i][1] = dp[i][0] = dp[i][1] = zero4();
    if constexpr (D == 256) {
      F kf[2][2][2], vf[2][2][2];
      batches<NS / 2, true>([&](int b) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            kf[b & 1][c][e] = TL::row8(kt, 16 * e + r, b * 2 + c, q);
            vf[b & 1][c][e] = TL::row8(vt, 16 * e + r, b * 2 + c, q);
          }
      }, [&](int b) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
              At<T>::mma(s[i][e], kf[b & 1][c][e], qf[i][b * 2 + c]);
              At<T>::mma(dp[i][e], vf[b & 1][c][e], gf[i][b * 2 + c]);
            }
      });
    } else {
#pragma unroll
      for (int c = 0; c < NS; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const F kf = TL::row8(kt, 16 * e + r, c, q);
          const F vf = TL::row8(vt, 16 * e + r, c, q);
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            At<T>::mma(s[i][e], kf, qf[i][c]);
            At<T>::mma(dp[i][e], vf, gf[i][c]);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float pr = fast_exp2(__builtin_fmaf(s[i][e][x], f.sc, -ls[i]));
          dp[i][e][x] = pr * (dp[i][e][x] - de[i]);
          if (MASKED) {
            const int key = key0 + 16 * e + 4 * q + x;
            dp[i][e][x] = key <= pos[i] && key >= low[i] ? dp[i][e][x] : 0.f;
          }
        }
    if constexpr (F16) fit16(dp, dq, power);
    F df[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) df[i] = frag8<T>(dp[i][0], dp[i][1]);
    const bool bad = MASKED && TL::odd32(kt);   // (a query that sees such a key is NaN by its scores)
    F kc[2][4];
    batches<NC / 4, D == 256>([&](int b) {
#pragma unroll
      for (int c = 0; c < 4; ++c) kc[b & 1][c] = TL::col8(kt, b * 4 + c, r, q);
    }, [&](int b) {
      if (MASKED && bad) {
#pragma unroll
        for (int c = 0; c < 4; ++c) kc[b & 1][c] = finite8<T>(kc[b & 1][c]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NQ; ++i) At<T>::mma(dq[i][b * 4 + c], kc[b & 1][c], df[i]);
    });
  };
  fetch(j0);
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    loads_barrier();
    if (j + 1 < j1) fetch(j + 1);
    const T* kt = lds + (j & 1) * 2 * BN * D;
    const T* vt = kt + BN * D;
    if (j * BN + BN - 1 > p0 || j * BN < lo1) {
#pragma unroll 1
      for (int u = 0; u < BN; u += 32) step(std::true_type{}, kt + u * 32, vt + u * 32, j * BN + u);
    } else {
#pragma unroll
      for (int u = 0; u < BN; u += 32) step(std::false_type{}, kt + u * 32, vt + u * 32, j * BN + u);
    }
  }

#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = row0 + (w * NQ + i) * 16 + r;
    if (row >= nrow) continue;
    const int t = over_g(f, row), g = row - t * f.G;
    T* op = (T*)p.dq + (((int64_t)b * f.T + t) * Hq + h * f.G + g) * D;
    const float back16 = 1.f / power[i];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if constexpr (F16) dq[i][c] *= back16;
      const float x[4] = {dq[i][c][0] * p.scale, dq[i][c][1] * p.scale, dq[i][c][2] * p.scale, dq[i][c][3] * p.scale};
      st4<T>(op + 16 * c + 4 * q, x);
    }
  }
}

template <class T, int D> struct Shape {
  static constexpr bool f32 = sizeof(T) == 4;
  static constexpr int BT = f32 ? 32 : 64;   // rows of a tile in LDS
  static constexpr int NK = !f32 && D < 256 ? 2 : 1, keys = 64 * NK;
  // dq: 32 rows per wave (767 us at 2 x 8192 tokens, D 128; 16 rows 797); 16 at
  // D = 256 (80 us at 2048 tokens; 32 rows 107 against 87 then)
  static constexpr int NW = 4, NQ = D == 256 ? 1 : 2;
};

// Parts of the walk over query rows, so that dkv fills the card (kFill workgroups),
// none shorter than two tiles of rows: 140 us with the sum in place of 272 at 2048
// tokens, D = 256.
constexpr int64_t kFill = 512;
template <class T, int D> int splits(const AF& f) {
  using Sh = Shape<T, D>;
  const int64_t wg = ((int64_t)f.T + Sh::keys - 1) / Sh::keys * f.B * f.Hkv;
  const int64_t tiles = ((int64_t)f.T * f.G + Sh::BT - 1) / Sh::BT;
  return (int)std::max<int64_t>(1, std::min<int64_t>({kFill / wg, tiles / 2, 8}));
}

template <class T, int D> hipError_t run(const AB& p, hipStream_t st) {
  using Sh = Shape<T, D>;
  constexpr int NW = Sh::NW;
  const AF& f = p.f;
  const int64_t rows = (int64_t)f.N * f.Hkv * f.G, groups = (int64_t)f.B * f.Hkv;
  hipLaunchKernelGGL((k_attn_delta<T, D>), dim3((unsigned)((rows * (D / 8) + 255) / 256)), dim3(256), 0, st, p, rows);
  const int S = splits<T, D>(f);
  const int64_t kt = ((int64_t)f.T + Sh::keys - 1) / Sh::keys;
  hipLaunchKernelGGL((k_attn_dkv<T, D, Sh::NK, Sh::BT>), dim3((unsigned)(kt * groups), S), dim3(512), 0, st, p);
  if (S > 1) {
    const int64_t n = (int64_t)f.N * f.Hkv * D;
    hipLaunchKernelGGL((k_attn_dkv_sum<T>), dim3((unsigned)((2 * n / 4 + 255) / 256)), dim3(256), 0, st, p, n, S);
  }
  // half the rows per wave where that is needed to fill the card: 25 us in place of
  // 39 at 2 x 300 tokens, float32
  const int64_t nrow = (int64_t)f.T * f.G, qt = (nrow + 16 * Sh::NQ * NW - 1) / (16 * Sh::NQ * NW);
  if (Sh::NQ == 2 && qt * groups <= kFill)
    hipLaunchKernelGGL((k_attn_dq<T, D, 1, NW, Sh::BT>), dim3((unsigned)((nrow + 16 * NW - 1) / (16 * NW) * groups)), dim3(64 * NW), 0, st, p);
  else
    hipLaunchKernelGGL((k_attn_dq<T, D, Sh::NQ, NW, Sh::BT>), dim3((unsigned)(qt * groups)), dim3(64 * NW), 0, st, p);
  return hipGetLastError();
}

// f(T, D) for a type and head dimension
template <class F> auto choose(int D, int dtype, F f) {
  auto go = [&](auto z) {
    if (D == 64) return f(z, std::integral_constant<int, 64>{});
    if (D == 128) return f(z, std::integral_constant<int, 128>{});
    return f(z, std::integral_constant<int, 256>{});
  };
  return dtype == DN_BF16 ? go((bf16)0.f) : dtype == DN_F16 ? go((f16)0.f) : go(0.f);
}

}  // namespace

size_t attn_backward_part_bytes(const AF& f, int D, int dtype) {
  const int S = choose(D, dtype, [&](auto z, auto d) { return splits<decltype(z), decltype(d)::value>(f); });
  return S > 1 ? (size_t)S * 2 * f.N * f.Hkv * D * sizeof(float) : 0;
}

hipError_t attn_backward(const AB& p, int D, int dtype, hipStream_t st) {
  return choose(D, dtype, [&](auto z, auto d) { return run<decltype(z), decltype(d)::value>(p, st); });
}

}  // namespace dn
