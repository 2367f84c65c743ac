// Forward softmax attention over many rows: training and prompts.
//
// One pass over the keys per tile of query rows (rows of a key head's whole group,
// token first, so that a tile of keys is read once for all of them): S^T = K Q^T,
// exponentials against a reference that is known before the loop (and raised within
// it in float16 alone), O^T += V^T P^T, everything in registers but the tiles of keys
// and values, which direct loads bring into LDS a tile ahead.  Bound by the matrix
// units and what keeps them waiting, LDS reads and the exponentials of two waves per
// SIMD: 46 % of the matrix units' time at 2 x 8192 tokens, D = 128 (525 to 580 us,
// 950 to 1050 TFLOP/s), 43 % at D = 256 (prompts of 4096 over 4096 cached: 860 to 900
// us, 915 to 957 TFLOP/s), where each LDS operand serves 16 rows, not 32.  A library
// product reaches 1414 TFLOP/s here.
#include <type_traits>

#include "dn_attn_fwd.h"

namespace dn {
namespace {

// One workgroup: NW waves of 16 NQ query rows each over one head's keys, KG times:
// with KG = 2 a second set of waves takes every other tile of keys, and the sums,
// which have the same reference, are added at the end.
template <class T, int D, int NQ, int NW, int KG, int BN, bool PAGED>
__global__ __launch_bounds__(64 * NW * KG, sizeof(T) == 2 ? 2 : 1) void k_attn(const AF p) {
  using TL = Tile<T, D, BN>;
  using F = typename At<T>::F;
  constexpr int BM = 16 * NQ * NW, NS = D / 32, NC = D / 16;
  __shared__ __align__(16) T smem[KG * 4 * BN * D];   // [KG][2][K, V][BN][D]; at the end the other waves' sums
  __shared__ float s_top[KG][BM], s_sum[KG][BM];

  const int l = lane_id(), r = l & 15, q = l >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = wave % NW, kg = wave / NW;
  T* lds = smem + kg * 4 * BN * D;

  // head innermost, then the tiles of all sequences, the last (longest) first
  const int nt = gridDim.x / p.Hkv;
  const int h = blockIdx.x % p.Hkv;
  Seq s;
  const Rest rest(p);
  const bool found = find_tile(p, nt - 1 - (int)(blockIdx.x / p.Hkv), BM, s);
  if constexpr (PAGED) rest.clear<T, D>(p);
  if (!found) return;
  s.b = __builtin_amdgcn_readfirstlane(s.b);
  s.c0 = __builtin_amdgcn_readfirstlane(s.c0);
  s.n = __builtin_amdgcn_readfirstlane(s.n);
  s.m = __builtin_amdgcn_readfirstlane(s.m);
  int len = s.n;
  if (PAGED) len = min(max(p.lens[s.b], 0), p.max_pages << p.shift);
  const int off = len - s.n;                       // position of the first new token
  const int rows = s.n * p.G, row0 = s.m * BM;
  const int row1 = min(row0 + BM, rows);           // the tile's rows
  const int p0 = off + over_g(p, row0), p1 = off + over_g(p, row1 - 1);   // their positions

  const float scale = exponent_scale(p);
  // queries: row -> token row / G, head h G + row % G
  F qf[NQ][NS];
  int pos[NQ], low[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = min(row0 + (w * NQ + i) * 16 + r, rows - 1);
    const int t = over_g(p, row), g = row - t * p.G;
    const T* qp = (const T*)p.q + (p.cu ? (int64_t)(s.c0 + t) * p.qs[1] : s.b * p.qs[0] + t * p.qs[1]) + (h * p.G + g) * p.qs[2];
#pragma unroll
    for (int c = 0; c < NS; ++c) qf[i][c] = *reinterpret_cast<const F*>(qp + 32 * c + 8 * q);
    if (p.sc < 0.f)
#pragma unroll
      for (int c = 0; c < NS; ++c) qf[i][c] = minus8<T>(qf[i][c]);
    pos[i] = off + t;
    low[i] = first_key(p, pos[i]);
    if (!PAGED && p.start) low[i] = max(low[i], p.start[s.b * p.T + t]);
  }
  int lo0 = first_key(p, p0), lo1 = first_key(p, p1);   // first keys of the first and last row
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

  // The exponents' reference is a query's score with itself, which it always sees:
  // no maximum has to be known while the sums run.  Sums of exponentials up to
  // 2^kRange above it are as exact as any in a type with float32's range; the
  // rare row that goes beyond is found at the end, and the tile done again with
  // the maxima that are known then.
  // float16 has no such range, and loses bits below 2^-14: there the own key starts
  // at 2^6, and a row whose largest gets to 2^15 has its reference raised on the way
  // (raise_reference), and what is summed scaled down, so that the largest is 2^8.
  // Half a step, 2^-25, is 2^-31 of a row's largest at most.  (2 x 8192 tokens at
  // D = 128: 594 us, bf16 530; no such check but the own key at 2^-6, as far as the
  // range allows without one, 545 with half of the probabilities' bits gone.)
  constexpr bool F16 = std::is_same<T, f16>::value;
  constexpr float kRange = F16 ? 15.f : 60.f, kOwn = F16 ? 6.f : 0.f, kRaised = 8.f;
  f32x4 o[NQ][NC];
  float mx[NQ], top[NQ], sum[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const T* kp = kr(max(pos[i], 0));
    float x = 0.f;
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      const F kf = *reinterpret_cast<const F*>(kp + 32 * c + 8 * q);
#pragma unroll
      for (int e = 0; e < 8; ++e) x += (float)kf[e] * (float)qf[i][c][e];
    }
    const float own = sum_q(x) * scale;
    mx[i] = pos[i] < 0 || own == -INFINITY ? 0.f : own - kOwn;
  }
  // At D = 256 a tile's loads go out in four parts between the products of the
  // tile before it: all at once they fill the memory queue, and the waves wait to
  // issue (600 to 1600 of 5700 clocks per tile; 893 us for 2 x 4096 tokens over
  // 4096 cached, 1008 otherwise).  At 128 that costs registers that are not there (773 us
  // for 2 x 8192, 580 otherwise).
  constexpr bool SPREAD = D == 256 && BN == 64;
  const T *ks = nullptr, *vs = nullptr;
  T* to = nullptr;
  auto aim = [&](int j) {
    ks = TL::template source<NW>(w, [&](int x) { return kr(j * BN + x); });
    vs = TL::template source<NW>(w, [&](int x) { return vr(j * BN + x); });
    to = lds + ((j - j0) / KG & 1) * 2 * BN * D;
  };
  auto fetch = [&](auto part) {
    constexpr int P = decltype(part)::value;
    if constexpr (P < 2) TL::template load_part<NW, P, 2>(to, w, ks);
    else TL::template load_part<NW, P - 2, 2>(to + BN * D, w, vs);
  };
  auto fetch_all = [&] {
    fetch(std::integral_constant<int, 0>{});
    fetch(std::integral_constant<int, 1>{});
    fetch(std::integral_constant<int, 2>{});
    fetch(std::integral_constant<int, 3>{});
  };
  auto raise_reference = [&] {
    bool over = false;
#pragma unroll
    for (int i = 0; i < NQ; ++i) over |= __builtin_fmaf(top[i], scale, -mx[i]) > kRange;
    if (__builtin_expect(__any(over), 0)) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const float t = max_q(top[i]) * scale;
        const float m = t > mx[i] + kRange ? t - kRaised : mx[i];
        const float f = fast_exp2(mx[i] - m);
        mx[i] = m;
        sum[i] *= f;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[i][c] *= f;
      }
    }
  };
  bool odd = false;   // infinities or NaNs in a masked tile were left out
  // 32 keys of a tile; MASKED: some query must not see some of them.  16-bit types
  // multiply the values by such tiles' probabilities in two parts, SPLIT, where a
  // gradient may follow: short rows and documents lie in them, where the rounding of
  // few probabilities is an error of the output (2.0e-3 to 2.1e-3 of it in bf16, 1.5e-3
  // with both parts) and, by the row sums that read it, of the gradient (dq 2.6e-3,
  // 2.35e-3).  (Over pages: 86.6 to 89.3 us under a window of 1024, 12 x
  // 400 tokens over 3000.)  At D = 256
  // the first values are read under the exponentials and the others VB operands
  // ahead, in this order (1006 against 1066 us for 2 x 4096 tokens over 4096 cached); at 128 the
  // compiler's own order is better (601 against 668 us for 2 x 8192).
  constexpr int VB = D == 256 ? 4 : NC, NB = NC / VB;
  auto in_order = [] {
    if constexpr (D == 256) __builtin_amdgcn_sched_barrier(0);
  };
  auto step = [&](auto masked, auto between, const T* kt, const T* vt, int key0) {
    constexpr bool MASKED = decltype(masked)::value, SPLIT = MASKED && !PAGED && sizeof(T) == 2;
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
    F vf[2][VB];
    auto values = [&](int n) {
#pragma unroll
      for (int c = 0; c < VB; ++c) vf[n & 1][c] = TL::col8(vt, n * VB + c, r, q);
    };
    in_order();
    values(0);
    in_order();
    F pf[NQ], pr[NQ];   // probabilities, and what their rounding cut off
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (MASKED) {
            const int key = key0 + 16 * e + 4 * q + x;
            sc[i][e][x] = key <= pos[i] && key >= low[i] ? sc[i][e][x] : -INFINITY;
          }
          top[i] = fmaxf(top[i], sc[i][e][x]);
        }
    if constexpr (F16) raise_reference();
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          sc[i][e][x] = fast_exp2(__builtin_fmaf(sc[i][e][x], scale, -mx[i]));
          sum[i] += sc[i][e][x];
        }
      pf[i] = frag8<T>(sc[i][0], sc[i][1]);
      if constexpr (SPLIT) pr[i] = rest8<T>(sc[i][0], sc[i][1], pf[i]);
    }
    between();
    const bool bad = MASKED && TL::odd32(vt);
    if (MASKED) odd |= bad;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if (n + 1 < NB) values(n + 1);
      in_order();
      if (MASKED && bad) {
#pragma unroll
        for (int c = 0; c < VB; ++c) vf[n & 1][c] = finite8<T>(vf[n & 1][c]);
      }
#pragma unroll
      for (int c = 0; c < VB; ++c)
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
          At<T>::mma(o[i][n * VB + c], vf[n & 1][c], pf[i]);
          if constexpr (SPLIT) At<T>::mma(o[i][n * VB + c], vf[n & 1][c], pr[i]);
        }
    }
  };
  // the waits for the queries land here and not, for all loads in flight there, in
  // every trip of the loop (registers pinned by settle() instead: 1041 us for 987)
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
#pragma unroll 1
  for (int pass = 0;; ++pass) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      top[i] = -INFINITY;
      sum[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c] = zero4();
    }
    if (j0 + kg < j1) {
      aim(j0 + kg);
      fetch_all();
    }
#pragma unroll 1
    for (int jj = j0; jj < j1; jj += KG) {
      loads_barrier();   // the tiles are there, those before them no longer read
      const int j = jj + kg;
      if (KG > 1 && j >= j1) continue;
      const bool more = j + KG < j1;
      if (more) aim(j + KG);
      if (!SPREAD && more) fetch_all();
      const T* kt = lds + ((j - j0) / KG & 1) * 2 * BN * D;
      const T* vt = kt + BN * D;
      if (j * BN + BN - 1 > p0 || j * BN < lo1) {
        if (SPREAD && more) fetch_all();
#pragma unroll 1
        for (int u = 0; u < BN; u += 32) step(std::true_type{}, [] {}, kt + u * 32, vt + u * 32, j * BN + u);
      } else if constexpr (SPREAD) {
        if (more) fetch(std::integral_constant<int, 0>{});
        step(std::false_type{}, [&] { if (more) fetch(std::integral_constant<int, 1>{}); }, kt, vt, j * BN);
        if (more) fetch(std::integral_constant<int, 2>{});
        step(std::false_type{}, [&] { if (more) fetch(std::integral_constant<int, 3>{}); }, kt + 32 * 32, vt + 32 * 32, j * BN + 32);
      } else {
#pragma unroll
        for (int u = 0; u < BN; u += 32) step(std::false_type{}, [] {}, kt + u * 32, vt + u * 32, j * BN + u);
      }
    }
    bool over = false;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      top[i] = max_q(top[i]) * scale;
      over |= top[i] > mx[i] + kRange;
      if (!F16 && KG > 1 && q == 0) s_top[kg][(w * NQ + i) * 16 + r] = top[i];
    }
    if (F16 || pass == 1 || !__syncthreads_or(over)) break;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
#pragma unroll
      for (int g = 0; g < KG; ++g)
        if (KG > 1) top[i] = fmaxf(top[i], s_top[g][(w * NQ + i) * 16 + r]);
      mx[i] = top[i] > mx[i] + kRange ? top[i] : mx[i];   // (the other rows keep their bits)
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < NQ; ++i) sum[i] = sum_q(sum[i]);
  if constexpr (F16 && KG > 1) {   // one reference for both sets of waves
#pragma unroll
    for (int i = 0; i < NQ; ++i)
      if (q == 0) s_top[kg][(w * NQ + i) * 16 + r] = mx[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const float m = fmaxf(mx[i], s_top[kg ^ 1][(w * NQ + i) * 16 + r]);
      const float f = fast_exp2(mx[i] - m);
      mx[i] = m;
      sum[i] *= f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c] *= f;
    }
  }
  if constexpr (KG > 1) {   // (2: the second set hands its sums over)
    static_assert(KG == 2 && BM * D * 4 <= sizeof(smem), "room for one set of sums");
    f32x4* os = reinterpret_cast<f32x4*>(smem) + w * NQ * NC * 64 + l;
    odd = __syncthreads_or(odd);   // (and nobody reads a tile any more)
    if (kg) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (q == 0) s_sum[1][(w * NQ + i) * 16 + r] = sum[i];
#pragma unroll
        for (int c = 0; c < NC; ++c) os[(i * NC + c) * 64] = o[i][c];
      }
    }
    __syncthreads();
    if (kg) return;
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      sum[i] += s_sum[1][(w * NQ + i) * 16 + r];
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c] += os[(i * NC + c) * 64];
    }
  }

#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const int row = row0 + (w * NQ + i) * 16 + r;
    const float z = sum[i];
    if (row >= rows) continue;
    const int t = over_g(p, row), g = row - t * p.G;
    const int64_t at = (int64_t)(s.c0 + t) * p.Hkv * p.G + h * p.G + g;
    const float f = pos[i] < 0 ? 0.f : 1.f / z;   // (a sum of 0 over keys that are seen is no number)
    T* op = (T*)p.out + at * D;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float x[4] = {o[i][c][0] * f, o[i][c][1] * f, o[i][c][2] * f, o[i][c][3] * f};
      if (odd) {
#pragma unroll 1
        for (int key = j0 * BN; key < j1 * BN; ++key) {
          if (key >= low[i] && key <= pos[i] && (key / BN * BN + BN - 1 > p0 || key / BN * BN < lo1)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = (float)vr(key)[16 * c + 4 * q + e];
              if (!__builtin_isfinite(y)) x[e] += y;
            }
          }
        }
      }
      st4<T>(op + 16 * c + 4 * q, x);
      if (!PAGED && p.low) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] -= (float)(T)x[e];
        st4<T>((T*)p.low + at * D + 16 * c + 4 * q, x);
      }
    }
    if (p.lse && q == 0) p.lse[at] = z == 0.f ? -INFINITY : kLn2 * (mx[i] + __log2f(z));
  }
}

// rows are whole tiles per sequence: at most one more tile each
int64_t tiles_of(const AF& p, int BM) {
  return p.cu ? (int64_t)p.N * p.G / BM + p.B : (int64_t)p.B * (((int64_t)p.T * p.G + BM - 1) / BM);
}

template <class T, int D, bool PAGED> hipError_t run(const AF& p, hipStream_t st) {
  // 32 query rows per wave read each LDS operand for two products; at D = 256
  // their sums leave no room for two waves on a SIMD, and 16 rows are faster.
  // D = 128: four waves, two workgroups on a CU (601 us at 2 x 8192; eight waves
  // around one copy of the keys 666, 64 rows per wave 869, 16 rows 793).  D = 256:
  // eight waves of 16 rows (1006 us for 2 x 4096 over 4096 cached; 32 rows 1687, four
  // waves and tiles of 32 keys 1103).
  constexpr bool f32 = sizeof(T) == 4;
  constexpr int NQ = f32 || D < 256 ? 2 : 1, NW = f32 || D < 256 ? 4 : 8, BN = f32 ? 32 : 64;
  const int64_t tiles = tiles_of(p, 16 * NQ * NW) * p.Hkv;
  // With few tiles of a long walk over the keys the longest walk is what takes the
  // time: tiles of 64 rows, two sets of waves on every other tile of keys.  us, this
  // form / the other, 16 query and 4 key heads: bf16 D = 128 20 / 30 (1024 tokens, 128
  // tiles), 39 / 53 (2048, 256 tiles), 82 / 80 (3104, 388), but 23 / 20 (4 x 512, 256);
  // D = 256 37 / 43, 74 / 81, 160 / 119, 41 / 31; float32 D = 128 179 / 317 (2048), 416 /
  // 475 (3104), 206 / 285 (4 x 1024, 512), 85 / 87 (4 x 512).
  const int64_t walk = std::min<int64_t>(PAGED ? (int64_t)p.max_pages << p.shift : p.T, p.window ? p.window : INT64_MAX);
  if (f32 ? tiles <= 512 : tiles <= 128 || (tiles <= 256 && walk >= 1024)) {
    constexpr int SQ = 1, SW = 4, SG = f32 && D == 256 ? 1 : 2, SN = f32 || D == 256 ? 32 : 64;
    hipLaunchKernelGGL((k_attn<T, D, SQ, SW, SG, SN, PAGED>), dim3((unsigned)(tiles_of(p, 16 * SQ * SW) * p.Hkv)), dim3(64 * SW * SG), 0, st, p);
  } else {
    hipLaunchKernelGGL((k_attn<T, D, NQ, NW, 1, BN, PAGED>), dim3((unsigned)tiles), dim3(64 * NW), 0, st, p);
  }
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
