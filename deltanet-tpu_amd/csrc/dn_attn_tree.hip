// Attention of drafted trees over a paged cache: many rows per key head (new tokens
// times the heads of a group) over long contexts, the keys split over the card.
//
// A tile of query rows stays in a workgroup's registers, keys and values come through
// LDS a tile ahead by direct loads, and a workgroup takes an even share of all
// sequences' keys, wherever tiles of rows begin and end in it; what several hold parts
// of is joined by a second launch.  Only the last keys, the trees' own, are masked.
//
// Up to 64 rows it is bound by reading the keys once: 64 x 4 tokens over 4096 (1.08 GB, D =
// 128) 188 us and 4 for the join, 5.6 TB/s, where a copy of 4 GB reaches 4.8.  Ragged trees
// of up to 64 nodes, 18 on average, over up to 16384 tokens (0.58 GB, some of it read for two
// tiles of 128 rows) 153 to 162 + 14 us, of up to 25 over up to 4096 (D = 256, float16, 0.29
// GB) 73 to 81 + 12.  With more rows the products, the exponentials and the waits between
// them: 64 x 64 over 2000 204 us, 680 TFLOP/s; 16 x 64 over 16384 369 + 15 us, 716 TFLOP/s,
// where the matrix units are busy 39 % of the time, vector instructions are issued 49 %, LDS
// is read 19 % without a conflict, and waves wait 40 % of theirs.  float32 is bound by its
// matrix instruction, busy 70 % (8 x 16 over 8192, 180 us) to 76 % (8 x 64, 619 us).  16 tokens
// over 1000: 13 + 4 us, the chain of lengths, page table, keys, products and the join.
#include <type_traits>

#include "dn_attn_split.h"

namespace dn {
namespace {

// Waits until at most N of this wave's direct loads into LDS are in flight, then for
// everyone's: the tile that was asked for first is there, and nobody reads any more
// the one before it.
template <int N> __device__ __forceinline__ void loads_but() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// (Two sets of waves on every other tile of keys, joined in LDS, for half the parts: 214 us
// in place of 179 for trees of up to 64, 112 of 84 at D = 256.)
//
// NW waves of 16 NQ rows, tiles of BN keys, ST of them in LDS: one that is read, the
// others on their way.  PG: pages of 16 tokens or more, so that the rows of one load
// lie in one page, whose number is read through the scalar cache (a vector load's wait
// would be one for all loads in flight).
template <class T, int D, int NQ, int NW, int BN, int ST, bool PG, int UNITS>
__global__ __launch_bounds__(64 * NW, 2 * ST * BN * D * (int)sizeof(T) <= 80 * 1024 ? 2 : 1) void k_attn_tree(const AF p) {
  using TL = Tile<T, D, BN>;
  using F = typename At<T>::F;
  constexpr bool F16 = std::is_same<T, f16>::value;
  constexpr float kLift = F16 ? 7.f : 0.f, kRange = 60.f;   // (kLift: as in the kernel of few rows)
  constexpr int BM = 16 * NQ * NW, NS = D / 32, NC = D / 16;
  constexpr int kLoads = 2 * (BN / TL::kLoad) * NS / NW;   // of a wave and tile
  __shared__ __align__(16) T lds[ST * 2 * BN * D];   // [ST][K, V][BN][D]
  const int l = lane_id(), r = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  const float scale = exponent_scale(p);
  const Rest rest(p);
  const PlanOf<true> plan(p, BM, BN);
  rest.clear<T, D>(p);
  const int W = shares<UNITS>(gridDim.x, plan.C);
  // neighbours in work on one die: the tiles of rows over the same keys meet in its cache
  const int me = W == (int)gridDim.x && W % 8 == 0 ? (int)blockIdx.x % 8 * (W / 8) + (int)blockIdx.x / 8 : (int)blockIdx.x;
  if (me >= W) return;
  int u = first_unit(me, W, plan.C);
  const int uend = first_unit(me + 1, W, plan.C);
#pragma unroll 1
  while (u < uend) {
    Task t;
    if (!plan.of_unit(u, t)) break;
    const int rows = t.s.n * p.G, row0 = t.m * BM;
    // off: keys that every row sees, but for the window; the new tokens are behind them, if
    // the page table has a place for any
    const int first = t.s.len - t.s.n, len = min(t.s.len, table_end(p)), off = min(first, len), last = max(len - 1, 0);
    int k0, k1;
    units_of<true>(p, t.s, 0, 1, BN, k0, k1);
    const int skip = u - t.first, take = min(t.units - skip, uend - u);
    const int j0 = k0 + skip, j1 = j0 + take;
    const int lo1 = p.window ? max(first + min(t.s.n, 64 * p.words) - p.window, 0) : 0;   // no row's first key is later

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
      low[i] = tree_low(p, tree_words(p, token[i]), first, t.s.n);
    }
    Rows<T, true> vr;   // (for the values that are not finite)
    vr.base = (const T*)p.v + t.h * p.vs[2];
    vr.token = p.vs[1]; vr.page = p.vs[0]; vr.pt = p.pt + t.b * p.pts; vr.shift = p.shift; vr.pages = p.pages; vr.last = last;
    const T* kb = (const T*)p.k + t.h * p.ks[2];
    const auto pt = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)vr.pt;
    // where this lane reads of tile j
    constexpr int groups = BN / TL::kLoad;
    const T *ks = nullptr, *vs = nullptr;
    T* to = nullptr;
    auto aim = [&](int j) {
      const int row = j * BN + w % groups * TL::kLoad + l / TL::kPieces;
      int at = min(row, last), pg;
      if constexpr (PG) {
        const int first = min(__builtin_amdgcn_readfirstlane(row), last);
        pg = pt[first >> p.shift];
        at = min(at, first | ((1 << p.shift) - 1));
      } else {
        pg = vr.pt[at >> p.shift];
      }
      pg = min(max(pg, 0), p.pages - 1);
      const int in = at & ((1 << p.shift) - 1), x = TL::piece(w % groups * TL::kLoad + l / TL::kPieces, l % TL::kPieces) * TL::kPer;
      ks = kb + pg * p.ks[0] + in * p.ks[1] + x;
      vs = vr.base + pg * p.vs[0] + in * p.vs[1] + x;
      to = lds + (j - j0) % ST * 2 * BN * D;
    };
    // Tiles of 64 keys at D = 256 are asked for in four parts between the products of the
    // one before, as in the kernel of whole rows; others at once.
    constexpr bool SPREAD = D == 256 && BN == 64;
    auto fetch = [&](auto part) {
      constexpr int P = decltype(part)::value;
      if constexpr (P < 2) TL::template load_part<NW, P, 2>(to, w, ks);
      else TL::template load_part<NW, P - 2, 2>(to + BN * D, w, vs);
    };
    auto fetch_all = [&] {
      TL::template load_part<NW, 0, 1>(to, w, ks);
      TL::template load_part<NW, 0, 1>(to + BN * D, w, vs);
    };
    f32x4 o[NQ][NC];
    float mx[NQ], top[NQ], sum[NQ];
    bool late = false;   // scores of the tiles between were beyond the reference of their time
#pragma unroll
    for (int i = 0; i < NQ; ++i) mx[i] = -INFINITY;
    bool odd = false;
    auto rescale = [&](int i, float m) {
      const float f = m == -INFINITY ? 1.f : fast_exp2(mx[i] - m);
      mx[i] = m;
      sum[i] *= f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c] *= f;
    };
    // 32 keys.  Probabilities are relative to mx, the maximum of a piece's first tile
    // and of its masked ones (LEARN, kept up to 2^kLazy); the tiles between only note what
    // their largest scores were.  A row that went more than 2^kRange beyond the mx that it
    // was summed by is found before a masked tile raises that, or at the piece's end, and the
    // piece done again from the largest score that is known then, which nothing raises any
    // more: sums are as exact with any reference up to 2^kRange below.  A row whose products
    // with the values left the range all the same (values from 2^68 on) goes that way too.
    // float16 has no such range, its rows are raised on the way.  (The tile that begins with the last of the
    // windows' first keys is the first of which that row sees any: it is LEARN too.)
    auto hides = [&](int key0) { return key0 + 32 > off || key0 < lo1; };   // some row must not see some of 32 keys
    auto learns = [&](int j) { return j == j0 || (j + 1) * BN > off || j * BN <= lo1; };
    constexpr bool AHEAD = D == 256 && sizeof(T) == 2;
    constexpr int VB = AHEAD ? 4 : 1, NB = NC / VB;
    auto in_order = [] {
      if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
    };
    auto step = [&](auto learn, auto between, const T* kt, const T* vt, int key0) {
      constexpr bool LEARN = decltype(learn)::value;
      const bool masked = LEARN && hides(key0);
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
      if constexpr (AHEAD) {
        in_order();
        values(0);
        in_order();
      }
      bool grow = false;
      float mt[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (LEARN && masked) {
          const uint32_t bits = tree_bits(p, tree_words(p, token[i]), off, len, low[i], key0) >> (4 * q);
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[i][e][x] = bits >> (16 * e + x) & 1 ? sc[i][e][x] : -INFINITY;
        }
        const float m = fmaxf(fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3])),
                              fmaxf(fmaxf(sc[i][1][0], sc[i][1][1]), fmaxf(sc[i][1][2], sc[i][1][3])));
        if constexpr (LEARN) {
          mt[i] = max_q(m) * scale - kLift;
          grow |= mt[i] > mx[i] + kLazy;
        } else {
          top[i] = fmaxf(top[i], m);
          if (F16) grow |= __builtin_fmaf(m, scale, -mx[i]) > kLift + kLazy;
        }
      }
      if constexpr (LEARN || F16) {
        if (__any(grow)) {
#pragma unroll
          for (int i = 0; i < NQ; ++i) {
            if (!F16) late |= __any(max_q(top[i]) * scale > mx[i] + kRange);
            rescale(i, fmaxf(mx[i], LEARN ? mt[i] : max_q(top[i]) * scale - kLift));
          }
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
      between();
      const bool bad = LEARN && masked && TL::odd32(vt);
      if (LEARN) odd |= bad;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if (!AHEAD || n + 1 < NB) values(AHEAD ? n + 1 : n);
        in_order();
        if (LEARN && bad) {
#pragma unroll
          for (int c = 0; c < VB; ++c) vf[n & 1][c] = finite8<T>(vf[n & 1][c]);
        }
#pragma unroll
        for (int c = 0; c < VB; ++c)
#pragma unroll
          for (int i = 0; i < NQ; ++i) At<T>::mma(o[i][n * VB + c], vf[n & 1][c], pf[i]);
      }
    };
    // the waits for the queries land here and not, for all loads in flight, in the loop
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int c = 0; c < NS; ++c) settle(qf[i][c]);
#pragma unroll 1
    for (int pass = 0;; ++pass) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        top[i] = -INFINITY;
        sum[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[i][c] = zero4();
      }
#pragma unroll
      for (int i = 0; i + 1 < ST; ++i)
        if (j0 + i < j1) {
          aim(j0 + i);
          fetch_all();
        }
#pragma unroll 1
      for (int j = j0; j < j1; ++j) {
        if (ST > 2 && j + ST - 2 < j1) loads_but<(ST - 2) * kLoads>();
        else loads_but<0>();
        const bool more = j + ST - 1 < j1;
        if (more) aim(j + ST - 1);
        const T* kt = lds + (j - j0) % ST * 2 * BN * D;
        const T* vt = kt + BN * D;
        if (learns(j)) {
          if (more) fetch_all();
#pragma unroll 1
          for (int x = 0; x < BN; x += 32) step(std::true_type{}, [] {}, kt + x * 32, vt + x * 32, j * BN + x);
        } else if constexpr (SPREAD) {
          if (more) fetch(std::integral_constant<int, 0>{});
          step(std::false_type{}, [&] { if (more) fetch(std::integral_constant<int, 1>{}); }, kt, vt, j * BN);
          if (more) fetch(std::integral_constant<int, 2>{});
          step(std::false_type{}, [&] { if (more) fetch(std::integral_constant<int, 3>{}); }, kt + 32 * 32, vt + 32 * 32, j * BN + 32);
        } else {
          if (more) fetch_all();
#pragma unroll
          for (int x = 0; x < BN; x += 32) step(std::false_type{}, [] {}, kt + x * 32, vt + x * 32, j * BN + x);
        }
      }
      if (F16 || pass == 1) break;
      bool over = late, out = false;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        top[i] = max_q(top[i]) * scale;
        over |= top[i] > mx[i] + kRange;
        out |= left_range(o[i]);
      }
      if (__builtin_expect(!__syncthreads_or(over || out), 1)) break;
      // (values that are not finite: once more as it was, to the same bits)
      const bool raise = __syncthreads_or(over) || has_large<D>(vr, j0 * BN, min(j1 * BN, len));
#pragma unroll
      for (int i = 0; i < NQ; ++i) mx[i] = raise ? fmaxf(top[i], mx[i]) : -INFINITY;
    }
    if (odd) {   // infinities and NaNs that some row must not see: to those that do
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll 1
          for (int key = j0 * BN; key < min(j1 * BN, len); ++key) {
            if (!hides(key & ~31) || !(tree_bits(p, tree_words(p, token[i]), off, len, low[i], key & ~31) >> (key & 31) & 1)) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float y = (float)vr(key)[16 * c + 4 * q + e];
              if (!__builtin_isfinite(y)) o[i][c][e] += y;
            }
          }
        }
    }
    const bool whole = take == t.units;
    float* slot = p.part + (2 * (int64_t)me + (skip == 0 ? 1 : 0)) * slot_floats<D, BM>();
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
template <class T, int D, int NQ, int NW, int BN, int ST> struct FormOf {
  static constexpr int BM = 16 * NQ * NW, kUnits = 64 / BN;
  static constexpr int kPerCU = NW == 4 && 2 * ST * BN * D * (int)sizeof(T) <= 80 * 1024 ? 2 : 1;
  static int64_t groups(const AF& p) {
    return std::min<int64_t>(256 * kPerCU, most_tasks(p, BM) * ((((int64_t)p.max_pages << p.shift) + BN - 1) / BN));
  }
  static size_t bytes(const AF& p) { return (size_t)groups(p) * 2 * BM * (D + 2) * sizeof(float); }
  static hipError_t run(const AF& p, hipStream_t st) {
    const unsigned W = (unsigned)groups(p);
    if (p.shift >= 4) hipLaunchKernelGGL((k_attn_tree<T, D, NQ, NW, BN, ST, true, kUnits>), dim3(W), dim3(64 * NW), 0, st, p);
    else hipLaunchKernelGGL((k_attn_tree<T, D, NQ, NW, BN, ST, false, kUnits>), dim3(W), dim3(64 * NW), 0, st, p);
    launch_tree_join<T, D, BM, BN, kUnits>(p, W, most_tasks(p, BM), st);
    return hipGetLastError();
  }
};
// The form, by the mean number of rows of a sequence and key head; us with the join,
// bf16, of 64 / 128 / 256 rows a tile (at D = 256: 64 / 128), sequences x new tokens over
// cached tokens, 4 query heads a key head:
// - D = 128: 64 x 4 / 4096 193, 208, 370; 32 x 8 / 4096 108, 127, 187; 8 x 16 / 8192 65, 70,
//   104; 16 x 21 / 8192 (64 and 16384 at most) 173, 166, 243; 8 x 64 / 8192 143, 105, 112;
//   64 x 64 / 2000 408, 270, 203;
// - D = 64: 64 x 4 / 4096 112, 125, 212; 8 x 32 / 8192 58, 48, 66; 64 x 64 / 2000 211, 158, 132;
// - D = 256: 64 x 4 / 4096 196, 222; 16 x 21 / 8192 170, 182; 8 x 64 / 8192 131, 116; 64 x 64
//   / 2000 280, 262; 1 x 16 / 1000, where the card has less to do than it holds, 18, 16.5;
// - float32: D = 128 8 x 16 / 8192 180, 310; 8 x 64 / 8192 619, 621; D = 256 213, 314 and 741,
//   598.
template <class T, int D, class G> auto by_rows(const AF& p, G g) {
  const int64_t rows = (int64_t)p.N * p.G, B = p.B;
  if constexpr (sizeof(T) == 4) {
    if (rows <= 128 * B) return g(FormOf<T, D, 1, 4, 32, 2>{});
    return g(FormOf<T, D, 1, 8, 32, 2>{});
  } else if constexpr (D == 256) {
    const int64_t units = most_tasks(p, 64) * ((((int64_t)p.max_pages << p.shift) + 63) / 64);
    if (rows <= 96 * B && units > 512) return g(FormOf<T, D, 1, 4, 32, 2>{});
    return g(FormOf<T, D, 1, 8, 64, 2>{});
  } else {
    if (rows <= 64 * B) return g(FormOf<T, D, 1, 4, 32, D == 64 ? 3 : 2>{});
    if (rows < 192 * B) return g(FormOf<T, D, 2, 4, 64, 2>{});
    return g(FormOf<T, D, 2, 8, 64, 2>{});
  }
}
template <class G> auto by_form(const AF& p, int D, int dtype, G g) {
  auto go = [&](auto z) {
    using T = decltype(z);
    return D == 64 ? by_rows<T, 64>(p, g) : D == 128 ? by_rows<T, 128>(p, g) : by_rows<T, 256>(p, g);
  };
  return dtype == DN_BF16 ? go((bf16)0.f) : dtype == DN_F16 ? go((f16)0.f) : go(0.f);
}

}  // namespace

size_t attn_tree_bytes(const AF& p, int D, int dtype) {
  if (tree_few(p, D, dtype)) return attn_few_bytes(p, D);
  return by_form(p, D, dtype, [&](auto f) { return decltype(f)::bytes(p); });
}

hipError_t attn_tree(const AF& p, int D, int dtype, hipStream_t st) {
  if (tree_few(p, D, dtype)) return attn_tree_few(p, D, st);
  return by_form(p, D, dtype, [&](auto f) { return decltype(f)::run(p, st); });
}

}  // namespace dn
