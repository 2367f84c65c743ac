// Attention of few query rows over a paged cache: single tokens, drafts and chunks
// of a few sequences over a long one.
//
// Bound by reading the keys and values once.  A workgroup takes an even share of
// all sequences' keys (Task), its four waves 32 keys each of a unit of 128, with
// no barrier between units: a wave loads the keys straight into the operand
// layout and the values into registers one unit ahead, puts the values into LDS
// of its own to read them transposed, and keeps its own running maximum and sums.
// The waves' results are joined in LDS; a task that several workgroups hold parts
// of is joined by a second launch, in the order of its keys.
//
// 64 sequences of up to 16384 tokens (2.2 GB of keys and values, D = 128): 409 + 9 us,
// 5.4 TB/s, where a copy reaches 5.2; 32 drafts of up to 5 tokens (283 MB, D = 256):
// 62 to 70 + 6 us; one token over 1000: 10 + 5 us, the chain of lengths, page table,
// keys, products and the join.
#include <type_traits>

#include "dn_attn_split.h"

namespace dn {
namespace {

constexpr int kWaves = 4, kUnit = 32 * kWaves;
constexpr int kGroups = 512;   // workgroups of a launch: two per CU

// TREE: which of its sequence's new tokens a row sees stands in its words (tree_bits);
// the keys in front of them are those of every row.
template <class T, int D, int NQ, bool TREE>
__global__ __launch_bounds__(64 * kWaves) void k_attn_few(const AF p) {
  using TL = Tile<T, D, 32>;
  using F = typename At<T>::F;
  typedef uint32_t U4 __attribute__((ext_vector_type(4)));
  // float16: a running maximum's probability is 2^7 to 2^15, not 1 to 2^8, so that
  // those far below it keep their bits (half a step is 2^-25)
  constexpr float kLift = std::is_same<T, f16>::value ? 7.f : 0.f;
  constexpr int BM = 16 * NQ, NS = D / 32, NC = D / 16, NG = 32 / TL::kLoad, NV = NG * NS;   // NV: loads of a wave's 32 value rows, NG groups of rows by slabs
  // values of a wave's 32 keys; at a task's end the waves' sums
  constexpr int kV = 32 * D * (int)sizeof(T), kO = BM * D * 4;
  __shared__ __align__(16) char smem[kWaves * (kV > kO ? kV : kO)];
  __shared__ float wm[kWaves][BM], wl[kWaves][BM];
  const int l = lane_id(), r = l & 15, q = l >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  T* vt = reinterpret_cast<T*>(smem + w * kV);

  const float scale = exponent_scale(p);
  const Rest rest(p);
  const PlanOf<TREE> plan(p, BM, kUnit);
  rest.clear<T, D>(p);
  const int W = min((int)gridDim.x, plan.C);   // each has a unit at least
  if ((int)blockIdx.x >= W) return;
  int u = first_unit(blockIdx.x, W, plan.C);
  const int uend = first_unit(blockIdx.x + 1, W, plan.C);
#pragma unroll 1
  while (u < uend) {
    Task t;
    if (!plan.of_unit(u, t)) break;
    const int rows = t.s.n * p.G, row0 = t.m * BM, row1 = min(row0 + BM, rows);
    // the keys that all rows see end with p0, those that any sees with p1
    const int first = t.s.len - t.s.n, len = TREE ? min(t.s.len, table_end(p)) : t.s.len, off = TREE ? min(first, len) : first;
    const int p0 = TREE ? off - 1 : off + over_g(p, row0), p1 = TREE ? len - 1 : off + over_g(p, row1 - 1);
    int k0, k1;
    units_of<TREE>(p, t.s, row0, row1, kUnit, k0, k1);
    const int skip = u - t.first, take = min(t.units - skip, uend - u);
    const int j0 = k0 + skip, j1 = j0 + take;   // units of this piece
    const int last = max(p1, 0);
    const int lo1 = first_key(p, TREE ? t.s.len - 1 : p1);   // (none later, of any row)

    F qf[NQ][NS];
    int pos[NQ], low[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int row = min(row0 + i * 16 + r, rows - 1);
      const int tk = over_g(p, row), g = row - tk * p.G;
      const T* qp = (const T*)p.q + (p.cu ? (int64_t)(t.s.c0 + tk) * p.qs[1] : t.b * p.qs[0] + tk * p.qs[1]) + (t.h * p.G + g) * p.qs[2];
#pragma unroll
      for (int c = 0; c < NS; ++c) qf[i][c] = *reinterpret_cast<const F*>(qp + 32 * c + 8 * q);
      if (p.sc < 0.f)
#pragma unroll
        for (int c = 0; c < NS; ++c) qf[i][c] = minus8<T>(qf[i][c]);
      pos[i] = TREE ? t.s.c0 + tk : off + tk;   // trees: the token, whose words say what it sees
      low[i] = TREE ? tree_low(p, tree_words(p, pos[i]), first, t.s.n) : first_key(p, pos[i]);
    }
    auto bits_of = [&](int i, int key0) { return tree_bits(p, tree_words(p, pos[i]), off, len, low[i], key0); };

#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int c = 0; c < NS; ++c) settle(qf[i][c]);
    f32x4 o[NQ][NC];
    float mx[NQ], sum[NQ];
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      mx[i] = -INFINITY;
      sum[i] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[i][c] = zero4();
    }

    const int32_t* pt = p.pt + t.b * p.pts;
    const T* kb = (const T*)p.k + t.h * p.ks[2];
    const T* vb = (const T*)p.v + t.h * p.vs[2];
    // the page of 16 keys from `key` on (a page holds 16 keys or more)
    auto page_of = [&](int key) { return __builtin_amdgcn_readfirstlane(min(max(pt[min(key, last) >> p.shift], 0), p.pages - 1)); };
    F kf[2][NS];
    U4 vr[NV];
    int pg0 = page_of(j0 * kUnit + 32 * w), pg1 = page_of(j0 * kUnit + 32 * w + 16);
    auto fetch = [&](int j) {
      const int key = j * kUnit + 32 * w, mask = (1 << p.shift) - 1;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int a = key + 16 * e, base = min(a, last & ~15);   // 16 keys, none past the last
        const int rel = min(r, last - base);
        const T* s = kb + (e ? pg1 : pg0) * p.ks[0] + (int64_t)((base & mask) + rel) * p.ks[1];
#pragma unroll
        for (int c = 0; c < NS; ++c) kf[e][c] = *reinterpret_cast<const F*>(s + 32 * c + 8 * q);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int row = g * TL::kLoad + l / TL::kPieces, e = g >= NG / 2;
        const int a = key + 16 * e, base = min(a, last & ~15), rel = min(row & 15, last - base);
        const T* s = vb + (e ? pg1 : pg0) * p.vs[0] + (int64_t)((base & mask) + rel) * p.vs[1] + l % TL::kPieces * TL::kPer;
#pragma unroll
        for (int c = 0; c < NS; ++c) vr[g * NS + c] = *reinterpret_cast<const U4*>(s + 32 * c);
      }
    };
    fetch(j0);
    pg0 = page_of((j0 + 1) * kUnit + 32 * w);
    pg1 = page_of((j0 + 1) * kUnit + 32 * w + 16);
    bool odd = false;
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
      const int key0 = j * kUnit + 32 * w;
      f32x4 sc[NQ][2];
#pragma unroll
      for (int i = 0; i < NQ; ++i) sc[i][0] = sc[i][1] = zero4();
#pragma unroll
      for (int c = 0; c < NS; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < NQ; ++i) At<T>::mma(sc[i][e], kf[e][c], qf[i][c]);
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int c = 0; c < NS; ++c)
          *reinterpret_cast<U4*>(vt + c * TL::kSlab + TL::at(g * TL::kLoad + l / TL::kPieces, l % TL::kPieces)) = vr[g * NS + c];
      if (j + 1 < j1) {
        fetch(j + 1);
        pg0 = page_of((j + 2) * kUnit + 32 * w);
        pg1 = page_of((j + 2) * kUnit + 32 * w + 16);
      }
      const bool masked = key0 + 31 > p0 || key0 < lo1;
      F pf[NQ];
      float mt[NQ];
      bool grow = false;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        if (masked) {
          const uint32_t bits = TREE ? bits_of(i, key0) >> (4 * q) : 0;
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int key = key0 + 16 * e + 4 * q + x;
              const bool sees = TREE ? bits >> (16 * e + x) & 1 : key <= pos[i] && key >= low[i];
              sc[i][e][x] = sees ? sc[i][e][x] : -INFINITY;
            }
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
      const bool bad = masked && TL::odd32(vt);
      odd |= bad;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        F vf = TL::col8(vt, c, r, q);
        if (bad) vf = finite8<T>(vf);
#pragma unroll
        for (int i = 0; i < NQ; ++i) At<T>::mma(o[i][c], vf, pf[i]);
      }
    }
    if (odd) {   // infinities and NaNs that some row of the piece must not see: to those that do
      Rows<T, true> rv;
      rv.base = vb; rv.token = p.vs[1]; rv.page = p.vs[0]; rv.pt = pt; rv.shift = p.shift; rv.pages = p.pages; rv.last = last;
#pragma unroll
      for (int i = 0; i < NQ; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll 1
          for (int j = j0; j < j1; ++j) {
            const int key0 = j * kUnit + 32 * w;
            if (!(key0 + 31 > p0 || key0 < lo1)) continue;
#pragma unroll 1
            for (int key = max(key0, low[i]); key <= min(key0 + 31, TREE ? p1 : pos[i]); ++key)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (TREE && !(bits_of(i, key0) >> (key - key0) & 1)) continue;
                const float y = (float)rv(key)[16 * c + 4 * q + e];
                if (!__builtin_isfinite(y)) o[i][c][e] += y;
              }
          }
        }
    }

    // join the waves: row r of tile i, channels 16 c + 4 q ..
    __syncthreads();   // the values have been read
    float* os = reinterpret_cast<float*>(smem);   // [wave][BM][D], the row's 16-byte pieces rotated by the row
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const float z = sum_q(sum[i]);
      if (q == 0) {
        wm[w][16 * i + r] = mx[i];
        wl[w][16 * i + r] = z;
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
        *reinterpret_cast<f32x4*>(os + (w * BM + 16 * i + r) * D + (((4 * c + q) + r) % (D / 4)) * 4) = o[i][c];
    }
    __syncthreads();
    const bool whole = take == t.units;
    float* slot = p.part + (2 * (int64_t)blockIdx.x + (skip == 0 ? 1 : 0)) * slot_floats<D, BM>();
    for (int x = threadIdx.x; x < (row1 - row0) * (D / 4); x += 64 * kWaves) {
      const int row = x / (D / 4), ch = x % (D / 4);
      float m = wm[0][row];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) m = fmaxf(m, wm[k][row]);
      f32x4 a = zero4();
      float z = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float f = wm[k][row] == -INFINITY ? 0.f : fast_exp2(wm[k][row] - m);
        const f32x4 y = *reinterpret_cast<const f32x4*>(os + (k * BM + row) * D + ((ch + (row & 15)) % (D / 4)) * 4);
        if (f != 0.f) a += f * y;
        z += f * wl[k][row];
      }
      if (whole) {
        const int tk = over_g(p, row0 + row), g = row0 + row - tk * p.G;
        const int64_t at = (int64_t)(t.s.c0 + tk) * p.Hkv * p.G + t.h * p.G + g;
        const bool none = TREE ? tree_empty(p, t.s.c0 + tk, t.s) : off + tk < 0;
        const float f = none ? 0.f : 1.f / z;   // (a sum of 0 over keys that are seen is no number)
        const float y[4] = {a[0] * f, a[1] * f, a[2] * f, a[3] * f};
        st4<T>((T*)p.out + at * D + 4 * ch, y);
        if (p.lse && ch == 0) p.lse[at] = z == 0.f ? -INFINITY : kLn2 * (m + __log2f(z));
      } else {
        *reinterpret_cast<f32x4*>(slot + row * D + 4 * ch) = a;
        if (ch == 0) {
          slot[BM * D + row] = m;
          slot[BM * D + BM + row] = z;
        }
      }
    }
    __syncthreads();   // the next piece writes its values there
    u += take;
  }
}

// Joins the parts of a query row if more than one workgroup had some: D/4 threads
// per part, 1024/D parts at a time.
template <class T, int D, int BM>
__global__ __launch_bounds__(256) void k_attn_join(const AF p, int groups) {
  constexpr int NP = 1024 / D;
  __shared__ float ps[NP][D + 4];
  Task t;
  int row;
  const int Hq = p.Hkv * p.G, i = blockIdx.x / Hq, hq = blockIdx.x - i * Hq;
  const Plan plan(p, BM, kUnit);
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
  const float f = t.s.len - t.s.n + i - t.s.c0 < 0 ? 0.f : 1.f / z;   // (as above)
  const float y[4] = {a[0] * f, a[1] * f, a[2] * f, a[3] * f};
  st4<T>((T*)p.out + (int64_t)blockIdx.x * D + 4 * ch, y);
  if (p.lse && ch == 0) p.lse[blockIdx.x] = z == 0.f ? -INFINITY : kLn2 * (m + __log2f(z));
}

int row_tile(const AF& p) { return (int64_t)p.N * p.G <= (int64_t)16 * p.B ? 16 : 32; }
int64_t most_tasks(const AF& p) {
  const int BM = row_tile(p);
  return (p.cu ? (int64_t)p.N * p.G / BM + p.B : (int64_t)p.B * ((p.T * p.G + BM - 1) / BM)) * p.Hkv;
}
// No more workgroups than there can be units.
int64_t most_units(const AF& p) { return most_tasks(p) * ((((int64_t)p.max_pages << p.shift) + kUnit - 1) / kUnit); }
int64_t groups_of(const AF& p) { return std::min<int64_t>(kGroups, most_units(p)); }

template <class T, int D> hipError_t run(const AF& p, hipStream_t st) {
  const unsigned W = (unsigned)groups_of(p), rows = (unsigned)p.N * p.Hkv * p.G;
  if (row_tile(p) == 16) {
    hipLaunchKernelGGL((k_attn_few<T, D, 1, false>), dim3(W), dim3(64 * kWaves), 0, st, p);
    if (W > 1) hipLaunchKernelGGL((k_attn_join<T, D, 16>), dim3(rows), dim3(256), 0, st, p, (int)W);
  } else {
    hipLaunchKernelGGL((k_attn_few<T, D, 2, false>), dim3(W), dim3(64 * kWaves), 0, st, p);
    if (W > 1) hipLaunchKernelGGL((k_attn_join<T, D, 32>), dim3(rows), dim3(256), 0, st, p, (int)W);
  }
  return hipGetLastError();
}

// trees in float32 (tree_few)
template <int D, int NQ> hipError_t run_tree(const AF& p, hipStream_t st) {
  const unsigned W = (unsigned)groups_of(p);
  hipLaunchKernelGGL((k_attn_few<float, D, NQ, true>), dim3(W), dim3(64 * kWaves), 0, st, p);
  launch_tree_join<float, D, 16 * NQ, kUnit, 1>(p, W, most_tasks(p), st);
  return hipGetLastError();
}

}  // namespace

// This kernel reads the keys once per 16 or 32 rows and spreads them over the card
// at the cost of a join; that of many rows reads them once per 64 or 128 rows, by
// one workgroup.  It is the length of that one walk (the page table's width, or the
// window) against the tiles of rows that share the card here which decides.  us, this
// kernel / the other, tokens cached, 8 key heads at D = 128 and 4 at D = 256:
// - tiles of 16 rows, one token, 16 bits: 1 sequence 17 / 13 (512), 17 / 17 (1024),
//   18 / 50 (4096); 64 sequences 53 / 45 (1024), 109 / 110 (2048), 196 / 209 (4096),
//   and less than half of it when lengths differ;
// - tiles of 32, 16 bits: D = 128 16 tiles 19 / 30 (2048), 64 38 / 30 (2048), 56 / 98
//   (8192), 128 95 / 101 (8192), 146 / 191 (16384), 256 183 / 112 (8192), 333 / 282
//   (16384); D = 256 64 tiles 65 / 55 (2048), 119 / 194 (8192), 128 242 / 194 (8192);
// - float32, whose products take the time: D = 128 128 tiles 60 / 46 (512), 94 / 159
//   (2048), 512 804 / 615 (8192), but with up to 32 rows of a sequence, which fill half
//   of the other's tile, 440 / 641 (512 tiles, 4096); D = 256 64 tiles 73 / 91 (512),
//   818 / 1376 (8192), 128 1545 / 1366 (8192).
// Pages of 16 tokens at least: 16 keys of a wave's 32 lie in one page.
bool attn_few_takes(const AF& p, int D, int dtype) {
  if (p.shift < 4 || most_units(p) >= (1 << 30)) return false;
  const int64_t walk = std::min<int64_t>((int64_t)p.max_pages << p.shift, p.window ? p.window : INT64_MAX);
  const int64_t tiles = most_tasks(p);
  if (dtype == DN_F32) {
    if (walk < 256) return false;
    if (row_tile(p) == 16 || (D < 256 && (int64_t)p.N * p.G <= (int64_t)32 * p.B)) return true;
    return tiles <= (D == 256 ? 64 : 256) && walk >= 8 * tiles;
  }
  if (row_tile(p) == 16) return walk >= (tiles <= 128 ? 1024 : 4096);
  return tiles <= (D == 256 ? 64 : 128) && walk >= std::max<int64_t>(1024, 64 * tiles);
}

// Drafted trees in float32 whose rows fill 16 or 32 of a tile: the products take the
// time there, and the kernel of trees makes 64 rows of them (us, this kernel / that one,
// D = 128: 64 x 4 tokens over 4096 372 / 627, 32 x 8 261 / 326; D = 64 206 / 333, 153 / 176;
// D = 256 423 / 746).  At D = 256 there are no registers for 32 rows (815 / 390).  In 16 bits
// that kernel is the faster one (D = 128 64 x 4 207 / 193, 32 x 8 129 / 108).
bool tree_few(const AF& p, int D, int dtype) {
  return dtype == DN_F32 && p.shift >= 4 && (int64_t)p.N * p.G <= (int64_t)(D == 256 ? 16 : 32) * p.B;
}

size_t attn_few_bytes(const AF& p, int D) { return (size_t)groups_of(p) * 2 * row_tile(p) * (D + 2) * sizeof(float); }

hipError_t attn_few(const AF& p, int D, int dtype, hipStream_t st) {
  auto go = [&](auto z) {
    using T = decltype(z);
    return D == 64 ? run<T, 64>(p, st) : D == 128 ? run<T, 128>(p, st) : run<T, 256>(p, st);
  };
  return dtype == DN_BF16 ? go((bf16)0.f) : dtype == DN_F16 ? go((f16)0.f) : go(0.f);
}

hipError_t attn_tree_few(const AF& p, int D, hipStream_t st) {
  if (D == 256) return run_tree<256, 1>(p, st);
  if (row_tile(p) == 16) return D == 64 ? run_tree<64, 1>(p, st) : run_tree<128, 1>(p, st);
  return D == 64 ? run_tree<64, 2>(p, st) : run_tree<128, 2>(p, st);
}

}  // namespace dn
