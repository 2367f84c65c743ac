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
  uint32_t gm; int gs;       // division by G (set_heads)
  int window;                // keys that a query sees, itself the last; 0: all (as for any that no row is longer than)
  int shift, pages, max_pages;
  float sc;                  // scale * log2(e), any sign
  const void *q, *k, *v;
  void* out;                 // dense (tokens, Hkv G, D)
  void* low;                 // NULL or as out: what its rounding cut off
  float* lse;                // NULL or (tokens, Hkv G)
  float* part;               // partial results (dn_attn_few.hip)
  const int32_t *cu, *lens, *pt;
  const int32_t* start;      // contiguous: NULL or the first token of each token's document (B, T)
  int64_t qs[3], ks[3], vs[3];   // batch or page, token, head
  int64_t pts;
  const uint64_t* vis;       // trees: (tokens, words) bits of the new tokens that a new token sees
  int words;
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

// row / G for 0 <= row < 2^31: with 2^k >= G and M = ceil(2^(31+k) / G), row M is
// less than 2^(31+k) / G off, so the shift gives the quotient.  (The compiler's
// division is 30 instructions, and rows are found by it in every tile.)
__device__ __forceinline__ int over_g(const AF& p, int row) {
  return p.gs < 0 ? row : (int)(__umulhi((uint32_t)row, p.gm) >> p.gs);
}
inline void set_heads(AF& p, int Hq, int Hkv) {
  p.Hkv = Hkv;
  p.G = Hq / Hkv;
  int k = 0;
  while ((1 << k) < p.G) ++k;
  p.gs = k - 1;   // G = 1: no division
  p.gm = k ? (uint32_t)((((uint64_t)1 << (31 + k)) + p.G - 1) / p.G) : 0;
}

// What a forward kernel multiplies scores by, positive: it hides a score as -inf
// before it scales it and takes maxima of scores that are not scaled.  The sign of
// a negative scale goes into the queries where they are loaded (exactly), and 0
// becomes the least normal number: -inf stays -inf, and exponents of scores up to
// 2^100 are 0 to 2^-26.
__device__ __forceinline__ float exponent_scale(const AF& p) { return fmaxf(fabsf(p.sc), 0x1p-126f); }

// Rows and tokens are counted in 32 bits, in steps of up to 1024 past the last one.
constexpr int kMostIndex = 0x7fffffff - 1023;

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

// New tokens that cu gives to no sequence, in front of the first and after the last
// (a batch of fixed size that is not full): [0, c0) and [c1, N).  Their results are
// zeros (lse -inf), which all threads of a launch write together.
struct Rest {
  int c0, c1;
  __device__ __forceinline__ Rest(const AF& p) : c0(0), c1(p.N) {
    if (p.cu == nullptr) return;
    c0 = min(max(p.cu[0], 0), p.N);
    c1 = min(max(p.cu[p.B], c0), p.N);
  }
  template <class T, int D> __device__ __forceinline__ void clear(const AF& p) const {
    if (c0 == 0 && c1 == p.N) return;
    constexpr int per = D * sizeof(T) / 16;   // pieces of 16 bytes
    const int64_t Hq = p.Hkv * p.G, n = (c0 + p.N - c1) * Hq * per;
    for (int64_t x = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; x < n; x += (int64_t)gridDim.x * blockDim.x) {
      const int64_t i = x / per, row = i < c0 * Hq ? i : i + (c1 - c0) * Hq;
      *reinterpret_cast<f32x4*>((char*)p.out + (row * per + x % per) * 16) = zero4();
      if (p.lse && x % per == 0) p.lse[row] = -INFINITY;
    }
  }
};

// A sequence of a paged call: its first new token among all, new tokens, tokens in all
// (of trees, those past the page table too).
struct Span { int c0, n, len; };
__device__ __forceinline__ int table_end(const AF& p) { return p.max_pages << p.shift; }
template <bool TREE> __device__ __forceinline__ Span span_of(const AF& p, int b) {
  Span s;
  s.c0 = b * p.T;
  s.n = p.T;
  if (p.cu) {
    s.c0 = min(max(p.cu[b], 0), p.N);
    s.n = min(max(p.cu[b + 1], s.c0), p.N) - s.c0;
  }
  s.len = min(max(p.lens[b], 0), TREE ? kMostIndex : table_end(p));
  return s;
}

// The first key that a query at position pos sees by the window; positions below 0,
// which see none, count as 0, so that no difference leaves 32 bits.
__device__ __forceinline__ int first_key(const AF& p, int pos) { return p.window ? max(max(pos, 0) - p.window + 1, 0) : 0; }

// Whether a row's sums left float32's range, by all four lanes that share it.
template <int NC> __device__ __forceinline__ bool left_range(const f32x4 (&o)[NC]) {
  float x = 0.f;   // (0 times an infinity or a NaN is a NaN)
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) x = __builtin_fmaf(o[c][e], 0.f, x);
  return !(sum_q(x) == 0.f);
}

// Whether keys [key0, key1) have finite values that may have done it, by all threads of
// a workgroup: 2^32 times 2^60 (what an exponential may be) times as many keys as there
// can be stays within it.  (Values that are not finite call for no other reference, and
// the results that they are not part of keep their bits.)
template <int D, class T, bool PAGED> __device__ __forceinline__ bool has_large(const Rows<T, PAGED>& v, int key0, int key1) {
  bool large = false;
  int i = threadIdx.x;
  settle(i);   // (addresses are computed here, not in front of the callers' loops)
#pragma unroll 1
  for (int key = key0 + i / D; key < key1; key += blockDim.x / D) {
    const float y = fabsf((float)v(key)[i % D]);
    large |= y >= 0x1p32f && y < INFINITY;
  }
  return __syncthreads_or(large);
}

// Drafted trees.  A new token sees the keys in front of its sequence's new tokens, the
// window aside, and of those the ones whose bit is set in its words: key `off` is new
// token 0.  Tokens that the page table has no place for are seen by none.
// low: the first key that a window of all that it sees leaves (at least 64
// words of it, so that no new token falls out).
__device__ __forceinline__ const uint64_t* tree_words(const AF& p, int token) { return p.vis + (int64_t)token * p.words; }
__device__ __forceinline__ int tree_count(const AF& p, const uint64_t* w, int off, int n) {
  int c = 0;
  for (int i = 0; i < p.words && 64 * i < n; ++i) {
    uint64_t x = w[i];
    if (n - 64 * i < 64) x &= (1ull << (n - 64 * i)) - 1;
    const int d = -off - 64 * i;   // new tokens at positions below 0 are none
    if (d > 0) x = d < 64 ? x >> d << d : 0;
    c += __popcll(x);
  }
  return c;
}
__device__ __forceinline__ int tree_low(const AF& p, const uint64_t* w, int off, int n) {
  return p.window ? max(off + tree_count(p, w, off, n) - p.window, 0) : 0;
}
__device__ __forceinline__ bool tree_empty(const AF& p, int token, const Span& s) {
  const int off = s.len - s.n, len = min(s.len, table_end(p));
  if (off > 0 && off <= len) return false;   // (a window is wider than its words)
  const uint64_t* w = tree_words(p, token);
  return tree_low(p, w, off, s.n) >= min(off, len) && (len <= off || tree_count(p, w, off, len - off) == 0);
}
// Which of the 32 keys from key0 on it sees.
__device__ __forceinline__ uint32_t tree_bits(const AF& p, const uint64_t* w, int off, int len, int low, int key0) {
  const int rel = key0 - off;
  uint32_t m = ~0u;
  if (rel > -32) {
    uint64_t x = 0;
    if (rel < 0) {
      x = w[0] << -rel | ((1ull << -rel) - 1);
    } else {
      const int i = rel >> 6, s = rel & 63;
      if (i < p.words) x = w[i] >> s;
      if (s > 32 && i + 1 < p.words) x |= w[i + 1] << (64 - s);
    }
    m = (uint32_t)x;
  }
  if (low > key0) m &= low - key0 < 32 ? ~0u << (low - key0) : 0;
  if (len - key0 < 32) m &= len > key0 ? (1u << (len - key0)) - 1 : 0;
  return m;
}

// Keys [lo, hi) that rows [row0, row1) of a sequence see between them, in units.
template <bool TREE = false>
__device__ __forceinline__ void units_of(const AF& p, const Span& s, int row0, int row1, int unit, int& u0, int& u1) {
  const int off = s.len - s.n, p0 = TREE ? off - 1 : off + over_g(p, row0);
  const int p1 = TREE ? min(s.len, table_end(p)) - 1 : off + over_g(p, row1 - 1);
  u0 = first_key(p, p0) / unit;
  u1 = p1 < 0 ? u0 : p1 / unit + 1;
  u1 = max(u1, u0 + 1);   // a tile without keys is work too: it writes zeros
}

// The work of a paged call split evenly over the workgroups.  Its tasks are (b,
// key head, tile of BM rows), in that order, each of as many units as `unit`
// tokens its rows see; workgroup w of W takes the units [w C / W, (w+1) C / W) of
// the C in all, wherever tasks begin and end in them.  Lengths are known on the
// device alone, so every wave adds them up itself, a sequence per lane (the first
// 64 once for all its questions).
struct Task {
  Span s;
  int b, h, m;
  int first;   // its first unit
  int units;
};
__device__ __forceinline__ int scan(int x) {   // inclusive, over a wave
  const int l = lane_id();
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (l >= o) x += y;
  }
  return x;
}
template <bool TREE> struct PlanOf {
  const AF& p;
  int BM, unit;
  Span s0;       // of sequence `lane`
  int mine0, sum0;   // its units over all heads, and with those before it
  int C;         // units of the call
  __device__ __forceinline__ PlanOf(const AF& p_, int BM_, int unit_) : p(p_), BM(BM_), unit(unit_) {
    load(0, s0, mine0);
    sum0 = scan(mine0);
    C = __builtin_amdgcn_readfirstlane(__shfl(sum0, 63));
    for (int b0 = 64; b0 < p.B; b0 += 64) {
      Span s;
      int mine;
      load(b0, s, mine);
      C += __builtin_amdgcn_readfirstlane(__shfl(scan(mine), 63));
    }
  }
  __device__ __forceinline__ void load(int b0, Span& s, int& mine) const {
    const int b = b0 + lane_id();
    s = {0, 0, 0};
    mine = 0;
    if (b >= p.B) return;
    s = span_of<TREE>(p, b);
    const int rows = s.n * p.G;
    if constexpr (TREE) {   // (all its tiles see the same)
      int u0, u1;
      units_of<TREE>(p, s, 0, 1, unit, u0, u1);
      mine = (u1 - u0) * ((rows + BM - 1) / BM) * p.Hkv;
      return;
    }
    for (int r = 0; r < rows; r += BM) {
      int u0, u1;
      units_of<TREE>(p, s, r, min(r + BM, rows), unit, u0, u1);
      mine += u1 - u0;
    }
    mine *= p.Hkv;
  }
  // The sequence whose lane says so in hit(span, units before and with it), its
  // span and the units before it.
  template <class Hit> __device__ __forceinline__ bool find(Hit hit, Task& t, int& per) const {
    Span s = s0;
    int mine = mine0, sum = sum0, before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      if (b0) {
        before += __builtin_amdgcn_readfirstlane(__shfl(sum, 63));
        load(b0, s, mine);
        sum = scan(mine);
      }
      const unsigned long long in = __ballot(mine > 0 && hit(s, before + sum));
      if (in) {
        const int w = __builtin_ctzll(in);
        t.b = b0 + w;
        t.s.c0 = __builtin_amdgcn_readfirstlane(__shfl(s.c0, w));
        t.s.n = __builtin_amdgcn_readfirstlane(__shfl(s.n, w));
        t.s.len = __builtin_amdgcn_readfirstlane(__shfl(s.len, w));
        per = __builtin_amdgcn_readfirstlane(__shfl(mine, w)) / p.Hkv;
        t.first = before + __builtin_amdgcn_readfirstlane(__shfl(sum - mine, w));
        return true;
      }
    }
    return false;
  }
  __device__ __forceinline__ int tile_units(const Task& t, int m) const {
    int u0, u1;
    const int rows = t.s.n * p.G;
    units_of<TREE>(p, t.s, m * BM, min((m + 1) * BM, rows), unit, u0, u1);
    return u1 - u0;
  }
  // the task that holds unit u < C
  __device__ __forceinline__ bool of_unit(int u, Task& t) const {
    int per;
    if (!find([&](const Span&, int sum) { return sum > u; }, t, per)) return false;
    t.h = (u - t.first) / per;
    t.first += t.h * per;
    if constexpr (TREE) {
      t.units = tile_units(t, 0);
      t.m = (u - t.first) / t.units;
      t.first += t.m * t.units;
      return true;
    }
    for (t.m = 0;; ++t.m) {   // (one tile in all but ragged calls)
      t.units = tile_units(t, t.m);
      if (u < t.first + t.units) return true;
      t.first += t.units;
    }
  }
  // task number x of all
  __device__ __forceinline__ bool of_task(int x, Task& t) const {
    static_assert(TREE, "all tiles of a sequence have as many units");
    Span s = s0;
    int mine = mine0, before = 0;
    t.first = 0;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      if (b0) load(b0, s, mine);
      const int tasks = (s.n * p.G + BM - 1) / BM * p.Hkv, ts = scan(tasks), us = scan(mine);
      const unsigned long long in = __ballot(before + ts > x);
      if (in) {
        const int w = __builtin_ctzll(in);
        auto of = [&](int y) { return __builtin_amdgcn_readfirstlane(__shfl(y, w)); };
        t.b = b0 + w;
        t.s = {of(s.c0), of(s.n), of(s.len)};
        const int n = of(tasks), tiles = n / p.Hkv;
        x -= before + of(ts) - n;
        t.units = of(mine) / n;
        t.h = x / tiles;
        t.m = x - t.h * tiles;
        t.first += of(us) - of(mine) + x * t.units;
        return true;
      }
      before += __builtin_amdgcn_readfirstlane(__shfl(ts, 63));
      t.first += __builtin_amdgcn_readfirstlane(__shfl(us, 63));
    }
    return false;
  }
  // the task of new token i's row for query head hq, and the row
  __device__ __forceinline__ bool of_row(int i, int hq, Task& t, int& row) const {
    static_assert(!TREE, "parts of trees are joined by tasks");
    int per;
    if (!find([&](const Span& s, int) { return s.c0 + s.n > i && s.c0 <= i; }, t, per)) return false;
    t.h = over_g(p, hq);
    row = (i - t.s.c0) * p.G + hq - t.h * p.G;
    t.m = row / BM;
    t.first += t.h * per;
    for (int m = 0; m < t.m; ++m) t.first += tile_units(t, m);
    t.units = tile_units(t, t.m);
    return true;
  }
};

using Plan = PlanOf<false>;

// Attention over many rows per sequence (training, prompts): head dimension and
// type checked by the caller.
hipError_t attn_many(const AF& p, int D, int dtype, bool paged, hipStream_t st);

// Attention of few rows over a paged cache, the keys split over the
// workgroups: whether the call is one of these, the bytes it needs, the launches.
bool attn_few_takes(const AF& p, int D, int dtype);
size_t attn_few_bytes(const AF& p, int D);
hipError_t attn_few(const AF& p, int D, int dtype, hipStream_t st);

bool tree_few(const AF& p, int D, int dtype);
hipError_t attn_tree_few(const AF& p, int D, hipStream_t st);

// Drafted trees (p.vis set), of any number of rows and any pages.
size_t attn_tree_bytes(const AF& p, int D, int dtype);
hipError_t attn_tree(const AF& p, int D, int dtype, hipStream_t st);

// The gradient (contiguous rows): p with out, lse and start of the forward, d_out
// dense, the three gradients dense, delta (tokens, Hkv G) floats of scratch.
struct AB {
  AF f;
  float scale;
  const void* d_out;
  void *dq, *dk, *dv;
  float* delta;
  float* part;   // attn_backward_part_bytes
};
size_t attn_backward_part_bytes(const AF& f, int D, int dtype);
hipError_t attn_backward(const AB& p, int D, int dtype, hipStream_t st);

}  // namespace dn
