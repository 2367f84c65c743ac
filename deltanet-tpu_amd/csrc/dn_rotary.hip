// Rotary positions, and the store of rotated keys and of values in a paged cache.
//
// Both are streams: each element is read once and written once, and a token's
// row of the angle table (4 R bytes) is shared by its heads.  A thread owns 16
// channels of a token, as two groups of 8 that are each other's partners in the
// rotation (half layout: 8 channels and the 8 at distance R/2; interleaved: 16
// neighbours), loads the 8 cosines and 8 sines once and walks over heads with
// them: 16-byte loads and stores in 16-bit types, no exchange between lanes.
// 84 MB each way of queries and keys (168 MB moved) turn in 28 to 35 us, 79 MB of
// prompts are rotated and stored in 18 us (4.3 TB/s); a token of 64 sequences takes
// 4 us, most of it the launch and the chain of lengths, page table and store.
#include "dn_common.h"
#include "dn_host.h"

namespace dn {

namespace {

template <class T> __device__ __forceinline__ void ld8(const T* p, float* o) {
  typedef T V __attribute__((ext_vector_type(8)));
  const V a = *reinterpret_cast<const V*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
}
template <class T, bool PAST = false> __device__ __forceinline__ void st8(T* p, const float* v) {
  typedef T V __attribute__((ext_vector_type(8)));
  V a;
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
  if constexpr (PAST) __builtin_nontemporal_store(a, reinterpret_cast<V*>(p));
  else *reinterpret_cast<V*>(p) = a;
}

// The 16 channels of item `it` of a head row: groups of 8 starting at a and b.
// Items below R/16 are rotated, the others copied.
struct Item {
  int a, b, row;   // row: offset of the cosines in the table's row, -1 for a copy
};
__device__ __forceinline__ Item item_of(int it, int R, bool inter) {
  const int nr = R >> 4;
  if (it >= nr) return {R + (it - nr) * 16, R + (it - nr) * 16 + 8, -1};
  if (inter) return {it * 16, it * 16 + 8, it * 8};
  return {it * 8, (R >> 1) + it * 8, it * 8};
}

// (x, y) -> (x c - y s, y c + x s) for the 8 pairs of an item
__device__ __forceinline__ void turn8(float* x, float* y, const float* c, const float* s, bool inter) {
  if (inter) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1], d = y[2 * i], e = y[2 * i + 1];
      x[2 * i] = a * c[i] - b * s[i];
      x[2 * i + 1] = b * c[i] + a * s[i];
      y[2 * i] = d * c[4 + i] - e * s[4 + i];
      y[2 * i + 1] = e * c[4 + i] + d * s[4 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = x[i], b = y[i];
      x[i] = a * c[i] - b * s[i];
      y[i] = b * c[i] + a * s[i];
    }
  }
}

__device__ __forceinline__ void angles8(const float* table, int64_t pos, int rows, int R, int at, float sign, float* c, float* s) {
  if (pos < 0 || pos >= rows) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
    return;
  }
  const float* r = table + pos * R + at;
  ld8<float>(r, c);
  ld8<float>(r + (R >> 1), s);
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] *= sign;
}

struct RP {
  int B, L, Hq, H, D, R, rows, inter, pos64;
  float sign;
  const void *q, *k, *pos;
  void *qo, *ko;
  const float* table;
  int64_t qs[3], ks[3], ps[2];
};

__device__ __forceinline__ int64_t pos_of(const RP& p, int b, int l) {
  const int64_t i = b * p.ps[0] + l * p.ps[1];
  return p.pos64 ? ((const int64_t*)p.pos)[i] : (int64_t)((const int32_t*)p.pos)[i];
}

template <class T> __device__ __forceinline__ const T* src_row(const RP& p, int b, int l, int h) {
  return h < p.Hq ? (const T*)p.q + b * p.qs[0] + l * p.qs[1] + h * p.qs[2]
                  : (const T*)p.k + b * p.ks[0] + l * p.ks[1] + (h - p.Hq) * p.ks[2];
}
template <class T> __device__ __forceinline__ T* dst_row(const RP& p, int64_t t, int h) {
  return h < p.Hq ? (T*)p.qo + (t * p.Hq + h) * p.D : (T*)p.ko + (t * (p.H - p.Hq) + h - p.Hq) * p.D;
}

// x: (token, item), y: NH heads.  PAST: stores go past the caches.
template <class T, int NH, bool PAST>
__global__ __launch_bounds__(256) void k_rotary(const RP p) {
  const int per = p.D >> 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = id / per;
  if (t >= (int64_t)p.B * p.L) return;
  const int b = (int)(t / p.L), l = (int)(t % p.L);
  const Item it = item_of((int)(id % per), p.R, p.inter);
  const int h0 = blockIdx.y * NH;
  float x[NH][8], y[NH][8];
#pragma unroll
  for (int h = 0; h < NH; ++h)
    if (h0 + h < p.H) {
      const T* s = src_row<T>(p, b, l, h0 + h);
      ld8<T>(s + it.a, x[h]);
      ld8<T>(s + it.b, y[h]);
    }
  float c[8], s[8];
  if (it.row >= 0) angles8(p.table, pos_of(p, b, l), p.rows, p.R, it.row, p.sign, c, s);
#pragma unroll
  for (int h = 0; h < NH; ++h)
    if (h0 + h < p.H) {
      if (it.row >= 0) turn8(x[h], y[h], c, s, p.inter);
      T* d = dst_row<T>(p, t, h0 + h);
      st8<T, PAST>(d + it.a, x[h]);
      st8<T, PAST>(d + it.b, y[h]);
    }
}

// One pair, or one channel that is not rotated, per thread: any sizes and strides.
__device__ __forceinline__ void pair_of(int i, int R, bool inter, int& a, int& b) {
  const int half = R >> 1;
  if (i >= half) { a = R + (i - half); b = -1; }
  else if (inter) { a = 2 * i; b = a + 1; }
  else { a = i; b = i + half; }
}

template <class T>
__global__ __launch_bounds__(256) void k_rotary_any(const RP p) {
  const int per = p.D - (p.R >> 1);
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = id / per;
  if (t >= (int64_t)p.B * p.L) return;
  const int b = (int)(t / p.L), l = (int)(t % p.L), i = (int)(id % per);
  int ca, cb;
  pair_of(i, p.R, p.inter, ca, cb);
  float c = 0.f, s = 0.f;
  if (cb >= 0) {
    const int64_t pos = pos_of(p, b, l);
    const bool in = pos >= 0 && pos < p.rows;
    c = in ? p.table[pos * p.R + i] : __builtin_nanf("");
    s = in ? p.sign * p.table[pos * p.R + (p.R >> 1) + i] : __builtin_nanf("");
  }
  const int h = blockIdx.y;
  const T* sp = src_row<T>(p, b, l, h);
  T* dp = dst_row<T>(p, t, h);
  if (cb < 0) {
    dp[ca] = sp[ca];
  } else {
    const float x = (float)sp[ca], y = (float)sp[cb];
    dp[ca] = (T)(x * c - y * s);
    dp[cb] = (T)(y * c + x * s);
  }
}

// ---------------------------------------------------------------------------
// paged cache
// ---------------------------------------------------------------------------
struct AP {
  int N, B, H, D, R, rows, inter, pages, shift, max_pages;
  const void *k, *v;
  void *kc, *vc;
  const int32_t *pt, *lens, *cu;
  const float* table;
  int64_t ks[3], vs[3], kcs[3], vcs[3], pts;
};

// Where new token i is read (element offsets) and stored; false: nowhere.
struct Slot {
  int64_t pos, k_src, v_src, k_dst, v_dst;
};
__device__ __forceinline__ bool slot_of(const AP& p, int i, Slot& o) {
  int b, n, j;   // sequence, its new tokens, place among them
  if (p.cu == nullptr) {
    n = p.N / p.B;
    b = i / n;
    j = i - b * n;
    o.k_src = b * p.ks[0] + j * p.ks[1];
    o.v_src = b * p.vs[0] + j * p.vs[1];
  } else {
    int lo = 0, hi = p.B;   // the last b with cu[b] <= i
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (p.cu[m] <= i) lo = m;
      else hi = m;
    }
    b = lo;
    const int c0 = p.cu[b], c1 = p.cu[b + 1];
    if (i < c0 || i >= c1) return false;
    n = c1 - c0;
    j = i - c0;
    o.k_src = i * p.ks[1];
    o.v_src = i * p.vs[1];
  }
  o.pos = (int64_t)p.lens[b] - n + j;
  const int64_t pg = o.pos >> p.shift;
  if (o.pos < 0 || pg >= p.max_pages) return false;
  const int page = p.pt[b * p.pts + pg];
  if (page < 0 || page >= p.pages) return false;
  const int64_t in = o.pos & ((1 << p.shift) - 1);
  o.k_dst = page * p.kcs[0] + in * p.kcs[1];
  o.v_dst = page * p.vcs[0] + in * p.vcs[1];
  return true;
}

// x: (token, item), y: NH of the 2 H rows (keys, then values)
template <class T, class TC, int NH>
__global__ __launch_bounds__(256) void k_append(const AP p) {
  const int per = p.D >> 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = id / per;
  if (t >= p.N) return;
  const Item it = item_of((int)(id % per), p.R, p.inter);
  const int h0 = blockIdx.y * NH;
  Slot o;
  if (!slot_of(p, (int)t, o)) return;
  float x[NH][8], y[NH][8];
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const int h = h0 + i;
    if (h < 2 * p.H) {
      const T* s = h < p.H ? (const T*)p.k + o.k_src + h * p.ks[2] : (const T*)p.v + o.v_src + (h - p.H) * p.vs[2];
      ld8<T>(s + it.a, x[i]);
      ld8<T>(s + it.b, y[i]);
    }
  }
  float c[8], s[8];
  const bool rot = it.row >= 0 && h0 < p.H;
  if (rot) angles8(p.table, o.pos, p.rows, p.R, it.row, 1.f, c, s);
#pragma unroll
  for (int i = 0; i < NH; ++i) {
    const int h = h0 + i;
    if (h < 2 * p.H) {
      if (rot && h < p.H) turn8(x[i], y[i], c, s, p.inter);
      TC* d = h < p.H ? (TC*)p.kc + o.k_dst + h * p.kcs[2] : (TC*)p.vc + o.v_dst + (h - p.H) * p.vcs[2];
      st8<TC>(d + it.a, x[i]);
      st8<TC>(d + it.b, y[i]);
    }
  }
}

template <class T, class TC>
__global__ __launch_bounds__(256) void k_append_any(const AP p) {
  const int per = p.D - (p.R >> 1);
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = id / per;
  if (t >= p.N) return;
  const int i = (int)(id % per), h = blockIdx.y;
  Slot o;
  if (!slot_of(p, (int)t, o)) return;
  int ca, cb;
  pair_of(i, p.R, p.inter, ca, cb);
  const bool key = h < p.H;
  const T* sp = key ? (const T*)p.k + o.k_src + h * p.ks[2] : (const T*)p.v + o.v_src + (h - p.H) * p.vs[2];
  TC* dp = key ? (TC*)p.kc + o.k_dst + h * p.kcs[2] : (TC*)p.vc + o.v_dst + (h - p.H) * p.vcs[2];
  if (cb < 0 || !key) {
    dp[ca] = (TC)(float)sp[ca];
    if (cb >= 0) dp[cb] = (TC)(float)sp[cb];
    return;
  }
  const bool in = o.pos < p.rows;
  const float c = in ? p.table[o.pos * p.R + i] : __builtin_nanf(""), s = in ? p.table[o.pos * p.R + (p.R >> 1) + i] : __builtin_nanf("");
  const float x = (float)sp[ca], y = (float)sp[cb];
  dp[ca] = (TC)(x * c - y * s);
  dp[cb] = (TC)(y * c + x * s);
}

bool float_type(int dt) { return dt == DN_F32 || dt == DN_BF16 || dt == DN_F16; }
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
// rows that start on 16 bytes whatever their index
bool wide(const void* p, const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] % 8) return false;
  return aligned(p);
}

// Threads of one head each that fill the card a few times over.  From there on (2^24
// elements) a thread takes several heads and reads its angles once for them: four in
// the append; two in the rotation, which stores past the caches, for its result does
// not fit the L2s (8 x 4 MB) and is not in them when it is read next: 84 MB of queries
// and keys take 32.5 us (5.2 TB/s) in place of 44.
constexpr int64_t kManyThreads = 1 << 20;

template <class F> void by_type(int dt, F f) {
  if (dt == DN_BF16) f((bf16)0.f);
  else if (dt == DN_F16) f((f16)0.f);
  else f(0.f);
}

int rot_error(const char* m) { return set_error(DN_E_INVALID, m); }

}  // namespace
}  // namespace dn

using namespace dn;

extern "C" int dn_rotary(const dn_rotary_args* a, void* stream) {
  if (a == nullptr) return rot_error("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_rotary_args built for another ABI version");
  if (a->B < 0 || a->L < 0 || a->Hq < 0 || a->Hk < 0 || a->Hq > 32768 || a->Hk > 32767 || a->D <= 0)
    return rot_error("bad rotary sizes");
  if (a->R <= 0 || a->R % 2 || a->R > a->D) return rot_error("rotary channels must be even, positive and at most D");
  if (!float_type(a->dtype) || (a->pos_dtype != DN_I32 && a->pos_dtype != DN_I64)) return rot_error("rotary dtype not supported");
  const int H = a->Hq + a->Hk;
  const int64_t N = (int64_t)a->B * a->L;
  if (N == 0 || H == 0) return DN_OK;
  if ((a->Hq && (!a->q || !a->q_out)) || (a->Hk && (!a->k || !a->k_out)) || !a->pos || !a->table || a->rows <= 0)
    return rot_error("missing tensor pointer");
  RP p{};
  p.B = a->B; p.L = a->L; p.Hq = a->Hq; p.H = H; p.D = a->D; p.R = a->R; p.rows = a->rows;
  p.inter = a->interleaved != 0; p.pos64 = a->pos_dtype == DN_I64; p.sign = a->inverse ? -1.f : 1.f;
  p.q = a->q; p.k = a->k; p.pos = a->pos; p.qo = a->q_out; p.ko = a->k_out; p.table = a->table;
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_strides[i]; p.ks[i] = a->k_strides[i]; }
  p.ps[0] = a->pos_strides[0]; p.ps[1] = a->pos_strides[1];
  const bool fast = a->D % 16 == 0 && a->R % 16 == 0 && aligned(a->table) && (!a->Hq || (wide(a->q, a->q_strides, 3) && aligned(a->q_out))) &&
                    (!a->Hk || (wide(a->k, a->k_strides, 3) && aligned(a->k_out)));
  const int64_t n = N * (fast ? a->D / 16 : a->D - a->R / 2), blocks = (n + 255) / 256;
  if (blocks > 0x7fffffff) return rot_error("too many tokens");
  hipStream_t st = (hipStream_t)stream;
  by_type(a->dtype, [&](auto z) {
    using T = decltype(z);
    if (!fast) hipLaunchKernelGGL((k_rotary_any<T>), dim3((unsigned)blocks, H), dim3(256), 0, st, p);
    else if (n * H < kManyThreads) hipLaunchKernelGGL((k_rotary<T, 1, false>), dim3((unsigned)blocks, H), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_rotary<T, 2, true>), dim3((unsigned)blocks, (H + 1) / 2), dim3(256), 0, st, p);
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}

extern "C" int dn_kv_append(const dn_kv_append_args* a, void* stream) {
  if (a == nullptr) return rot_error("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_kv_append_args built for another ABI version");
  if (a->N < 0 || a->B < 0 || a->H < 0 || a->H > 32767 || a->D <= 0) return rot_error("bad append sizes");
  if (a->R < 0 || a->R % 2 || a->R > a->D) return rot_error("rotary channels must be even and at most D");
  if (!float_type(a->dtype) || !float_type(a->cache_dtype)) return rot_error("append dtype not supported");
  if (a->pages <= 0 || a->max_pages <= 0 || a->page_size <= 0 || (a->page_size & (a->page_size - 1)))
    return rot_error("the cache needs pages of a power of two tokens");
  if (a->N == 0 || a->B == 0 || a->H == 0) return DN_OK;
  if (a->cu_seqlens == nullptr && a->N % a->B) return rot_error("without cu_seqlens every sequence has N / B new tokens");
  if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->page_table || !a->seq_lens || (a->R && (!a->table || a->rows <= 0)))
    return rot_error("missing tensor pointer");
  AP p{};
  p.N = a->N; p.B = a->B; p.H = a->H; p.D = a->D; p.R = a->R; p.rows = a->rows; p.inter = a->interleaved != 0;
  p.pages = a->pages; p.max_pages = a->max_pages;
  while ((1 << p.shift) < a->page_size) ++p.shift;
  p.k = a->k; p.v = a->v; p.kc = a->k_cache; p.vc = a->v_cache;
  p.pt = a->page_table; p.lens = a->seq_lens; p.cu = a->cu_seqlens; p.table = a->table; p.pts = a->page_table_stride;
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = a->k_strides[i]; p.vs[i] = a->v_strides[i];
    p.kcs[i] = a->kc_strides[i]; p.vcs[i] = a->vc_strides[i];
  }
  const bool fast = a->D % 16 == 0 && a->R % 16 == 0 && (!a->R || aligned(a->table)) && wide(a->k, a->k_strides, 3) &&
                    wide(a->v, a->v_strides, 3) && wide(a->k_cache, a->kc_strides, 3) && wide(a->v_cache, a->vc_strides, 3);
  const int64_t n = (int64_t)a->N * (fast ? a->D / 16 : a->D - a->R / 2), blocks = (n + 255) / 256;
  if (blocks > 0x7fffffff) return rot_error("too many tokens");
  hipStream_t st = (hipStream_t)stream;
  const int H2 = 2 * a->H;
  by_type(a->dtype, [&](auto z) {
    by_type(a->cache_dtype, [&](auto zc) {
      using T = decltype(z);
      using TC = decltype(zc);
      if (!fast) hipLaunchKernelGGL((k_append_any<T, TC>), dim3((unsigned)blocks, H2), dim3(256), 0, st, p);
      else if (n * H2 < kManyThreads || a->H % 4) hipLaunchKernelGGL((k_append<T, TC, 1>), dim3((unsigned)blocks, H2), dim3(256), 0, st, p);
      else hipLaunchKernelGGL((k_append<T, TC, 4>), dim3((unsigned)blocks, H2 / 4), dim3(256), 0, st, p);
    });
  });
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}
