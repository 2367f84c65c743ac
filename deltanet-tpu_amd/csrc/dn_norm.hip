// Norms of queries and keys for each head, with the rotation by the token's position
// in the same pass; the same with the store into a paged cache; and the gradient.
//
// Of a head x with D channels: r = 1 / sqrt(mean(x^2) + eps), y = x r (offset + w),
// z = rotation(y).  For dz: g = rotation^T(dz), h = g (offset + w),
// dx = r (h - x r^2 mean(h x)), dw = sum of g x r over tokens and heads.
//
// Streams: every head is read once and written once.  A thread owns two groups of 16
// bytes of a head that are each other's partners in the rotation of halves (and hold
// whole pairs of the interleaved one), and its neighbours the groups beside them, so
// that every load and store of a wave is of whole lines; D / 16 (float32: D / 8) lanes
// exchange a head's sums in registers.  The angles and the weights are read once for
// the heads of a thread.
// Measured on inputs that no cache holds: queries and keys of 2 x 4096 tokens (168 MB in
// and out) 44 us, their gradients (252 MB) 58.5 + 4.5 us; prompts of 9040 tokens stored
// (227 MB) 50 us, 4.5 TB/s; a token of 64 sequences 4.7 us, launch and chain of loads.
// Other sizes and alignments take a wave a head, bound by its own chain: 8192 tokens, 32 + 8
// heads of 80 (105 MB) 191 us, of 128 off 16 bytes (168 MB) 201, their gradients 580 and 674;
// 2048 tokens, heads of 640 (210 MB) 138 and 705.
#include <type_traits>

#include "dn_attn.h"
#include "dn_host.h"

namespace dn {

namespace {

struct HP {
  int N, L, H[3], D, R, rows, inter, pos64, wdt, cdt, pages, shift;   // H: query, key and value heads
  float eps, offset;
  const void* x[3];          // q, k, v
  const void* w[2];          // NULL: no norm
  void* out[3];              // q', and k' or the caches
  const void* pos;
  const int64_t* slots;
  const float* table;
  int64_t xs[3][3], cs[2][3], ps[2];   // batch, token, head; page, token, head
};

// what the gradient has besides: dz in, dx out, partial sums of dw
struct GP {
  const void* dz[2];
  void* dx[2];               // NULL: not wanted
  float* part;               // (blocks, D), those of q in front
  int64_t zs[2][3];
};

// x summed over groups of P neighbouring lanes, the same bits in each of them
template <int CTRL> __device__ __forceinline__ float moved(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int P> __device__ __forceinline__ float sum_lanes(float x) {
  if constexpr (P >= 2) x += moved<0xB1>(x);    // lanes 1 apart
  if constexpr (P >= 4) x += moved<0x4E>(x);    // 2 apart
  if constexpr (P >= 8) x += moved<0x141>(x);   // mirrored in 8
  if constexpr (P >= 16) x += moved<0x140>(x);  // mirrored in 16
  if constexpr (P >= 32) {
    float a, b;
    both<16>(x, a, b);
    x = a + b;
  }
  if constexpr (P >= 64) {
    float a, b;
    both<32>(x, a, b);
    x = a + b;
  }
  return x;
}

// 1 / sqrt(a): the instruction's result (one step off at most) and a Newton step.
__device__ __forceinline__ float rsqrt32(float a) {
  const float y = __builtin_amdgcn_rsqf(a);
  const float z = __builtin_fmaf(y * 0.5f, __builtin_fmaf(-a * y, y, 1.f), y);
  return __builtin_isfinite(z) ? z : y;   // (0 and infinity)
}

// A head whose mean square (with eps) a is below 2^-96, where squares vanish (channels
// below 2^-48, eps as good as 0), or past the largest number (channels from 2^59 on) is
// taken times a power of two by which they are all well inside, and eps times its square:
// x r is the same.
constexpr float kUp = 0x1p100f, kDown = 0x1p-70f;
__device__ __forceinline__ bool far_off(float a) { return a < 0x1p-96f || a == INFINITY; }
__device__ __forceinline__ float scale_of(float a) { return a < 1.f ? kUp : kDown; }

__device__ __forceinline__ int64_t pos_of(const HP& p, int b, int l) {
  const int64_t i = b * p.ps[0] + l * p.ps[1];
  return p.pos64 ? ((const int64_t*)p.pos)[i] : (int64_t)((const int32_t*)p.pos)[i];
}

template <class T> constexpr int kWidth = 16 / (int)sizeof(T);   // channels of a group
// W values of a type, in floats
template <int W, bool PAST = false, class T> __device__ __forceinline__ void load(const T* p, float* o) {
  typedef T V __attribute__((ext_vector_type(W)));
  V a;
  if constexpr (PAST) a = __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
  else a = *reinterpret_cast<const V*>(p);
#pragma unroll
  for (int i = 0; i < W; ++i) o[i] = (float)a[i];
}
template <int W, bool PAST, class T> __device__ __forceinline__ void store(T* p, const float* v) {
  typedef T V __attribute__((ext_vector_type(W)));
  V a;
#pragma unroll
  for (int i = 0; i < W; ++i) a[i] = (T)v[i];
  if constexpr (PAST) __builtin_nontemporal_store(a, reinterpret_cast<V*>(p));
  else *reinterpret_cast<V*>(p) = a;
}

// The two groups of lane `it` of a head; those of the first R channels are rotated.
struct Item { int a, b; bool turn; };
template <int W> __device__ __forceinline__ Item item_of(int it, int D, int R) {
  const int nr = R / (2 * W);
  if (it < nr) return {it * W, (R >> 1) + it * W, true};
  return {R + (it - nr) * W, R + ((D - R) >> 1) + (it - nr) * W, false};
}
// Cosines and sines of its pairs: one set for the halves, W / 2 for each group of
// interleaved ones.  A position outside the table: NaN.
template <int W> __device__ __forceinline__ void angles(const float* table, int64_t pos, int rows, int R, const Item& it, bool inter, float sign, float* c, float* s) {
  if (pos < 0 || pos >= rows) {
#pragma unroll
    for (int i = 0; i < W; ++i) c[i] = s[i] = __builtin_nanf("");
    return;
  }
  const float* r = table + pos * R;
  if (inter) {
    load<W / 2>(r + it.a / 2, c);
    load<W / 2>(r + it.b / 2, c + W / 2);
    load<W / 2>(r + (R + it.a) / 2, s);
    load<W / 2>(r + (R + it.b) / 2, s + W / 2);
  } else {
    load<W>(r + it.a, c);
    load<W>(r + (R >> 1) + it.a, s);
  }
#pragma unroll
  for (int i = 0; i < W; ++i) s[i] *= sign;
}
// (x, y) -> (x c - y s, y c + x s) for its pairs
template <int W> __device__ __forceinline__ void turn(float* x, float* y, const float* c, const float* s, bool inter) {
  if (inter) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1], d = y[2 * i], e = y[2 * i + 1];
      x[2 * i] = a * c[i] - b * s[i];
      x[2 * i + 1] = b * c[i] + a * s[i];
      y[2 * i] = d * c[W / 2 + i] - e * s[W / 2 + i];
      y[2 * i + 1] = e * c[W / 2 + i] + d * s[W / 2 + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float a = x[i], b = y[i];
      x[i] = a * c[i] - b * s[i];
      y[i] = b * c[i] + a * s[i];
    }
  }
}
// One pair, or one channel that is not rotated: any sizes.
__device__ __forceinline__ void pair_of(int i, int R, bool inter, int& a, int& b) {
  const int half = R >> 1;
  if (i >= half) { a = R + (i - half); b = -1; }
  else if (inter) { a = 2 * i; b = a + 1; }
  else { a = i; b = i + half; }
}

// weights of any type, plus the offset
template <int W> __device__ __forceinline__ void weights(const void* w, int dt, int at, float offset, float* o) {
  if (dt == DT_F32) load<W>((const float*)w + at, o);
  else if (dt == DT_BF16) load<W>((const bf16*)w + at, o);
  else load<W>((const f16*)w + at, o);
#pragma unroll
  for (int i = 0; i < W; ++i) o[i] += offset;
}

template <int W, bool PAST> __device__ __forceinline__ void put(void* p, int dt, int64_t at, const float* v) {
  if (dt == DT_F32) store<W, PAST>((float*)p + at, v);
  else if (dt == DT_BF16) store<W, PAST>((bf16*)p + at, v);
  else store<W, PAST>((f16*)p + at, v);
}
__device__ __forceinline__ void put1(void* p, int dt, int64_t at, float v) {
  if (dt == DT_F32) ((float*)p)[at] = v;
  else if (dt == DT_BF16) ((bf16*)p)[at] = (bf16)v;
  else ((f16*)p)[at] = (f16)v;
}

// Where the heads of a token go.  Serving: a token at a negative position is none,
// its queries are zeros; a slot outside the cache is not stored.
template <class T> constexpr int type_of() { return sizeof(T) == 4 ? DT_F32 : __is_same(T, bf16) ? DT_BF16 : DT_F16; }
struct Dst {
  int64_t at, head;   // element offset of the first head, and from one to the next
  int dt;
  bool store, none;
};
template <class T, bool PAGED> __device__ __forceinline__ Dst dst_of(const HP& p, int side, int64_t t, int64_t pos) {
  Dst d;
  d.dt = type_of<T>();
  d.store = true;
  d.none = false;
  d.at = t * p.H[side] * p.D;
  d.head = p.D;
  if constexpr (PAGED) {
    d.none = pos < 0;
    if (side) {
      const int64_t slot = p.slots[t];
      const int64_t page = slot >> p.shift, in = slot & ((1 << p.shift) - 1);
      d.store = !d.none && slot >= 0 && page < p.pages;
      d.dt = p.cdt;
      d.head = p.cs[side - 1][2];
      d.at = page * p.cs[side - 1][0] + in * p.cs[side - 1][1];
    }
  }
  return d;
}

template <int NH> __host__ __device__ __forceinline__ int chunks_of(const HP& p) {
  return (p.H[0] + NH - 1) / NH + (p.H[1] + NH - 1) / NH + (p.H[2] + NH - 1) / NH;
}

// Blocks: chunks of NH heads of q, k or v innermost, so that a token's heads are read
// and written at about the same time, then (token, item) in groups of P threads.
template <class T, int P, int NH, bool PAGED, bool PAST>
__global__ __launch_bounds__(256) void k_heads(const HP p) {
  constexpr int W = kWidth<T>;
  const uint32_t nc = chunks_of<NH>(p);
  const int64_t id = (int64_t)(blockIdx.x / nc) * 256 + threadIdx.x;
  const int i = threadIdx.x % P;
  const bool live = id / P < p.N && i < p.D / (2 * W);
  const int64_t t = min(id / P, (int64_t)p.N - 1);
  int y = blockIdx.x % nc, side = 0;
  for (; side < 2; ++side) {
    const int n = (p.H[side] + NH - 1) / NH;
    if (y < n) break;
    y -= n;
  }
  const int h0 = y * NH, H = p.H[side], b = (int)(t / p.L), l = (int)(t % p.L);
  const Item it = item_of<W>(i, p.D, p.R);
  const T* s = (const T*)p.x[side] + b * p.xs[side][0] + l * p.xs[side][1] + h0 * p.xs[side][2];
  float u[NH][W], v[NH][W];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    if (live && h0 + h < H) {
      load<W, PAGED && PAST>(s + h * p.xs[side][2] + it.a, u[h]);
      load<W, PAGED && PAST>(s + h * p.xs[side][2] + it.b, v[h]);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) u[h][e] = v[h][e] = 0.f;
    }
  }
  const int64_t pos = PAGED || p.R ? pos_of(p, b, l) : 0;
  float c[W], sn[W], wa[W], wb[W];
  const bool turns = side < 2 && live && it.turn, norm = side < 2 && p.w[0];
  if (turns) angles<W>(p.table, pos, p.rows, p.R, it, p.inter, 1.f, c, sn);
  if (norm && live) {
    weights<W>(p.w[side], p.wdt, it.a, p.offset, wa);
    weights<W>(p.w[side], p.wdt, it.b, p.offset, wb);
  }
  const Dst d = dst_of<T, PAGED>(p, side, t, pos);
  const float over = 1.f / p.D;
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    if (norm) {
      float z = 0.f;
#pragma unroll
      for (int e = 0; e < W; ++e) z += u[h][e] * u[h][e] + v[h][e] * v[h][e];
      const float a = sum_lanes<P>(z) * over + p.eps;
      float r = rsqrt32(a);
      if (__builtin_expect(far_off(a), 0)) {
        const float s = scale_of(a);
        z = 0.f;
#pragma unroll
        for (int e = 0; e < W; ++e) z += (u[h][e] * s) * (u[h][e] * s) + (v[h][e] * s) * (v[h][e] * s);
        const float rs = rsqrt32(sum_lanes<P>(z) * over + p.eps * s * s);
        // the factor that keeps small channels' bits first
        const float first = s > 1.f ? s : rs;
        r = s > 1.f ? rs : s;
#pragma unroll
        for (int e = 0; e < W; ++e) u[h][e] *= first, v[h][e] *= first;
      }
#pragma unroll
      for (int e = 0; e < W; ++e) {
        u[h][e] = u[h][e] * r * wa[e];
        v[h][e] = v[h][e] * r * wb[e];
      }
    }
    if (!live || h0 + h >= H) continue;
    if (turns) turn<W>(u[h], v[h], c, sn, p.inter);
    if (PAGED && side == 0 && d.none) {
#pragma unroll
      for (int e = 0; e < W; ++e) u[h][e] = v[h][e] = 0.f;
    }
    if (!d.store) continue;
    const int64_t at = d.at + (h0 + h) * d.head;
    put<W, PAST>(p.out[side], d.dt, at + it.a, u[h]);
    put<W, PAST>(p.out[side], d.dt, at + it.b, v[h]);
  }
}

// A wave per head at a time: any sizes, strides and alignment.
template <class T, bool PAGED>
__global__ __launch_bounds__(256) void k_heads_any(const HP p) {
  const int H = p.H[0] + p.H[1] + p.H[2];
#pragma unroll 1
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < (int64_t)p.N * H; row += (int64_t)gridDim.x * 4) {
    const int64_t t = row / H;
    int h = (int)(row % H), side = 0;
    for (; side < 2 && h >= p.H[side]; ++side) h -= p.H[side];
    const int b = (int)(t / p.L), l = (int)(t % p.L);
    const T* s = (const T*)p.x[side] + b * p.xs[side][0] + l * p.xs[side][1] + h * p.xs[side][2];
    const int64_t pos = PAGED || p.R ? pos_of(p, b, l) : 0;
    const Dst d = dst_of<T, PAGED>(p, side, t, pos);
    const int64_t at = d.at + h * d.head;
    const bool norm = side < 2 && p.w[0];
    float r = 1.f, first = 1.f;
    if (norm) {
      float by = 1.f;
      auto mean = [&] {
        float z = 0.f;
        for (int c = lane_id(); c < p.D; c += 64) z += ((float)s[c] * by) * ((float)s[c] * by);
        return sum_lanes<64>(z) * (1.f / p.D) + p.eps * by * by;
      };
      const float a = mean();
      r = rsqrt32(a);
      if (far_off(a)) {
        by = scale_of(a);
        const float rs = rsqrt32(mean());
        first = by > 1.f ? by : rs;
        r = by > 1.f ? rs : by;
      }
    }
    if (!d.store) continue;
    const bool zero = PAGED && side == 0 && d.none;
    auto value = [&](int c) {
      const float x = (float)s[c];
      return norm ? x * first * r * (p.offset + ld_f(p.w[side], c, p.wdt)) : x;
    };
    for (int i = lane_id(); i < p.D - (p.R >> 1); i += 64) {
      int ca, cb;
      pair_of(i, p.R, p.inter, ca, cb);
      float x = value(ca), y = cb >= 0 ? value(cb) : 0.f;
      if (cb >= 0 && side < 2) {
        const bool in = pos >= 0 && pos < p.rows;
        const float c = in ? p.table[pos * p.R + i] : __builtin_nanf(""), sn = in ? p.table[pos * p.R + (p.R >> 1) + i] : __builtin_nanf("");
        const float a = x, e = y;
        x = a * c - e * sn;
        y = e * c + a * sn;
      }
      put1(p.out[side], d.dt, at + ca, zero ? 0.f : x);
      if (cb >= 0) put1(p.out[side], d.dt, at + cb, zero ? 0.f : y);
    }
  }
}

// The gradient.  Groups of P threads walk over tokens; y: NH heads of q or k.
template <class T, int P, int NH>
__global__ __launch_bounds__(256) void k_heads_grad(const HP p, const GP g) {
  constexpr int W = kWidth<T>;
  __shared__ float sums[256 / P][P * 2 * W];
  const int i = threadIdx.x % P;
  const bool own = i < p.D / (2 * W);
  int y = blockIdx.y, side = 0;
  const int nq = (p.H[0] + NH - 1) / NH;
  if (y >= nq) {
    side = 1;
    y -= nq;
  }
  const int h0 = y * NH, H = p.H[side];
  const Item it = item_of<W>(i, p.D, p.R);
  float wa[W], wb[W], da[W], db[W];
#pragma unroll
  for (int e = 0; e < W; ++e) wa[e] = wb[e] = da[e] = db[e] = 0.f;
  if (own) {
    weights<W>(p.w[side], p.wdt, it.a, p.offset, wa);
    weights<W>(p.w[side], p.wdt, it.b, p.offset, wb);
  }
  const float over = 1.f / p.D;
#pragma unroll 1
  for (int64_t t = (int64_t)blockIdx.x * (256 / P) + threadIdx.x / P; t < p.N; t += (int64_t)gridDim.x * (256 / P)) {
    const int b = (int)(t / p.L), l = (int)(t % p.L);
    const T* s = (const T*)p.x[side] + b * p.xs[side][0] + l * p.xs[side][1] + h0 * p.xs[side][2];
    const T* z = (const T*)g.dz[side] + b * g.zs[side][0] + l * g.zs[side][1] + h0 * g.zs[side][2];
    float u[NH][W], v[NH][W], gu[NH][W], gv[NH][W];
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      if (own && h0 + h < H) {
        load<W>(s + h * p.xs[side][2] + it.a, u[h]);
        load<W>(s + h * p.xs[side][2] + it.b, v[h]);
        load<W>(z + h * g.zs[side][2] + it.a, gu[h]);
        load<W>(z + h * g.zs[side][2] + it.b, gv[h]);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e) u[h][e] = v[h][e] = gu[h][e] = gv[h][e] = 0.f;
      }
    }
    float c[W], sn[W];
    const bool turns = own && it.turn;
    if (turns) angles<W>(p.table, pos_of(p, b, l), p.rows, p.R, it, p.inter, -1.f, c, sn);
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      if (turns) turn<W>(gu[h], gv[h], c, sn, p.inter);
      float xx = 0.f, hx = 0.f;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        xx += u[h][e] * u[h][e] + v[h][e] * v[h][e];
        hx += gu[h][e] * wa[e] * u[h][e] + gv[h][e] * wb[e] * v[h][e];
      }
      const float a = sum_lanes<P>(xx) * over + p.eps;
      float r = rsqrt32(a), by = 1.f;
      if (__builtin_expect(far_off(a), 0)) {   // x r, and with it dw, is as it was; dx has r once
        by = scale_of(a);
        xx = hx = 0.f;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          u[h][e] *= by;
          v[h][e] *= by;
          xx += u[h][e] * u[h][e] + v[h][e] * v[h][e];
          hx += gu[h][e] * wa[e] * u[h][e] + gv[h][e] * wb[e] * v[h][e];
        }
        r = rsqrt32(sum_lanes<P>(xx) * over + p.eps * by * by);
      }
      const float k = sum_lanes<P>(hx) * over * r * r;
      if (!own || h0 + h >= H) continue;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        da[e] += gu[h][e] * u[h][e] * r;
        db[e] += gv[h][e] * v[h][e] * r;
        gu[h][e] = r * (gu[h][e] * wa[e] - u[h][e] * k) * by;
        gv[h][e] = r * (gv[h][e] * wb[e] - v[h][e] * k) * by;
      }
      if (g.dx[side] == nullptr) continue;
      T* d = (T*)g.dx[side] + (t * H + h0 + h) * p.D;
      store<W, true>(d + it.a, gu[h]);
      store<W, true>(d + it.b, gv[h]);
    }
  }
  if (own) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      sums[threadIdx.x / P][it.a + e] = da[e];
      sums[threadIdx.x / P][it.b + e] = db[e];
    }
  }
  __syncthreads();
  for (int ch = threadIdx.x; ch < p.D; ch += 256) {
    double a = 0.0;   // (the sums of sums lose nothing more)
#pragma unroll 8
    for (int x = 0; x < 256 / P; ++x) a += sums[x][ch];
    g.part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * p.D + ch] = (float)a;
  }
}

// Waves of one block each walk over heads; a lane always has the same channels, and
// adds up their dw in the block's row of the partial sums.
template <class T>
__global__ __launch_bounds__(64) void k_heads_grad_any(const HP p, const GP g) {
  const int side = blockIdx.y, H = p.H[side];
  float* part = g.part + ((int64_t)side * gridDim.x + blockIdx.x) * p.D;
  const float over = 1.f / p.D;
  for (int i = lane_id(); i < p.D - (p.R >> 1); i += 64) {
    int ca, cb;
    pair_of(i, p.R, p.inter, ca, cb);
    part[ca] = 0.f;
    if (cb >= 0) part[cb] = 0.f;
  }
#pragma unroll 1
  for (int64_t row = blockIdx.x; row < (int64_t)p.N * H; row += gridDim.x) {
    const int64_t t = row / H;
    const int h = (int)(row % H), b = (int)(t / p.L), l = (int)(t % p.L);
    const T* s = (const T*)p.x[side] + b * p.xs[side][0] + l * p.xs[side][1] + h * p.xs[side][2];
    const T* z = (const T*)g.dz[side] + b * g.zs[side][0] + l * g.zs[side][1] + h * g.zs[side][2];
    T* d = (T*)g.dx[side] + row * p.D;
    const bool wanted = g.dx[side] != nullptr;
    const int64_t pos = p.R ? pos_of(p, b, l) : 0;
    const bool in = pos >= 0 && pos < p.rows;
    float r = 1.f, k = 0.f, xx = 0.f, hx = 0.f, by = 1.f;
    auto pass = [&](auto sums) {
      for (int i = lane_id(); i < p.D - (p.R >> 1); i += 64) {
        int ca, cb;
        pair_of(i, p.R, p.inter, ca, cb);
        const float x = (float)s[ca] * by, wx = p.offset + ld_f(p.w[side], ca, p.wdt);
        float gx = (float)z[ca], y = 0.f, wy = 0.f, gy = 0.f;
        if (cb >= 0) {
          y = (float)s[cb] * by;
          wy = p.offset + ld_f(p.w[side], cb, p.wdt);
          const float c = in ? p.table[pos * p.R + i] : __builtin_nanf(""), sn = in ? p.table[pos * p.R + (p.R >> 1) + i] : __builtin_nanf("");
          const float a = gx, e = (float)z[cb];
          gx = a * c + e * sn;
          gy = e * c - a * sn;
        }
        if constexpr (decltype(sums)::value) {
          xx += x * x + y * y;
          hx += gx * wx * x + gy * wy * y;
        } else {
          if (wanted) d[ca] = (T)(r * (gx * wx - x * k) * by);
          part[ca] += gx * x * r;
          if (cb >= 0) {
            if (wanted) d[cb] = (T)(r * (gy * wy - y * k) * by);
            part[cb] += gy * y * r;
          }
        }
      }
    };
    pass(std::true_type{});
    float a = sum_lanes<64>(xx) * over + p.eps;
    if (far_off(a)) {   // once more
      by = scale_of(a);
      xx = hx = 0.f;
      pass(std::true_type{});
      a = sum_lanes<64>(xx) * over + p.eps * by * by;
    }
    r = rsqrt32(a);
    k = sum_lanes<64>(hx) * over * r * r;
    pass(std::false_type{});
  }
}

// dw of 4 channels of one side: the rows of partial sums, in 64 bits and an order of
// their own.
__global__ __launch_bounds__(256) void k_weight_grad(const float* part, int D, int rows_q, int rows_k, int wdt, void* dwq, void* dwk) {
  const int side = blockIdx.y, n = side ? rows_k : rows_q;
  void* out = side ? dwk : dwq;
  if (out == nullptr) return;
  part += side ? (int64_t)rows_q * D : 0;
  const int ch = blockIdx.x * 4 + (threadIdx.x & 3);
  double a = 0.0;
  if (ch < D)
#pragma unroll 4
    for (int x = threadIdx.x >> 2; x < n; x += 64) a += part[(int64_t)x * D + ch];
  // over the lanes with the same channel, then over the waves
#pragma unroll
  for (int o = 4; o < 64; o <<= 1) a += __shfl_xor(a, o);
  __shared__ double s[4][4];
  if (lane_id() < 4) s[threadIdx.x >> 6][lane_id()] = a;
  __syncthreads();
  if (threadIdx.x < 4 && ch < D)
    put1(out, wdt, ch, (float)((s[0][threadIdx.x] + s[1][threadIdx.x]) + (s[2][threadIdx.x] + s[3][threadIdx.x])));
}

bool float_type(int dt) { return dt == DN_F32 || dt == DN_BF16 || dt == DN_F16; }
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
// rows that start on 16 bytes whatever their index
bool wide(const void* p, const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] % 8) return false;
  return aligned(p);
}
int bad(const char* m) { return set_error(DN_E_INVALID, m); }
template <class F> void by_type(int dt, F f) {
  if (dt == DN_BF16) f((bf16)0.f);
  else if (dt == DN_F16) f((f16)0.f);
  else f(0.f);
}
template <int N> struct Num { static constexpr int value = N; };
// lanes of a head: a power of two, two groups each
template <class T, class F> void by_lanes(int D, F f) {
  constexpr int W = kWidth<T>;
  if (D <= 64) f(Num<32 / W>{});
  else if (D <= 128) f(Num<64 / W>{});
  else if (D <= 256) f(Num<128 / W>{});
  else f(Num<256 / W>{});
}
constexpr int kMostD = 512;   // of these kernels
constexpr int kMostTokens = 0x7fffffff, kMostBlocks = 0xffffff;   // a launch has fewer than 2^32 threads

// Threads of one head each that fill the card a few times over; from there on a thread
// takes two heads and stores past the caches, and in serving, where no gradient reads
// them again, loads past them too (9040 tokens of prompts, 227 MB, that no cache holds:
// 49 us, stores alone past them 51, neither 52; blocks of one chunk of heads for all
// tokens before the next 56).  us of launches in a loop, one head a thread / two, queries and
// keys normed and, behind the comma, stored with values: bf16 of 32 + 8 heads of 128, 1024
// tokens (0.3 M threads of one head) 7.7 / 8.2, 11.0 / 9.6; 4096 25.1 / 29.0, 30.7 / 31.4;
// 16384 89 / 93, 101 / 110; of 64, 8192 tokens (1.25 M) 29.4 / 27.6, 32.2 / 37.7; 16 + 4 heads
// of 256, 1024 tokens (0.3 M) 7.7 / 6.7, 11.1 / 9.0; 4096 24.8 / 19.7, 30.8 / 24.5; float32 of
// 256, 512 tokens (0.3 M) 7.1 / 6.3, 9.5 / 8.3; 2048 22.6 / 18.4, 27.7 / 21.9.  Neither side
// wins for all heads: at 256 channels two heads would pay from the smallest sizes on.
constexpr int64_t kManyThreads = 1 << 20;

// the checks that the entries share; NULL if all is well
const char* heads_error(const HP& p, int dtype, int pos_dtype) {
  if (p.N < 0 || p.L < 0 || p.H[0] < 0 || p.H[1] < 0 || p.H[2] < 0 || p.D <= 0) return "bad sizes";
  if (p.H[0] > 16384 || p.H[1] > 16384 || p.H[2] > 16384) return "too many heads";
  if (p.R < 0 || p.R % 2 || p.R > p.D) return "rotary channels must be even and at most D";
  if (!float_type(dtype) || !float_type(p.wdt) || !float_type(p.cdt) || (pos_dtype != DN_I32 && pos_dtype != DN_I64)) return "dtype not supported";
  if (!(p.eps >= 0.f) || !(p.eps - p.eps == 0.f) || !(p.offset - p.offset == 0.f)) return "eps and offset must be finite, eps not negative";
  return nullptr;
}
bool fast_heads(const HP& p, int dtype) {
  const int two = dtype == DN_F32 ? 8 : 16;   // channels of a lane
  if (p.D % two || p.R % two || p.D > kMostD || !aligned(p.table) || !aligned(p.w[0]) || !aligned(p.w[1])) return false;
  for (int i = 0; i < 3; ++i)
    if (p.H[i] && !(wide(p.x[i], p.xs[i], 3) && aligned(p.out[i]))) return false;
  return true;
}
template <bool PAGED> int launch_heads(const HP& p, int dtype, bool fast, hipStream_t st) {
  const int H = p.H[0] + p.H[1] + p.H[2];
  bool ok = true;
  by_type(dtype, [&](auto z) {
    using T = decltype(z);
    if (!fast) {
      const int64_t blocks = std::min<int64_t>(((int64_t)p.N * H + 3) / 4, kMostBlocks);
      hipLaunchKernelGGL((k_heads_any<T, PAGED>), dim3((unsigned)blocks), dim3(256), 0, st, p);
      return;
    }
    by_lanes<T>(p.D, [&](auto lanes) {
      constexpr int P = decltype(lanes)::value;
      const bool few = (int64_t)p.N * P * H < kManyThreads;
      const int64_t blocks = ((int64_t)p.N * P + 255) / 256 * (few ? chunks_of<1>(p) : chunks_of<2>(p));
      if (!(ok = blocks <= kMostBlocks)) return;
      if (few) hipLaunchKernelGGL((k_heads<T, P, 1, PAGED, false>), dim3((unsigned)blocks), dim3(256), 0, st, p);
      else hipLaunchKernelGGL((k_heads<T, P, 2, PAGED, true>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    });
  });
  if (!ok) return bad("too many tokens");
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}

int norm_params(const dn_norm_rotary_args* a, HP& p) {
  if (a == nullptr) return bad("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_norm_rotary_args built for another ABI version");
  if (a->B < 0 || a->L < 0 || (int64_t)a->B * a->L > kMostTokens) return bad("bad sizes");
  p.N = a->B * a->L; p.L = a->L; p.H[0] = a->Hq; p.H[1] = a->Hk; p.H[2] = 0; p.D = a->D; p.R = a->R; p.rows = a->rows;
  p.inter = a->interleaved != 0; p.pos64 = a->pos_dtype == DN_I64; p.wdt = a->weight_dtype; p.cdt = a->dtype;
  p.eps = a->eps; p.offset = a->weight_offset;
  p.x[0] = a->q; p.x[1] = a->k; p.w[0] = a->q_weight; p.w[1] = a->k_weight; p.out[0] = a->q_out; p.out[1] = a->k_out;
  p.pos = a->pos; p.table = a->table;
  for (int i = 0; i < 3; ++i) { p.xs[0][i] = a->q_strides[i]; p.xs[1][i] = a->k_strides[i]; }
  p.ps[0] = a->pos_strides[0]; p.ps[1] = a->pos_strides[1];
  if (const char* m = heads_error(p, a->dtype, a->pos_dtype)) return bad(m);
  if (p.N == 0 || p.H[0] + p.H[1] == 0) return DN_OK;
  // (a side without heads takes the other's weights, so that both pointers say whether there is a norm)
  if (!p.H[0]) p.w[0] = p.w[1];
  if (!p.H[1]) p.w[1] = p.w[0];
  if ((p.H[0] && !p.x[0]) || (p.H[1] && !p.x[1]) || !p.w[0] || !p.w[1] || (p.R && (!p.pos || !p.table || p.rows <= 0)))
    return bad("missing tensor pointer");
  return DN_OK;
}

// Blocks of the gradient's walk over tokens for each chunk of heads, and the rows of
// partial sums of q and k.
constexpr int kGradHeads = 2;
constexpr int64_t kGradBlocks = 2048;   // eight a CU
struct GradPlan { int x, rows_q, rows_k; };
GradPlan grad_plan(const HP& p, int dtype, bool fast) {
  if (!fast) {
    const int x = (int)std::min<int64_t>((int64_t)p.N * std::max(p.H[0], p.H[1]), kGradBlocks);
    return {x, x, x};
  }
  int P = dtype == DN_F32 ? 8 : 4;
  while (P * (dtype == DN_F32 ? 8 : 16) < p.D) P *= 2;
  const int64_t most = ((int64_t)p.N * P + 255) / 256;
  const int x = (int)std::max<int64_t>(1, std::min(most, kGradBlocks / chunks_of<kGradHeads>(p)));
  return {x, x * ((p.H[0] + kGradHeads - 1) / kGradHeads), x * ((p.H[1] + kGradHeads - 1) / kGradHeads)};
}
// (the two forms' plans may differ: the larger)
size_t grad_bytes(const HP& p, int dtype) {
  size_t n = 0;
  for (const bool fast : {false, true}) {
    if (fast && p.D > kMostD) continue;
    const GradPlan g = grad_plan(p, dtype, fast);
    n = std::max(n, ((size_t)g.rows_q + g.rows_k) * p.D * sizeof(float));
  }
  return n + 256;
}

}  // namespace
}  // namespace dn

using namespace dn;

extern "C" int dn_norm_rotary(const dn_norm_rotary_args* a, void* stream) {
  HP p{};
  if (const int rc = norm_params(a, p)) return rc;
  if (p.N == 0 || p.H[0] + p.H[1] == 0) return DN_OK;
  if ((p.H[0] && !p.out[0]) || (p.H[1] && !p.out[1])) return bad("missing tensor pointer");
  return launch_heads<false>(p, a->dtype, fast_heads(p, a->dtype), (hipStream_t)stream);
}

extern "C" size_t dn_norm_rotary_bwd_workspace_size(const dn_norm_rotary_args* a) {
  HP p{};
  if (norm_params(a, p) != DN_OK || p.N == 0 || p.H[0] + p.H[1] == 0) return 0;
  return grad_bytes(p, a->dtype);
}

extern "C" int dn_norm_rotary_bwd(const dn_norm_rotary_args* a, const dn_norm_rotary_grads* d, void* workspace, size_t workspace_bytes, void* stream) {
  HP p{};
  if (d == nullptr) return bad("null args");
  if (const int rc = norm_params(a, p)) return rc;
  if (p.N == 0 || p.H[0] + p.H[1] == 0) return DN_OK;
  if ((p.H[0] && !d->d_q) || (p.H[1] && !d->d_k)) return bad("missing tensor pointer");
  if (!workspace || workspace_bytes < grad_bytes(p, a->dtype)) return set_error(DN_E_WORKSPACE, "workspace missing or too small");
  GP g{};
  g.dz[0] = d->d_q; g.dz[1] = d->d_k; g.dx[0] = d->dq; g.dx[1] = d->dk;
  for (int i = 0; i < 3; ++i) { g.zs[0][i] = d->d_q_strides[i]; g.zs[1][i] = d->d_k_strides[i]; }
  g.part = (float*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
  p.out[0] = d->dq; p.out[1] = d->dk;
  bool fast = fast_heads(p, a->dtype);
  for (int i = 0; i < 2; ++i) fast = fast && (!p.H[i] || wide(g.dz[i], g.zs[i], 3));
  const GradPlan plan = grad_plan(p, a->dtype, fast);
  hipStream_t st = (hipStream_t)stream;
  by_type(a->dtype, [&](auto z) {
    using T = decltype(z);
    if (!fast) {
      hipLaunchKernelGGL((k_heads_grad_any<T>), dim3(plan.x, 2), dim3(64), 0, st, p, g);
      return;
    }
    by_lanes<T>(p.D, [&](auto lanes) {
      constexpr int P = decltype(lanes)::value;
      hipLaunchKernelGGL((k_heads_grad<T, P, kGradHeads>), dim3(plan.x, chunks_of<kGradHeads>(p)), dim3(256), 0, st, p, g);
    });
  });
  if (d->dq_weight || d->dk_weight)
    hipLaunchKernelGGL(k_weight_grad, dim3((p.D + 3) / 4, 2), dim3(256), 0, st, g.part, p.D, plan.rows_q, plan.rows_k, p.wdt, d->dq_weight, d->dk_weight);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}

extern "C" int dn_qkv_append(const dn_qkv_append_args* a, void* stream) {
  if (a == nullptr) return bad("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_qkv_append_args built for another ABI version");
  if (a->B < 0 || a->L < 0 || (int64_t)a->B * a->L > kMostTokens) return bad("bad sizes");
  HP p{};
  p.N = a->B * a->L; p.L = a->L; p.H[0] = a->Hq; p.H[1] = p.H[2] = a->Hkv; p.D = a->D; p.R = a->R; p.rows = a->rows;
  p.inter = a->interleaved != 0; p.pos64 = a->pos_dtype == DN_I64; p.wdt = a->weight_dtype; p.cdt = a->cache_dtype;
  p.pages = a->pages; p.eps = a->eps; p.offset = a->weight_offset;
  p.x[0] = a->q; p.x[1] = a->k; p.x[2] = a->v; p.w[0] = a->q_weight; p.w[1] = a->k_weight;
  p.out[0] = a->q_out; p.out[1] = a->k_cache; p.out[2] = a->v_cache;
  p.pos = a->pos; p.slots = a->slots; p.table = a->table;
  for (int i = 0; i < 3; ++i) {
    p.xs[0][i] = a->q_strides[i]; p.xs[1][i] = a->k_strides[i]; p.xs[2][i] = a->v_strides[i];
    p.cs[0][i] = a->kc_strides[i]; p.cs[1][i] = a->vc_strides[i];
  }
  p.ps[0] = a->L; p.ps[1] = 1;
  if (const char* m = heads_error(p, a->dtype, a->pos_dtype)) return bad(m);
  if (a->pages < 0 || a->page_size <= 0 || (a->page_size & (a->page_size - 1))) return bad("the cache needs pages of a power of two tokens");
  while ((1 << p.shift) < a->page_size) ++p.shift;
  if (p.pages == 0) p.H[1] = p.H[2] = 0;
  if (p.N == 0 || p.H[0] + p.H[1] == 0) return DN_OK;
  if ((p.H[0] && (!p.x[0] || !p.out[0])) || (p.H[1] && (!p.x[1] || !p.x[2] || !p.out[1] || !p.out[2])) || !p.pos || !p.slots ||
      (p.R && (!p.table || p.rows <= 0)))
    return bad("missing tensor pointer");
  if (!p.w[0] != !p.w[1]) return bad("both of the norms' weights, or none");
  const bool fast = fast_heads(p, a->dtype) && (!p.H[1] || (wide(p.out[1], p.cs[0], 3) && wide(p.out[2], p.cs[1], 3)));
  return launch_heads<true>(p, a->dtype, fast, (hipStream_t)stream);
}
