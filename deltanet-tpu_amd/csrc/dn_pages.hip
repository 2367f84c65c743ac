// Page tables and slots of a paged cache from the sequences' lengths, and the
// accepted tokens of drafted trees moved to the front.
//
// Nothing here computes: bound by the launch and a chain of two or three dependent
// loads (lengths, page table, store) at a token or two per sequence, 2.7 us a launch, by
// the stores in long queues of prompts: 5.6 million tokens' positions and slots (67 MB)
// 15 us.  Accepted tokens of 64 sequences in 12 layers (13 MB) move in 7 us, one
// user's in 4.7.
#include <atomic>

#include "dn_common.h"
#include "dn_host.h"

namespace dn {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int scan64(int x) {   // inclusive, over a wave
  const int l = lane_id();
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (l >= o) x += y;
  }
  return x;
}

// x summed over the block's threads in front, and over all of them
template <int NT> __device__ __forceinline__ int block_scan(int x, int* waves, int& all) {
  const int w = threadIdx.x >> 6, s = scan64(x);
  __syncthreads();   // (its last use)
  if (lane_id() == 63) waves[w] = s;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    if (i < w) before += waves[i];
    all += waves[i];
  }
  return before + s - x;
}

// The last i of n with a[i] <= x (a rises, a[0] <= x).
__device__ __forceinline__ int last_at_most(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (a[m] <= x) lo = m;
    else hi = m;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// pages
// ---------------------------------------------------------------------------
struct RP {
  int32_t *pool, *table, *held, *short_of;
  const int32_t* lens;
  int64_t stride;
  int capacity, max_pages, B, shift;
  uint32_t tag;   // of this launch; not 0
};
constexpr int kTagShift = 9;   // (256 blocks at most)

// Every block adds up all sequences' needs itself and moves an even share of the
// pages: a page that is taken is read off the stack, or, if it lies among those given
// back in this call, from the row of the sequence that gives it, which nothing
// overwrites.  Lengths and counts are written by the block that comes to its end last,
// when all others have read them; it reads nothing that they wrote, so that the count
// of those that ended needs no fence.  The count lies in the pool's second word under
// the launch's tag, so that whatever else that word holds counts as none.
template <int NT> __global__ __launch_bounds__(NT) void k_reserve(const RP p) {
  extern __shared__ int lds[];   // [2][B]: pages taken, given back by the sequences in front
  int *taken = lds, *given = lds + p.B;
  __shared__ int waves[NT / 64], s_last;
  const int count = min(max(p.pool[0], 0), p.capacity);
  uint32_t* ended = reinterpret_cast<uint32_t*>(&p.pool[1]);
  if (gridDim.x > 1 && threadIdx.x == 0) {   // (where it fails, another block has put the tag there)
    uint32_t was = __hip_atomic_load(ended, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (was >> kTagShift != p.tag)
      __hip_atomic_compare_exchange_strong(ended, &was, p.tag << kTagShift, __ATOMIC_RELAXED, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  auto needs = [&](int b, int& h, int& need) {
    h = min(max(p.held[b], 0), p.max_pages);
    const int n = max(p.lens[b], 0);
    need = (n >> p.shift) + ((n & ((1 << p.shift) - 1)) != 0);
  };
#pragma unroll 4
  for (int b = threadIdx.x; b < p.B; b += NT) {
    int h, need;
    needs(b, h, need);
    taken[b] = need <= p.max_pages ? max(need - h, 0) : 0;
    given[b] = max(h - need, 0);
  }
  __syncthreads();
  // a run of sequences per thread
  const int per = (p.B + NT - 1) / NT, b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
  int grow = 0, back = 0;
  for (int b = b0; b < b1; ++b) {
    grow += taken[b];
    back += given[b];
  }
  int F, all;
  int f = block_scan<NT>(back, waves, F), a = block_scan<NT>(grow, waves, all);
  const int full = count + F;
  // sequences take while what all up to them need is there
  int got = 0;
  for (int b = b0; b < b1; ++b) {
    const int g = taken[b], x = given[b];
    taken[b] = a;
    given[b] = f;
    a += g;
    f += x;
    if (a <= full) got = a;   // (what those that fit take is what all up to the last of them need)
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) got = max(got, __shfl_xor(got, o));
  __syncthreads();
  if (lane_id() == 0) waves[threadIdx.x >> 6] = got;
  __syncthreads();
  int A = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) A = max(A, waves[i]);
  const int left = full - A;
  // page number x of those given back, in the order of the sequences and their pages
  // (bounded, as below, for lengths that something changes meanwhile)
  auto given_page = [&](int x) {
    const int b = last_at_most(given, p.B, x);
    int h, need;
    needs(b, h, need);
    return p.table[b * p.stride + min(need + (x - given[b]), p.max_pages - 1)];
  };
  const int me = blockIdx.x * NT + threadIdx.x, step = gridDim.x * NT;
#pragma unroll 2
  for (int k = me; k < A; k += step) {
    const int b = last_at_most(taken, p.B, k), at = full - 1 - k;
    const int col = min(max(p.held[b], 0), p.max_pages) + (k - taken[b]);
    p.table[b * p.stride + min(col, p.max_pages - 1)] = at < count ? p.pool[2 + at] : given_page(F - 1 - (at - count));
  }
#pragma unroll 2
  for (int k = me; k < min(left, p.capacity) - count; k += step) p.pool[2 + count + k] = given_page(F - 1 - k);
  __syncthreads();
  if (gridDim.x > 1) {
    if (threadIdx.x == 0)
      s_last = __hip_atomic_fetch_add(ended, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (p.tag << kTagShift) + gridDim.x - 1;
    __syncthreads();
    if (!s_last) return;
  }
#pragma unroll 4
  for (int b = threadIdx.x; b < p.B; b += NT) {
    int h, need;
    needs(b, h, need);
    const bool fits = need <= p.max_pages && (need <= h || taken[b] + (need - h) <= full);
    p.short_of[b] = fits ? 0 : need - h;
    p.held[b] = fits ? need : h;
  }
  if (threadIdx.x == 0) {
    p.pool[0] = min(left, p.capacity);
    p.pool[1] = 0;
  }
}

// ---------------------------------------------------------------------------
// slots
// ---------------------------------------------------------------------------
struct SP {
  int N, B, T, shift, max_pages, words;   // T: new tokens per sequence (cu NULL)
  const int32_t *pt, *lens, *cu, *held, *parents;
  int32_t* pos;
  int64_t* slots;
  uint64_t* visible;
  int64_t pts;
};

__device__ __forceinline__ void no_token(const SP& p, int i) {
  p.pos[i] = -1;
  p.slots[i] = -1;
  for (int w = 0; w < p.words; ++w) p.visible[(int64_t)i * p.words + w] = 0;
}

struct Seq { int c0, n, len, held; };
__device__ __forceinline__ Seq seq_of(const SP& p, int b) {
  Seq s{b * p.T, p.T, p.lens[b], p.held ? p.held[b] : p.max_pages};
  if (p.cu) {
    s.c0 = min(max(p.cu[b], 0), p.N);
    s.n = min(max(p.cu[b + 1], s.c0), p.N) - s.c0;
  }
  s.held = min(s.held, p.max_pages);
  return s;
}

__device__ __forceinline__ int64_t slot_of(const SP& p, int b, const Seq& s, int64_t x) {
  const int64_t pg = x >> p.shift;
  if (x < 0 || pg >= s.held) return -1;
  const int page = p.pt[b * p.pts + pg];
  return page < 0 ? -1 : ((int64_t)page << p.shift) + (x & ((1 << p.shift) - 1));
}

// tokens in front of cu[0] and from cu[B] on
__device__ __forceinline__ void clear_rest(const SP& p) {
  if (p.cu == nullptr) return;
  const int c0 = min(max(p.cu[0], 0), p.N), c1 = min(max(p.cu[p.B], c0), p.N);
  const int64_t me = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kThreads + threadIdx.x, step = (int64_t)gridDim.x * gridDim.y * kThreads;
  for (int64_t i = me; i < c0; i += step) no_token(p, (int)i);
  for (int64_t i = c1 + me; i < p.N; i += step) no_token(p, (int)i);
}

// x: sequences, y: parts of their tokens
constexpr int kMostSequences = 0xffffff;   // a launch has fewer than 2^32 threads
__global__ __launch_bounds__(kThreads) void k_slots(const SP p) {
  clear_rest(p);
  const int b = blockIdx.x;
  const Seq s = seq_of(p, b);
  for (int64_t i = blockIdx.y * kThreads + threadIdx.x; i < s.n; i += gridDim.y * kThreads) {
    const int64_t x = (int64_t)s.len - s.n + i;
    p.pos[s.c0 + i] = (int)x;
    p.slots[s.c0 + i] = slot_of(p, b, s, x);
  }
}

// A block per sequence: every node's ancestors by doubling, in one word of 64 nodes
// after the other.  In each round a node takes over what its furthest known ancestor
// has, and that one's furthest: as many rounds as the depth has bits.
constexpr int kNodes = 1024, kMine = kNodes / kThreads;
__global__ __launch_bounds__(kThreads) void k_slots_tree(const SP p) {
  __shared__ uint64_t bits[kNodes];
  __shared__ short up[kNodes], deep[kNodes];
  clear_rest(p);
  const int b = blockIdx.x;
  const Seq s = seq_of(p, b);
  const int n = min(s.n, 64 * p.words);
  for (int i = n + threadIdx.x; i < s.n; i += kThreads) no_token(p, s.c0 + i);
  for (int w = 0; w < p.words && 64 * w < n; ++w) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int a = p.parents[s.c0 + i];
      up[i] = (short)(a < i ? max(a, -1) : -1);
      bits[i] = i >> 6 == w ? 1ull << (i & 63) : 0;
      deep[i] = 0;
      if (a >= 0 && a < i) deep[i] = 1;
    }
    __syncthreads();
    bool more = true;
#pragma unroll 1
    while (more) {
      uint64_t nb[kMine];
      int nu[kMine], nd[kMine];
      bool any = false;
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int i = threadIdx.x + k * kThreads;
        if (i >= n) continue;
        const int u = up[i];
        nb[k] = bits[i];
        nd[k] = deep[i];
        nu[k] = u;
        if (u >= 0) {
          nb[k] |= bits[u];
          nd[k] += deep[u];
          nu[k] = up[u];
          any |= nu[k] >= 0;
        }
      }
      more = __syncthreads_or(any);
#pragma unroll
      for (int k = 0; k < kMine; ++k) {
        const int i = threadIdx.x + k * kThreads;
        if (i >= n) continue;
        bits[i] = nb[k];
        deep[i] = (short)nd[k];
        up[i] = (short)nu[k];
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
      p.visible[(int64_t)(s.c0 + i) * p.words + w] = bits[i];
      if (w == 0) {
        const int64_t off = (int64_t)s.len - s.n;
        p.pos[s.c0 + i] = (int)(off + deep[i]);
        p.slots[s.c0 + i] = slot_of(p, b, s, off + i);
      }
    }
    __syncthreads();
  }
  for (int w = (n + 63) / 64; w < p.words; ++w)
    for (int i = threadIdx.x; i < n; i += kThreads) p.visible[(int64_t)(s.c0 + i) * p.words + w] = 0;
}

// ---------------------------------------------------------------------------
// accepted tokens
// ---------------------------------------------------------------------------
struct KP {
  int layers, B, most, pages, shift, max_pages;
  uint32_t H, pieces;   // pieces: of a head
  char *k, *v;
  const int32_t *pt, *starts, *kept, *held;
  int32_t* lens;
  int64_t ks[4], vs[4], pts;   // in bytes
};

// x: parts of a token's pieces over all layers, y: sequences.  A thread moves one
// piece of every kept token, kBatch of them read before the first is written: what is
// kept rises, so no later token lies where an earlier one goes.
constexpr int kBatch = 8, kPath = 64;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <class V> __global__ __launch_bounds__(kThreads) void k_keep(const KP p) {
  __shared__ int from_page[kPath], from_in[kPath], to_page[kPath], to_in[kPath];
  __shared__ int s_count;
  const int b = blockIdx.y;
  const int start = p.starts[b];
  const int64_t end = (int64_t)(p.held ? min(p.held[b], p.max_pages) : p.max_pages) * (1 << p.shift);   // (held may be anything)
  const uint32_t n = (uint32_t)p.layers * 2 * p.H * p.pieces;
  int before = -1, total = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < p.most; i0 += kPath) {
    __syncthreads();   // (the last part has been moved)
    if (threadIdx.x < 64) {
      const int l = threadIdx.x, i = i0 + l;
      const int at = i < p.most ? p.kept[(int64_t)b * p.most + i] : -1;
      const int left = __shfl_up(at, 1);
      const bool good = start >= 0 && at > (l ? left : before) && (int64_t)start + at < end;
      const unsigned long long stop = ~__ballot(good);
      const int c = stop ? __builtin_ctzll(stop) : 64;
      if (l < c) {
        const int64_t f = (int64_t)start + at, t = (int64_t)start + i;
        const int fp = p.pt[b * p.pts + (f >> p.shift)], tp = p.pt[b * p.pts + (t >> p.shift)];
        const bool move = f != t && fp >= 0 && fp < p.pages && tp >= 0 && tp < p.pages;
        from_page[l] = move ? fp : -1;
        from_in[l] = (int)(f & ((1 << p.shift) - 1));
        to_page[l] = tp;
        to_in[l] = (int)(t & ((1 << p.shift) - 1));
      }
      if (l == 63) s_count = c;
      before = __shfl(at, 63);
    }
    __syncthreads();
    const int c = s_count;
    total += c;
    for (uint32_t x = blockIdx.x * kThreads + threadIdx.x; x < n; x += gridDim.x * kThreads) {
      const uint32_t piece = x % p.pieces, head = x / p.pieces, h = head % p.H, y = head / p.H;
      const bool val = y & 1;
      const int64_t s0 = val ? p.vs[0] : p.ks[0], s1 = val ? p.vs[1] : p.ks[1], s2 = val ? p.vs[2] : p.ks[2], s3 = val ? p.vs[3] : p.ks[3];
      char* base = (val ? p.v : p.k) + (int64_t)(y >> 1) * s0 + h * s3 + piece * (int64_t)sizeof(V);
#pragma unroll 1
      for (int i = 0; i < c; i += kBatch) {
        V r[kBatch];
        bool move[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          move[e] = i + e < c && from_page[i + e] >= 0;
          if (move[e]) r[e] = *reinterpret_cast<const V*>(base + from_page[i + e] * s1 + from_in[i + e] * s2);
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
          if (move[e]) *reinterpret_cast<V*>(base + to_page[i + e] * s1 + to_in[i + e] * s2) = r[e];
      }
    }
    if (c < 64) break;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) p.lens[b] = start + total;
}

int bad(const char* m) { return set_error(DN_E_INVALID, m); }
int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}
const char* page_error(int page_size, int max_pages) {
  if (max_pages <= 0 || page_size <= 0 || (page_size & (page_size - 1))) return "the cache needs pages of a power of two tokens";
  return nullptr;
}
int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

}  // namespace
}  // namespace dn

using namespace dn;

extern "C" int dn_paged_reserve(const dn_paged_reserve_args* a, void* stream) {
  if (a == nullptr) return bad("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_paged_reserve_args built for another ABI version");
  if (a->capacity < 0 || a->B < 0) return bad("bad sizes");
  if (a->B > DN_MAX_SEQUENCES) return bad("at most 4096 sequences");
  if (const char* m = page_error(a->page_size, a->max_pages)) return bad(m);
  // (every count of pages stays within 32 bits)
  if ((int64_t)a->B * a->max_pages + a->capacity > 0x7fffffff) return bad("too many pages");
  if (a->B == 0) return DN_OK;
  if (!a->pool || !a->page_table || !a->held || !a->lens || !a->short_of) return bad("missing tensor pointer");
  if (a->B > 1 && a->page_table_stride < a->max_pages) return bad("the rows of the page table overlap");
  static std::atomic<uint32_t> launches{0};
  const uint32_t tag = launches.fetch_add(1, std::memory_order_relaxed) % ((1u << (32 - kTagShift)) - 1) + 1;
  const RP p{a->pool, a->page_table, a->held, a->short_of, a->lens, a->page_table_stride, a->capacity, a->max_pages, a->B, shift_of(a->page_size), tag};
  // Blocks of 16 waves hide the searches of many pages, those of 4 start sooner where there
  // are few.  us of a launch among others, 4 waves / 16, sequences x columns: a page or three
  // for each of 64 x 64 4.2 / 4.5, 64 x 512 4.8 / 5.5, 256 x 64 5.0 / 5.8, 256 x 512 5.1 / 5.7,
  // 1024 x 64 6.6 / 6.5, 2048 x 64 9.3 / 7.7, 2048 x 256 11.1 / 8.2; every page of 64 x 64
  // 9.8 / 6.7, 256 x 64 11.3 / 9.2, 64 x 1024 10.9 / 9.0, 256 x 512 12.3 / 9.7, 2048 x 171 16.8 /
  // 11.6.  Servers take a page or three at a time.
  const int64_t entries = (int64_t)a->B * a->max_pages;
  const size_t lds = 2 * a->B * sizeof(int);
  if (entries <= 65536) hipLaunchKernelGGL(k_reserve<256>, dim3((unsigned)((entries + 2047) / 2048)), dim3(256), lds, (hipStream_t)stream, p);
  else hipLaunchKernelGGL(k_reserve<1024>, dim3((unsigned)std::min<int64_t>(256, (entries + 4095) / 4096)), dim3(1024), lds, (hipStream_t)stream, p);
  return launched();
}

extern "C" int dn_paged_slots(const dn_paged_slots_args* a, void* stream) {
  if (a == nullptr) return bad("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_paged_slots_args built for another ABI version");
  if (a->N < 0 || a->B < 0) return bad("bad sizes");
  if (const char* m = page_error(a->page_size, a->max_pages)) return bad(m);
  if (a->N && !a->B) return bad("tokens without a sequence");
  if (a->B > kMostSequences) return bad("too many sequences");
  if (a->cu_seqlens == nullptr && a->B && a->N % a->B) return bad("without cu_seqlens every sequence has N / B new tokens");
  if (a->parents ? a->words < 1 || a->words * 64 > kNodes : a->words != 0) return bad("trees have 1 to 16 words of visible tokens");
  if (a->N == 0) return DN_OK;
  if (!a->page_table || !a->seq_lens || !a->positions || !a->slots || (a->words && !a->visible)) return bad("missing tensor pointer");
  SP p{};
  p.N = a->N; p.B = a->B; p.T = a->cu_seqlens ? 0 : a->N / a->B; p.shift = shift_of(a->page_size); p.max_pages = a->max_pages;
  p.words = a->words; p.pt = a->page_table; p.lens = a->seq_lens; p.cu = a->cu_seqlens; p.held = a->held; p.parents = a->parents;
  p.pos = a->positions; p.slots = a->slots; p.visible = a->visible; p.pts = a->page_table_stride;
  if (a->parents) {
    hipLaunchKernelGGL(k_slots_tree, dim3(p.B), dim3(kThreads), 0, (hipStream_t)stream, p);
  } else {
    // parts of 1024 tokens, as many as the longest sequence may have, but no more blocks than fill the card
    const int64_t parts = std::min<int64_t>((p.cu ? p.N : p.T) / 1024 + 1, std::max<int64_t>(1, 8192 / p.B));
    hipLaunchKernelGGL(k_slots, dim3(p.B, (unsigned)parts), dim3(kThreads), 0, (hipStream_t)stream, p);
  }
  return launched();
}

extern "C" int dn_kv_keep(const dn_kv_keep_args* a, void* stream) {
  if (a == nullptr) return bad("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_kv_keep_args built for another ABI version");
  if (a->layers < 0 || a->B < 0 || a->B > 65535 || a->H < 0 || a->D <= 0 || a->most < 0 || a->pages < 0) return bad("bad sizes");
  if (a->dtype != DN_F32 && a->dtype != DN_BF16 && a->dtype != DN_F16) return bad("dtype not supported");
  if (const char* m = page_error(a->page_size, a->max_pages)) return bad(m);
  if (a->B == 0) return DN_OK;
  if ((a->pages && a->layers && (!a->k_cache || !a->v_cache)) || !a->page_table || !a->starts || (a->most && !a->kept) || !a->lens) return bad("missing tensor pointer");
  KP p{};
  const int e = a->dtype == DN_F32 ? 4 : 2;
  p.layers = a->layers; p.B = a->B; p.H = a->H; p.most = a->most; p.pages = a->pages; p.max_pages = a->max_pages;
  p.shift = shift_of(a->page_size);
  p.k = (char*)a->k_cache; p.v = (char*)a->v_cache; p.pt = a->page_table; p.starts = a->starts; p.kept = a->kept; p.held = a->held; p.lens = a->lens;
  p.pts = a->page_table_stride;
  int64_t all = (int64_t)(uintptr_t)a->k_cache | (int64_t)(uintptr_t)a->v_cache | (int64_t)a->D * e;
  for (int i = 0; i < 4; ++i) {
    p.ks[i] = a->kc_strides[i] * e;
    p.vs[i] = a->vc_strides[i] * e;
    all |= p.ks[i] | p.vs[i];
  }
  const int piece = all % 16 == 0 ? 16 : e;
  p.pieces = a->D * e / piece;
  const int64_t n = (int64_t)p.layers * 2 * p.H * p.pieces;
  if (n > 0x7fffffff) return bad("too many layers and heads");
  const dim3 grid((unsigned)std::min<int64_t>(std::max<int64_t>((n + kThreads - 1) / kThreads, 1), 1024), p.B);
  hipStream_t st = (hipStream_t)stream;
  if (piece == 16) hipLaunchKernelGGL(k_keep<u32x4>, grid, dim3(kThreads), 0, st, p);
  else if (e == 4) hipLaunchKernelGGL(k_keep<uint32_t>, grid, dim3(kThreads), 0, st, p);
  else hipLaunchKernelGGL(k_keep<uint16_t>, grid, dim3(kThreads), 0, st, p);
  return launched();
}
