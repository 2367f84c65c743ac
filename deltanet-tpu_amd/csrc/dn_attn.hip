// C entry points of softmax attention: checks of the arguments, the choice of the
// kernel, and the document starts that training passes down.
#include "dn_attn_fwd.h"

namespace dn {
namespace {

constexpr int kScan = 1024;

// One workgroup per row: starts[i] = the last j <= i whose id differs from its
// predecessor's, as a running maximum over blocks of kScan tokens.
__global__ __launch_bounds__(kScan) void k_doc_starts(const void* seg, int i64, int batched, int L, int32_t* starts) {
  __shared__ int part[kScan / 64];
  const int64_t row = (int64_t)blockIdx.x * L, base = batched ? row : 0;
  auto id = [&](int i) { return i64 ? ((const int64_t*)seg)[base + i] : (int64_t)((const int32_t*)seg)[base + i]; };
  int carry = 0;
  for (int i0 = 0; i0 < L; i0 += kScan) {
    const int i = i0 + threadIdx.x, l = threadIdx.x & 63, w = threadIdx.x >> 6;
    int m = i < L && i > 0 && id(i) != id(i - 1) ? i : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(m, o);
      if (l >= o) m = max(m, x);
    }
    if (l == 63) part[w] = m;
    __syncthreads();
    int all = carry;
    for (int x = 0; x < kScan / 64; ++x) {
      if (x < w) m = max(m, part[x]);
      all = max(all, part[x]);
    }
    m = max(m, carry);
    carry = all;
    if (i < L) starts[row + i] = m;
    __syncthreads();
  }
}

int bad(const char* m) { return set_error(DN_E_INVALID, m); }
bool wide(const void* p, const int64_t* s, int dtype, int n) {
  const int64_t per = dtype == DN_F32 ? 4 : 8;
  for (int i = 0; i < n; ++i)
    if (s[i] % per) return false;
  return ((uintptr_t)p & 15) == 0;
}

// a window that no row is longer than is none
int window_of(int window, int64_t most) { return window >= most ? 0 : window; }

// checks that the entries share; NULL if all is well
const char* shape_error(int64_t tokens, int Hq, int Hkv, int D, int dtype, float scale, int window) {
  if (D != 64 && D != 128 && D != 256) return "head dimension must be 64, 128 or 256";
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv) return "query heads must be a multiple of the key heads";
  if (dtype != DN_F32 && dtype != DN_BF16 && dtype != DN_F16) return "attention dtype not supported";
  const float e = scale * kLog2e;
  if (!(e - e == 0.f)) return "scale must be finite";
  if (window < 0) return "window must not be negative";
  if (tokens * Hq >= kMostIndex) return "too many query rows";
  return nullptr;
}

int paged_params(const dn_paged_attention_args* a, AF& p) {
  if (a == nullptr) return bad("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_paged_attention_args built for another ABI version");
  if (a->N < 0 || a->B < 0) return bad("bad attention sizes");
  if (const char* m = shape_error(a->N, a->Hq, a->Hkv, a->D, a->dtype, a->scale, a->window)) return bad(m);
  if (a->pages <= 0 || a->max_pages <= 0 || a->page_size <= 0 || (a->page_size & (a->page_size - 1)))
    return bad("the cache needs pages of a power of two tokens");
  const int64_t most = (int64_t)a->max_pages * a->page_size;
  if (most >= kMostIndex) return bad("a sequence must have fewer than 2^31 - 1024 tokens");
  if (a->N && !a->B) return bad("tokens without a sequence");
  if (a->cu_seqlens == nullptr && a->B && a->N % a->B) return bad("without cu_seqlens every sequence has N / B new tokens");
  if (a->N && (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->page_table || !a->seq_lens)) return bad("missing tensor pointer");
  if (!wide(a->q, a->q_strides, a->dtype, 3) || !wide(a->k_cache, a->kc_strides, a->dtype, 3) ||
      !wide(a->v_cache, a->vc_strides, a->dtype, 3) || ((uintptr_t)a->out & 15))
    return bad("attention rows must start on 16 bytes");
  p.B = a->B; p.N = a->N; p.T = a->cu_seqlens ? 0 : a->B ? a->N / a->B : 0;
  set_heads(p, a->Hq, a->Hkv);
  p.window = window_of(a->window, most);
  p.pages = a->pages; p.max_pages = a->max_pages;
  while ((1 << p.shift) < a->page_size) ++p.shift;
  p.sc = a->scale * kLog2e;
  p.q = a->q; p.k = a->k_cache; p.v = a->v_cache; p.out = a->out; p.lse = a->lse;
  p.cu = a->cu_seqlens; p.lens = a->seq_lens; p.pt = a->page_table; p.pts = a->page_table_stride;
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_strides[i]; p.ks[i] = a->kc_strides[i]; p.vs[i] = a->vc_strides[i]; }
  return DN_OK;
}

}  // namespace
}  // namespace dn

using namespace dn;

extern "C" size_t dn_paged_attention_workspace_size(const dn_paged_attention_args* a) {
  AF p{};
  if (paged_params(a, p) != DN_OK || p.N == 0 || !attn_few_takes(p, a->D, a->dtype)) return 0;
  return attn_few_bytes(p, a->D) + 256;
}

extern "C" int dn_paged_attention(const dn_paged_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  AF p{};
  if (const int rc = paged_params(a, p)) return rc;
  if (p.N == 0) return DN_OK;
  hipError_t e;
  if (attn_few_takes(p, a->D, a->dtype)) {
    if (!workspace || workspace_bytes < attn_few_bytes(p, a->D) + 256) return set_error(DN_E_WORKSPACE, "workspace missing or too small");
    p.part = (float*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    e = attn_few(p, a->D, a->dtype, (hipStream_t)stream);
  } else {
    e = attn_many(p, a->D, a->dtype, true, (hipStream_t)stream);
  }
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}

namespace {
// (units of a call are counted in 32 bits: 32 keys of a tile of 16 rows at the least)
int tree_params(const dn_paged_attention_args* a, const uint64_t* visible, int words, AF& p) {
  if (const int rc = paged_params(a, p)) return rc;
  if (words < 1 || words > 16) return bad("trees have 1 to 16 words of visible tokens");
  if (a->window && a->window < 64 * words) return bad("the window of a tree must take in its words");
  if (p.N && !visible) return bad("missing tensor pointer");
  if (p.N && ((int64_t)p.N * p.G / 16 + p.B) * p.Hkv * ((((int64_t)p.max_pages << p.shift) + 31) / 32) >= (int64_t)1 << 31)
    return bad("too many rows over too many tokens");
  p.vis = visible; p.words = words;
  p.window = window_of(a->window, kMostIndex);   // (lengths may pass the page table)
  return DN_OK;
}
}  // namespace

extern "C" size_t dn_paged_tree_attention_workspace_size(const dn_paged_attention_args* a, int32_t words) {
  AF p{};
  if (tree_params(a, reinterpret_cast<const uint64_t*>(8), words, p) != DN_OK || p.N == 0) return 0;
  return attn_tree_bytes(p, a->D, a->dtype) + 256;
}

extern "C" int dn_paged_tree_attention(const dn_paged_attention_args* a, const uint64_t* visible, int32_t words, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  AF p{};
  if (const int rc = tree_params(a, visible, words, p)) return rc;
  if (p.N == 0) return DN_OK;
  if (!workspace || workspace_bytes < attn_tree_bytes(p, a->D, a->dtype) + 256) return set_error(DN_E_WORKSPACE, "workspace missing or too small");
  p.part = (float*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
  const hipError_t e = attn_tree(p, a->D, a->dtype, (hipStream_t)stream);
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}

extern "C" int dn_document_starts(const void* seg, int32_t seg_dtype, int32_t batched, int32_t B, int32_t L, int32_t* starts, void* stream) {
  if (B < 0 || L < 0 || L >= kMostIndex || (seg_dtype != DN_I32 && seg_dtype != DN_I64)) return bad("bad segment ids");
  if (B == 0 || L == 0) return DN_OK;
  if (!seg || !starts) return bad("missing tensor pointer");
  hipLaunchKernelGGL(k_doc_starts, dim3(B), dim3(kScan), 0, (hipStream_t)stream, seg, seg_dtype == DN_I64, batched, L, starts);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}

namespace {
int attention_params(const dn_attention_args* a, AF& p) {
  if (a == nullptr) return bad("null args");
  if (a->abi_version != DN_ABI_VERSION) return set_error(DN_E_ABI, "dn_attention_args built for another ABI version");
  if (a->B < 0 || a->L < 0) return bad("bad attention sizes");
  if (const char* m = shape_error((int64_t)a->B * a->L, a->Hq, a->Hkv, a->D, a->dtype, a->scale, a->window)) return bad(m);
  if (a->B && a->L && (!a->q || !a->k || !a->v || !a->out)) return bad("missing tensor pointer");
  if (!wide(a->q, a->q_strides, a->dtype, 3) || !wide(a->k, a->k_strides, a->dtype, 3) || !wide(a->v, a->v_strides, a->dtype, 3) ||
      (((uintptr_t)a->out | (uintptr_t)a->out_low) & 15))
    return bad("attention rows must start on 16 bytes");
  p.B = a->B; p.T = a->L; p.N = a->B * a->L;
  set_heads(p, a->Hq, a->Hkv);
  p.window = window_of(a->window, a->L);
  p.sc = a->scale * kLog2e;
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out; p.low = a->out_low; p.lse = a->lse; p.start = a->starts;
  for (int i = 0; i < 3; ++i) { p.qs[i] = a->q_strides[i]; p.ks[i] = a->k_strides[i]; p.vs[i] = a->v_strides[i]; }
  return DN_OK;
}
}  // namespace

extern "C" int dn_attention_fwd(const dn_attention_args* a, void* stream) {
  AF p{};
  if (const int rc = attention_params(a, p)) return rc;
  if (p.N == 0) return DN_OK;
  const hipError_t e = attn_many(p, a->D, a->dtype, false, (hipStream_t)stream);
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}

static size_t delta_bytes(const AF& p) { return ((size_t)p.N * p.Hkv * p.G * sizeof(float) + 255) / 256 * 256; }

extern "C" size_t dn_attention_bwd_workspace_size(const dn_attention_args* a) {
  AF p{};
  if (attention_params(a, p) != DN_OK) return 0;
  if (p.N == 0) return 0;
  return delta_bytes(p) + attn_backward_part_bytes(p, a->D, a->dtype) + 256;
}

extern "C" int dn_attention_bwd(const dn_attention_args* a, const void* d_out, void* dq, void* dk, void* dv, void* workspace,
                                size_t workspace_bytes, void* stream) {
  AB p{};
  if (const int rc = attention_params(a, p.f)) return rc;
  if (p.f.N == 0) return DN_OK;
  if (!a->lse || !d_out || !dq || !dk || !dv) return bad("missing tensor pointer");
  if (((uintptr_t)d_out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) return bad("attention rows must start on 16 bytes");
  if (!workspace || workspace_bytes < dn_attention_bwd_workspace_size(a)) return set_error(DN_E_WORKSPACE, "workspace missing or too small");
  p.scale = a->scale;
  p.d_out = d_out; p.dq = dq; p.dk = dk; p.dv = dv;
  p.delta = (float*)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
  p.part = (float*)((char*)p.delta + delta_bytes(p.f));
  const hipError_t e = attn_backward(p, a->D, a->dtype, (hipStream_t)stream);
  return e == hipSuccess ? DN_OK : set_error(DN_E_LAUNCH, hipGetErrorString(e));
}
