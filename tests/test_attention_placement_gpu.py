"""The attention operators where their operands lie and run: many sequences, one
long among short ones, far offsets, small pages, another stream, a captured graph."""

import math

import pytest
import torch

from deltanet_tpu_amd import apply_rotary, causal_attention, paged_attention, paged_kv_append, rotary_table
from tests import attn_ref as A
from tests.test_attention_gpu import _check_paged, _near, _paged, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["decode", "ragged", "long-among-short", "chunks"])
def test_many_sequences(dev, kind):
    """More sequences than a wave has lanes; some without a token."""
    g = torch.Generator().manual_seed(0)
    B = 150
    lens = torch.randint(1, 90, (B,), generator=g).tolist()
    lens[77] = 1500
    new = [1] * B
    if kind == "ragged":
        new = [int(x) % 4 for x in torch.randint(0, 100, (B,), generator=g)]
    elif kind == "long-among-short":   # several row tiles for one sequence of a call of few rows
        new[77] = 60
    elif kind == "chunks":
        new = [max(0, min(n, int(x))) for n, x in zip(lens, torch.randint(0, 60, (B,), generator=g))]
        new[77] = 300
    lens = [max(n, m) for n, m in zip(lens, new)]
    kc, vc, pt, sl, cu, ks, vs = _paged(3, new, lens, 1, 64, 16, "bf16", dev)
    q = _rows(4, sum(new), 4, 64)
    out, lse = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu, return_lse=True)
    _check_paged(out, lse, q, ks, vs, new, lens, "bf16")


@pytest.mark.parametrize("page", [1, 8])
def test_small_pages(dev, page):
    new, lens = [1, 1, 2], [37, 300, 64]
    kc, vc, pt, sl, cu, ks, vs = _paged(5, new, lens, 2, 128, page, "f16", dev)
    q = _rows(6, sum(new), 8, 128, dt="f16")
    _check_paged(paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu), None, q, ks, vs, new, lens, "f16")


def test_offsets_past_32_bits(dev):
    """Pages behind 2^32 elements of a cache: stored there and read from there."""
    pages, page, H, D = 33000, 128, 4, 256
    kc = torch.empty((pages, page, H, D), dtype=torch.bfloat16, device=dev)
    assert kc.numel() > 1 << 32
    vc = torch.empty_like(kc)
    pt = torch.tensor([[pages - 1, 5, pages - 2]], dtype=torch.int32, device=dev)
    n = 300
    sl = torch.tensor([n], dtype=torch.int32, device=dev)
    k, v, q = _rows(1, n, H, D), _rows(2, n, H, D), _rows(3, n, 8, D)
    cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
    paged_kv_append(k.to(dev), v.to(dev), kc, vc, pt, sl, cu_seqlens=cu)
    assert torch.equal(kc[pages - 1], k[:128].to(dev)) and torch.equal(vc[pages - 2, :44], v[256:].to(dev))
    _check_paged(paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu), None, q, [k], [v], [n], [n], "bf16")
    one = q[-1:].to(dev)
    _check_paged(paged_attention(one, kc, vc, pt, sl), None, q[-1:], [k], [v], [1], [n], "bf16")


def test_page_numbers_and_lengths_out_of_range(dev):
    """Whatever a page table holds past a sequence's tokens is not used; page numbers
    outside the cache and lengths past the table are read as the nearest there is."""
    new, lens = [1, 1], [40, 20]
    kc, vc, pt, sl, cu, ks, vs = _paged(7, new, lens, 1, 64, 16, "bf16", dev, junk=0.0)
    q = _rows(8, 2, 2, 64).to(dev)
    base = paged_attention(q, kc, vc, pt, sl)
    wild = pt.clone()
    wild[0, 3:], wild[1, 2:] = -7, 1 << 30
    assert torch.equal(base, paged_attention(q, kc, vc, wild, sl))
    wild[1, 0] = 1 << 30
    out = paged_attention(q, kc, vc, wild, torch.tensor([40, 10 ** 9], dtype=torch.int32, device=dev))
    assert torch.equal(out[0], base[0]) and torch.isfinite(out).all()


def test_another_stream(dev):
    """Inputs made on a stream, used there, with the default stream busy elsewhere."""
    s = torch.cuda.Stream(dev)
    L, Hq, Hkv, D = 600, 4, 2, 128
    q, k, v = _rows(1, 1, L, Hq, D), _rows(2, 1, L, Hkv, D), _rows(3, 1, L, Hkv, D)
    table = rotary_table(L, D, device=dev)
    pos = torch.arange(L, device=dev)
    ref_q, ref_k = apply_rotary(q.to(dev), k.to(dev), pos, table)
    ref = causal_attention(ref_q, ref_k, v.to(dev))
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=dev)
    for _ in range(10):
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(s):
        xs = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
        a, b = apply_rotary(xs[0], xs[1], pos, table)
        out = causal_attention(a, b, xs[2])
        (dq,) = torch.autograd.grad(out.float().sum(), xs[0])
    s.synchronize()
    assert torch.equal(out, ref) and torch.isfinite(dq).all()


def test_decode_step_in_a_graph(dev):
    """Append, rotate and attend captured once and replayed as the sequences grow; every
    replay against the eager calls on caches of their own."""
    B, Hq, Hkv, D, page, steps = 5, 8, 2, 128, 16, 6
    new = [1] * B
    lens = [3, 15, 16, 100, 400]
    kc, vc, pt, sl, _, _, _ = _paged(9, new, lens, Hkv, D, page, "bf16", dev, junk=0.0)
    pages = kc.shape[0] + B
    pt = pt[:, :-1]
    room = torch.full((B, 2), 0, dtype=torch.int32, device=dev)
    room[:, 0] = torch.arange(kc.shape[0], pages, dtype=torch.int32, device=dev)
    full = torch.zeros(B, pt.shape[1] + 2, dtype=torch.int32, device=dev)
    for b, n in enumerate(lens):
        c = -(-n // page)
        full[b, :c], full[b, c:c + 2] = pt[b, :c], room[b]
    grow = lambda c: torch.cat([c, torch.zeros((B,) + c.shape[1:], dtype=c.dtype, device=dev)])
    kc, vc = grow(kc), grow(vc)
    table = rotary_table(512, 64, device=dev)
    q, k, v = (torch.zeros(B, h, D, dtype=torch.bfloat16, device=dev) for h in (Hq, Hkv, Hkv))
    lens_g = sl.clone()

    def step(q, k, v, kc, vc, lens):
        paged_kv_append(k, v, kc, vc, full, lens, table=table)
        a, _ = apply_rotary(q, None, lens - 1, table)
        return paged_attention(a, kc, vc, full, lens)

    eager = [c.clone() for c in (kc, vc)]
    graph_caches = [c.clone() for c in (kc, vc)]
    side = torch.cuda.Stream(dev)
    with torch.cuda.stream(side):
        step(q, k, v, *(c.clone() for c in (kc, vc)), lens_g)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(q, k, v, *graph_caches, lens_g)
    # (capturing stores nothing: the first replay is the first step)
    gen = torch.Generator(device=dev).manual_seed(1)
    for t in range(steps):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=dev, generator=gen))
        lens_g.copy_(sl + t)
        g.replay()
        want = step(q, k, v, *eager, sl + t)
        torch.cuda.synchronize()
        assert torch.equal(out, want), t
        assert torch.equal(graph_caches[0], eager[0]) and torch.equal(graph_caches[1], eager[1])


def test_refusals_of_cuda_tensors(dev):
    """A cache whose rows do not start on 16 bytes, and a gradient of a gradient."""
    q = torch.randn(1, 2, 64, device=dev, dtype=torch.bfloat16)
    pt = torch.zeros(1, 1, device=dev, dtype=torch.int32)
    lens = torch.ones(1, device=dev, dtype=torch.int32)
    odd = torch.randn(2, 16, 1, 68, device=dev, dtype=torch.bfloat16)[..., :64]
    ok = torch.randn(2, 16, 1, 64, device=dev, dtype=torch.bfloat16)
    for kc, vc in ((odd, ok), (ok, odd)):
        with pytest.raises(ValueError, match="16 bytes"):
            paged_attention(q, kc, vc, pt, lens)
    x = torch.randn(1, 5, 2, 64, device=dev, requires_grad=True)
    y, = torch.autograd.grad(causal_attention(x, x, x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        y.sum().backward()


def _wide(pt, page, tokens=16384):
    """The page table with columns that no sequence uses: rules go by its width."""
    more = torch.full((pt.shape[0], tokens // page - pt.shape[1]), 1 << 30, dtype=torch.int32, device=pt.device)
    return torch.cat([pt, more], 1)


@pytest.mark.parametrize("new,lens", [([1], [1]), ([1], [1000]), ([1] * 9, [3, 2000, 16, 17, 129, 700, 1, 2, 33]), ([5, 5, 5], [5, 60, 300]),
                                      ([2, 3], [0, 1]), ([70], [1500]), ([300], [300]), ([9, 0, 40], [2000, 7, 40]), ([0, 0], [4, 0])])
@pytest.mark.parametrize("dt,Hq,Hkv,D,page,hf", [("bf16", 8, 2, 128, 16, False), ("bf16", 4, 1, 256, 64, True), ("f16", 3, 3, 64, 128, False),
                                                 ("f32", 4, 2, 128, 32, False), ("f32", 2, 1, 256, 64, True), ("f16", 16, 1, 256, 16, False)])
def test_wide_page_tables(dev, new, lens, dt, Hq, Hkv, D, page, hf):
    """The keys of tokens, drafts and chunks split over the card."""
    kc, vc, pt, sl, cu, ks, vs = _paged(17, new, lens, Hkv, D, page, dt, dev, hf)
    q = _rows(18, sum(new), Hq, D, dt=dt)
    out, lse = paged_attention(q.to(dev), kc, vc, _wide(pt, page), sl, cu_seqlens=cu, return_lse=True)
    _check_paged(out, lse, q, ks, vs, new, lens, dt)


@pytest.mark.parametrize("dt,window", [("bf16", 1024), ("bf16", 4100), ("f32", 256), ("f32", 300)])
@pytest.mark.parametrize("new,lens", [([1, 2, 1], [1400, 300, 1100]), ([50], [1500])])
def test_wide_page_tables_windows(dev, dt, window, new, lens):
    kc, vc, pt, sl, cu, ks, vs = _paged(19, new, lens, 1, 128, 16, dt, dev)
    q = _rows(20, sum(new), 4, 128, dt=dt)
    out = paged_attention(q.to(dev), kc, vc, _wide(pt, 16), sl, cu_seqlens=cu, window=window, scale=0.2)
    _check_paged(out, None, q, ks, vs, new, lens, dt, window, 0.2)


@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_wide_page_tables_hidden_infinities(dev, odd):
    """Later tokens of the same call that are not finite do not reach earlier ones."""
    kc, vc, pt, sl, cu, ks, vs = _paged(21, [20], [150], 1, 128, 16, "bf16", dev, junk=odd)
    pt = _wide(pt, 16)
    q = _rows(22, 20, 4, 128).to(dev)
    base = paged_attention(q, kc, vc, pt, sl, cu_seqlens=cu)
    vc[int(pt[0, 140 // 16]), 140 % 16] = odd   # the 11th new token
    out = paged_attention(q, kc, vc, pt, sl, cu_seqlens=cu)
    assert torch.equal(out[:10], base[:10])
    assert not torch.isfinite(out[10:]).any()


@pytest.mark.parametrize("kind", ["decode", "ragged", "long-among-short"])
def test_wide_page_tables_of_many_sequences(dev, kind):
    g = torch.Generator().manual_seed(1)
    B = 150
    lens = torch.randint(1, 90, (B,), generator=g).tolist()
    lens[77] = 1500
    new = [1] * B if kind != "ragged" else [int(x) % 4 for x in torch.randint(0, 100, (B,), generator=g)]
    if kind == "long-among-short":
        new[77] = 60
    lens = [max(n, m) for n, m in zip(lens, new)]
    kc, vc, pt, sl, cu, ks, vs = _paged(23, new, lens, 1, 64, 16, "bf16", dev)
    q = _rows(24, sum(new), 4, 64)
    out, lse = paged_attention(q.to(dev), kc, vc, _wide(pt, 16), sl, cu_seqlens=cu, return_lse=True)
    _check_paged(out, lse, q, ks, vs, new, lens, "bf16")
