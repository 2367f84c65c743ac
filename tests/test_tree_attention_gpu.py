"""Attention of drafted trees over a paged cache against float64 on the CPU."""

import math

import pytest
import torch

from deltanet_tpu_amd import paged_attention, paged_tree_attention
from tests import attn_ref as A
from tests import serving_ref as S
from tests.test_attention_gpu import _near, _paged, _rows

pytestmark = pytest.mark.gpu


def _check(out, lse, q, ks, vs, new, lens, seen, dt, window=None, scale=None, count=16):
    G, D = q.shape[1] // ks[0].shape[1], q.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    i = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        vis = S.tree_visible(seen[b], m, window, count)
        for h in range(q.shape[1]):
            x = q[i:i + n, h].double()
            ref, l, tol = A.attend(x, ks[b][:, h // G].double(), vs[b][:, h // G].double(), vis, scale, dt)
            _near(out[i:i + n, h], ref, tol, f"sequence {b} head {h}")
            if lse is not None:
                _near(lse[i:i + n, h], l, 4 * A.f32_error(x, ks[b][:, h // G].double(), scale, torch.zeros(1)) + 1e-6 * l.abs(), "lse")
        i += n


CASES = [   # new tokens, sequence lengths
    ([1], [1]), ([1], [700]), ([3, 1, 0, 5], [3, 64, 9, 700]), ([16], [1016]), ([25, 2, 64, 33], [60, 2, 1064, 500]), ([70, 129], [70, 400]),
    ([0, 0], [4, 0]), ([4, 6], [0, 3]), ([1] * 9, [3, 900, 16, 17, 129, 700, 1, 2, 33]),
]
FORMS = [("bf16", 8, 2, 128, 16, False), ("bf16", 4, 1, 256, 64, True), ("f16", 3, 3, 64, 128, False), ("f32", 4, 2, 128, 32, False),
         ("bf16", 20, 1, 128, 1, False), ("f32", 2, 1, 256, 64, True), ("f16", 16, 2, 256, 8, False), ("f32", 8, 1, 64, 4, False)]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dt,Hq,Hkv,D,page,hf", FORMS)
def test_trees(dev, case, dt, Hq, Hkv, D, page, hf):
    new, lens = CASES[case]
    kc, vc, pt, sl, cu, ks, vs = _paged(case, new, lens, Hkv, D, page, dt, dev, hf)
    q = _rows(50 + case, sum(new), Hq, D, dt=dt)
    _, seen = S.trees(new, case)
    W = max(1, -(-max(new) // 64))
    out, lse = paged_tree_attention(q.to(dev), kc, vc, pt, sl, S.words(seen, W).to(dev), cu_seqlens=cu, return_lse=True)
    assert out.dtype == q.dtype and out.shape == q.shape
    _check(out, lse, q, ks, vs, new, lens, seen, dt, count=W)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["random", "empty", "all", "less-words"])
def test_any_mask(dev, dt, kind):
    """Masks that are no trees: rows that see nothing at all, tokens that see later ones
    or not themselves, bits past the sequence's tokens, tokens without a bit."""
    new, lens, D = [20, 64, 3, 90], [20, 300, 3, 90], 128
    kc, vc, pt, sl, cu, ks, vs = _paged(3, new, lens, 2, D, 16, dt, dev)
    q = _rows(4, sum(new), 8, D, dt=dt)
    g = torch.Generator().manual_seed(5)
    seen = [torch.rand(n, n, generator=g) < {"random": 0.3, "empty": 0.02, "all": 2.0, "less-words": 0.5}[kind] for n in new]
    W = 1 if kind == "less-words" else 2
    words = S.words(seen, W)
    at = 0
    for n in new:
        for j in range(n, 64 * W):   # bits of tokens that are not there
            words[at:at + n, j // 64] |= (1 << (j % 64)) - (1 << 64 if j % 64 == 63 else 0)
        at += n
    out, lse = paged_tree_attention(q.to(dev), kc, vc, pt, sl, words.to(dev), cu_seqlens=cu, return_lse=True)
    _check(out, lse, q, ks, vs, new, lens, seen, dt, count=W)
    if kind == "empty":
        none = torch.cat([~S.tree_visible(m, n, None, W).any(1) for m, n in zip(seen, lens)])
        assert none.any() and not out[none.to(dev)].any() and torch.isneginf(lse[none.to(dev)]).all()


@pytest.mark.parametrize("dt,window", [("bf16", 64), ("bf16", 100), ("f32", 128), ("f16", 300), ("bf16", 2 ** 40)])
@pytest.mark.parametrize("new", [[30, 1, 64, 2], [5, 60, 64, 64]])
def test_windows(dev, dt, window, new):
    lens = [40, 400, 700, 64]
    lens = [max(n, m) for n, m in zip(lens, new)]
    kc, vc, pt, sl, cu, ks, vs = _paged(6, new, lens, 2, 64, 16, dt, dev)
    q = _rows(7, sum(new), 8, 64, dt=dt)
    _, seen = S.trees(new, 8)
    out = paged_tree_attention(q.to(dev), kc, vc, pt, sl, S.words(seen, 1).to(dev), cu_seqlens=cu, window=window, scale=0.2)
    _check(out, None, q, ks, vs, new, lens, seen, dt, min(window, 1 << 20), 0.2)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_chains_are_causal_attention(dev, D):
    """A tree of one branch is what paged_attention gives, to both tolerances."""
    B, T, lens = 3, 10, [300, 1200, 10]
    kc, vc, pt, sl, cu, ks, vs = _paged(9, [T] * B, lens, 2, D, 32, "bf16", dev)
    q = _rows(10, B, T, 8, D)
    words = ((1 << torch.arange(1, T + 1)) - 1).repeat(B)[:, None].contiguous()
    out = paged_tree_attention(q.to(dev), kc, vc, pt, sl, words.to(dev))
    assert out.shape == q.shape
    seen = [torch.ones(T, T, dtype=torch.bool).tril()] * B
    _check(out.flatten(0, 1), None, q.flatten(0, 1), ks, vs, [T] * B, lens, seen, "bf16")
    causal = paged_attention(q.to(dev), kc, vc, pt, sl)
    assert float((out.float() - causal.float()).abs().max()) <= 2.0 ** -5


@pytest.mark.parametrize("T,page", [(8, 16), (64, 16), (64, 4)])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_hidden_infinities(dev, T, page, odd):
    """Drafts whose keys and values are not finite reach those alone that see them."""
    kc, vc, pt, sl, cu, _, _ = _paged(11, [T, 3], [150 + T, 70], 1, 128, page, "bf16", dev, junk=odd)
    q = _rows(12, T + 3, 4, 128).to(dev)
    _, seen = S.trees([T, 3], 13)
    words = S.words(seen, 1).to(dev)
    base = paged_tree_attention(q, kc, vc, pt, sl, words, cu_seqlens=cu)
    assert torch.isfinite(base).all()
    at = 150 + T // 2
    vc[int(pt[0, at // page]), at % page, :, 5] = odd
    hit = torch.zeros(T + 3, dtype=torch.bool, device=dev)
    hit[:T] = seen[0][:, T // 2].to(dev)
    out = paged_tree_attention(q, kc, vc, pt, sl, words, cu_seqlens=cu)
    assert torch.equal(out[~hit], base[~hit])
    assert not torch.isfinite(out[hit][..., 5]).any() and torch.isfinite(out[hit][..., 6:]).all()
    vc[int(pt[0, at // page]), at % page, :, 5] = 0.0
    kc[int(pt[0, at // page]), at % page, :, 5] = odd
    out = paged_tree_attention(q, kc, vc, pt, sl, words, cu_seqlens=cu)
    assert torch.equal(out[~hit], base[~hit]) or float((out[~hit].float() - base[~hit].float()).abs().max()) <= 2.0 ** -5
    assert torch.isfinite(out[~hit]).all()


def test_tokens_of_no_sequence_and_wild_pages(dev):
    new, lens = [5, 70], [40, 200]
    kc, vc, pt, sl, cu, ks, vs = _paged(14, new, lens, 2, 64, 16, "bf16", dev, junk=0.0)
    q = _rows(15, 82, 4, 64)
    _, seen = S.trees(new, 16)
    words = torch.full((82, 2), -1, dtype=torch.int64)
    words[3:78] = S.words(seen, 2)
    out, lse = paged_tree_attention(q.to(dev), kc, vc, pt, sl, words.to(dev), cu_seqlens=cu + 3, return_lse=True)
    for part in (slice(0, 3), slice(78, 82)):
        assert not out[part].any() and torch.isneginf(lse[part]).all()
    _check(out[3:78], lse[3:78], q[3:78], ks, vs, new, lens, seen, "bf16", count=2)
    wild = pt.clone()
    wild[0, 3:], wild[1, 13:] = -9, 1 << 30
    assert torch.equal(out, paged_tree_attention(q.to(dev), kc, vc, wild, sl, words.to(dev), cu_seqlens=cu + 3))
    wild[1, 0] = 1 << 30
    far = torch.tensor([40, 10 ** 9], dtype=torch.int32, device=dev)
    assert torch.isfinite(paged_tree_attention(q.to(dev), kc, vc, wild, far, words.to(dev), cu_seqlens=cu + 3)).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(dev, scale):
    new, lens = [40, 3], [200, 90]
    kc, vc, pt, sl, cu, ks, vs = _paged(17, new, lens, 1, 128, 16, "f32", dev)
    q = _rows(18, 43, 4, 128, dt="f32")
    _, seen = S.trees(new, 19)
    out = paged_tree_attention(q.to(dev), kc, vc, pt, sl, S.words(seen, 1).to(dev), cu_seqlens=cu, scale=scale)
    _check(out, None, q, ks, vs, new, lens, seen, "f32", scale=scale)


def test_offsets_past_32_bits(dev):
    pages, page, H, D = 33000, 128, 4, 256
    kc = torch.empty((pages, page, H, D), dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    pt = torch.tensor([[pages - 1, 5, pages - 2]], dtype=torch.int32, device=dev)
    n, T = 300, 60
    k, v, q = _rows(1, n, H, D), _rows(2, n, H, D), _rows(3, T, 8, D)
    for i, pg in enumerate(pt[0].tolist()):
        m = min(page, n - i * page)
        kc[pg, :m], vc[pg, :m] = k[i * page:i * page + m].to(dev), v[i * page:i * page + m].to(dev)
    _, seen = S.trees([T], 4)
    cu, sl = torch.tensor([0, T], dtype=torch.int32, device=dev), torch.tensor([n], dtype=torch.int32, device=dev)
    for m in (T, 2):
        cu[1] = m
        sub = [seen[0][:m, :m]]
        sl[0] = n - T + m
        out = paged_tree_attention(q[:m].to(dev), kc, vc, pt, sl, S.words(sub, 1).to(dev), cu_seqlens=cu)
        _check(out, None, q[:m], [k[:n - T + m]], [v[:n - T + m]], [m], [n - T + m], sub, "bf16")
