"""Drafted trees in the forms that large calls run in: every size of a tile of rows,
more sequences than a wave has lanes, scores far beyond a piece's first ones, two calls
at once."""

import math

import pytest
import torch

from deltanet_tpu_amd import paged_tree_attention
from tests import attn_ref as A
from tests import serving_ref as S
from tests.test_attention_gpu import _near, _paged, _rows
from tests.test_tree_attention_gpu import _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G,new", [(2, [8, 5]), (4, [16, 2, 12]), (4, [33, 20]), (8, [30, 14]), (5, [61, 37])])
@pytest.mark.parametrize("page", [16, 4])
def test_rows_of_every_tile(dev, dt, D, G, new, page):
    lens = [700 + n if i == 0 else 90 + n for i, n in enumerate(new)]
    kc, vc, pt, sl, cu, ks, vs = _paged(G + D, new, lens, 1, D, page, dt, dev)
    q = _rows(G, sum(new), G, D, dt=dt)
    _, seen = S.trees(new, G)
    out, lse = paged_tree_attention(q.to(dev), kc, vc, pt, sl, S.words(seen, 1).to(dev), cu_seqlens=cu, return_lse=True)
    _check(out, lse, q, ks, vs, new, lens, seen, dt, count=1)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_many_sequences(dev, dt):
    """150 sequences, some without a token, one long among short ones."""
    g = torch.Generator().manual_seed(1)
    B = 150
    new = [int(x) % 9 for x in torch.randint(0, 100, (B,), generator=g)]
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 60, (B,), generator=g))]
    new[77], lens[77] = 60, 2000
    kc, vc, pt, sl, cu, ks, vs = _paged(23, new, lens, 2, 64, 16, dt, dev)
    q = _rows(24, sum(new), 4, 64, dt=dt)
    _, seen = S.trees(new, 25)
    out, lse = paged_tree_attention(q.to(dev), kc, vc, pt, sl, S.words(seen, 1).to(dev), cu_seqlens=cu, return_lse=True)
    _check(out, lse, q, ks, vs, new, lens, seen, dt, count=1)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T", [6, 50, 100])
@pytest.mark.parametrize("grow", [4.0, 40.0])
def test_scores_that_grow(dev, dt, T, grow):
    """Keys that point more and more to the queries: a row's largest score of the last
    tiles is up to 2^150 times that of the first."""
    D, n = 128, 1500
    kc, vc, pt, sl, cu, ks, vs = _paged(31, [T], [n], 1, D, 16, dt, dev)
    q = _rows(32, T, 4, D, dt=dt).abs()
    u = torch.ones(n, 1, 1) * torch.linspace(0.0, 1.0, n)[:, None, None].square() * grow / 40.0
    k = (ks[0].float() * 0.05 + u).to(A.DT[dt])
    for i in range(n):
        kc[int(pt[0, i // 16]), i % 16] = k[i].to(dev)
    _, seen = S.trees([T], 33)
    W = -(-T // 64)
    out, lse = paged_tree_attention(q.to(dev), kc, vc, pt, sl, S.words(seen, W).to(dev), cu_seqlens=cu, scale=1.0, return_lse=True)
    _check(out, lse, q, [k], vs, [T], [n], seen, dt, scale=1.0, count=W)


def test_two_calls_at_once(dev):
    """On two streams, each with a workspace of its own."""
    D, T, lens = 128, 40, [3000, 800]
    args = []
    for s in (1, 2):
        kc, vc, pt, sl, cu, ks, vs = _paged(40 + s, [T, T], lens, 2, D, 16, "bf16", dev)
        _, seen = S.trees([T, T], s)
        args.append((_rows(s, 2 * T, 8, D).to(dev), kc, vc, pt, sl, S.words(seen, 1).to(dev), cu))
    call = lambda a: paged_tree_attention(*a[:6], cu_seqlens=a[6])
    want = [call(a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev) for _ in args]
    for _ in range(5):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(call(a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_a_graph_of_two_calls(dev):
    """Two layers' calls in a graph, replayed while lengths and masks change."""
    D, T, B = 64, 12, 2
    kc, vc, pt, sl, cu, ks, vs = _paged(50, [T] * B, [500, 300], 1, D, 16, "bf16", dev, junk=0.0)
    q = _rows(51, B, T, 4, D).to(dev)
    words = torch.zeros(B * T, 1, dtype=torch.int64, device=dev)
    lens = sl.clone()

    def both():
        a = paged_tree_attention(q, kc, vc, pt, lens, words)
        return a, paged_tree_attention(a, vc, kc, pt, lens, words)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both()
    for t in range(5):
        words.copy_(S.words(S.trees([T] * B, t)[1], 1))
        lens.copy_(sl - 37 * t)
        g.replay()
        got = [x.clone() for x in out]
        assert all(torch.equal(a, b) for a, b in zip(got, both())), t
        torch.cuda.synchronize()


@pytest.mark.parametrize("new,G", [([4, 2, 7], 2), ([3, 8, 1], 4), ([20, 11], 4), ([40, 64], 6)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 256])
def test_windows_of_every_tile(dev, dt, D, new, G):
    """The window's first key in the middle of a tile, in the first tile, in front of all;
    what lies before it may hold anything."""
    lens = [n + x for n, x in zip(new, (333, 64, 20))]
    kc, vc, pt, sl, cu, ks, vs = _paged(60, new, lens, 1, D, 16, dt, dev)
    for c in (kc, vc):   # (the window of the first sequence leaves its first pages)
        c[int(pt[0, 2])] = math.nan
    q = _rows(61, sum(new), G, D, dt=dt)
    _, seen = S.trees(new, 62)
    for window in (64, 111, 250):
        out, lse = paged_tree_attention(q.to(dev), kc, vc, pt, sl, S.words(seen, 1).to(dev), cu_seqlens=cu, window=window, return_lse=True)
        _check(out, lse, q, ks, vs, new, lens, seen, dt, window, count=1)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("T,G", [(4, 2), (7, 4), (30, 4), (64, 8)])
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_hidden_values_of_every_tile(dev, dt, T, G, odd):
    """A draft whose value is not finite reaches those alone that see it, in every form."""
    D, n = 128, 150 + T
    kc, vc, pt, sl, cu, _, _ = _paged(63, [T], [n], 1, D, 16, dt, dev, junk=odd)
    q = _rows(64, T, G, D, dt=dt).to(dev)
    _, seen = S.trees([T], 65)
    words = S.words(seen, 1).to(dev)
    base = paged_tree_attention(q, kc, vc, pt, sl, words, cu_seqlens=cu)
    at = 150 + T // 2
    vc[int(pt[0, at // 16]), at % 16, :, 9] = odd
    out = paged_tree_attention(q, kc, vc, pt, sl, words, cu_seqlens=cu)
    hit = seen[0][:, T // 2].to(dev)
    assert torch.isfinite(base).all() and torch.equal(out[~hit], base[~hit])
    assert not torch.isfinite(out[hit][..., 9]).any() and torch.isfinite(out[hit][..., 10:]).all()
