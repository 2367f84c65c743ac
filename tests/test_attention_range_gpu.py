"""Values next to float32's largest under scores far above those that a kernel refers its
exponentials to: sums of products that leave the range on the way, results that do not."""

import math

import pytest
import torch

from deltanet_tpu_amd import causal_attention, paged_attention, paged_tree_attention
from tests import attn_ref as A
from tests import serving_ref as S
from tests.test_attention_gpu import _rows
from tests.test_tree_attention_pieces_gpu import HEADS, _masks, _run, _same

pytestmark = pytest.mark.gpu

LARGE = 2.0 ** 100


def _scores(seed, length, D, dt, peak, at):
    """Queries' first channel 1; keys whose first channel, the score, is `peak` at those places."""
    k, v = _rows(seed, length, D, dt=dt), _rows(seed + 1, length, D, dt="f32") * LARGE
    k[:, 0] = 0.0
    k[at, 0] = peak
    return k, v.to(A.DT[dt])


# rows of 700 tokens and one of 4 heads: small tiles, two sets of waves; 64 of 512: the large ones
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("B,L", [(1, 700), (64, 512)])
@pytest.mark.parametrize("peak", [35.0, 90.0])
def test_rows_of_large_values(dev, dt, D, B, L, peak):
    Hkv, G = 4, 4
    k, v = _scores(1, L, D, dt, peak, slice(100, 400, 7))
    q = _rows(3, L, G, D, dt=dt, scale=0.1)
    q[..., 0] = 1.0
    wide = lambda x: x[None, :, None].expand(B, L, Hkv, D).to(dev)
    qd = q[None, :, None].expand(B, L, Hkv, G, D).reshape(B, L, Hkv * G, D).to(dev)
    page = 16
    pages = L // page + 1
    cache = lambda x: torch.cat([x, x[:pages * page - L]]).view(pages, page, 1, D).expand(pages, page, Hkv, D).to(dev)
    pt = torch.arange(pages, dtype=torch.int32, device=dev).expand(B, pages).contiguous()
    lens = torch.full((B,), L, dtype=torch.int32, device=dev)
    rows = causal_attention(qd, wide(k), wide(v), scale=1.0)
    paged = paged_attention(qd, cache(k), cache(v), pt, lens, scale=1.0)
    vis = A.visible(L, L, 0)
    for g in range(G):
        ref, _, tol = A.attend(q[:, g].double(), k.double(), v.double(), vis, 1.0, dt)
        assert torch.isfinite(ref.to(A.DT[dt])).all()
        for out in (rows, paged):
            got = out.view(B, L, Hkv, G, D)[:, :, :, g].double().transpose(1, 2)
            _same(got, ref, tol, f"head {g}")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,n", [(64, 8), (64, 32), (64, 64), (128, 16), (128, 32), (128, 64), (256, 16), (256, 64)])
def test_trees_over_large_values(dev, dt, D, n):
    length = 1024 + n
    for peak, last in ((35.0, 0.0), (35.0, 12.0), (35.0, 37.0), (90.0, 70.0)):
        k, v = _scores(5, length, D, dt, peak, slice(300, 700, 7))
        k[960:, 0] = last
        q = _rows(7, n, 4, D, dt=dt, scale=0.1)
        q[..., 0] = 1.0
        for B, lens in ((64, [1024]), (41, [length, 777])):
            _run(dev, dt, q, k, v, 64, B, lens, _masks("tree", n), scale=1.0, tag=f"{peak} {last}")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,n", [(64, 8), (64, 64), (128, 16), (128, 32), (256, 16), (256, 64)])
def test_a_value_that_is_none_leaves_the_other_channels(dev, dt, D, n):
    """Seen by all, in the middle of long walks: its channel is not finite, the others keep
    their bits, also where the keys behind it score higher than those in front of it."""
    B, length, page, G = 41, 1024, 64, 4
    q, k, v = _rows(8, n, G, D, dt=dt, scale=0.1), _rows(9, length, D, dt=dt), _rows(10, length, D, dt=dt)
    q[..., 0] = 1.0
    for odd in (math.nan, math.inf):
        for last in (0.0, 25.0):
            k[:, 0] = 0.0
            k[900:, 0] = last
            outs = []
            for x in (0.0, odd):
                w = v.clone()
                w[500, 9] = x
                cache = lambda y: y.view(length // page, page, 1, D).expand(length // page, page, HEADS, D).to(dev)
                words = S.words([_masks("tree", n)], 1).repeat(B, 1).to(dev)
                pt = torch.arange(length // page, dtype=torch.int32, device=dev).expand(B, -1)
                qd = q[None, :, None].expand(B, n, HEADS, G, D).reshape(B, n, HEADS * G, D).to(dev)
                lens = torch.full((B,), length, dtype=torch.int32, device=dev)
                outs.append(paged_tree_attention(qd, cache(k), cache(w), pt, lens, words, scale=1.0))
            base, out = outs
            assert torch.isfinite(base).all() and not torch.isfinite(out[..., 9]).any()
            rest = [c for c in range(D) if c != 9]
            assert torch.equal(out[..., rest], base[..., rest]), (odd, last)
