"""float16's narrow range of exponents: one key far above thousands of others,
small and large cotangents."""

import math

import pytest
import torch

from deltanet_tpu_amd import causal_attention, paged_attention
from tests import attn_ref as A
from tests.test_attention_gpu import _near, _paged, _rows
from tests.test_attention_placement_gpu import _wide

pytestmark = pytest.mark.gpu


def _one_above(L, Hq, Hkv, D, nats, at):
    """Keys whose scores with the last query are 0 but for that of key `at`, `nats`
    above; values of mean 1, 0 at that key, so that the output is what the others
    leave."""
    g = torch.Generator().manual_seed(L + D)
    q, k = torch.randn(L, Hq, D, generator=g), torch.randn(L, Hkv, D, generator=g)
    v = 1.0 + 0.1 * torch.randn(L, Hkv, D, generator=g)
    k[..., 0] = 0.0
    q[-1] = 0.0
    x = math.sqrt(nats * math.sqrt(D))
    q[-1, :, 0], k[at, :, 0], v[at] = x, x, 0.0
    return q.half(), k.half(), v.half()


def _last(q, k, v, got):
    Hq, D = q.shape[1:]
    G = Hq // k.shape[1]
    vis = torch.ones(1, len(k), dtype=torch.bool)
    for h in range(Hq):
        ref, _, tol = A.attend(q[-1:, h].double(), k[:, h // G].double(), v[:, h // G].double(), vis, 1.0 / math.sqrt(D), "f16")
        _near(got[h:h + 1], ref, tol, f"head {h}")


@pytest.mark.parametrize("nats", [9.0, 12.0, 12.8, 13.2])
@pytest.mark.parametrize("other", [False, True])   # the one above: the query's own key, another
@pytest.mark.parametrize("L,Hq,Hkv,D", [(8192, 8, 2, 64), (8192, 2, 2, 128), (4000, 16, 8, 256), (8192, 1, 1, 256)])
def test_rows_one_key_above_many(dev, L, Hq, Hkv, D, nats, other):
    q, k, v = _one_above(L, Hq, Hkv, D, nats, 77 if other else L - 1)
    out = causal_attention(q[None].to(dev), k[None].to(dev), v[None].to(dev))
    _last(q, k, v, out[0, -1])


@pytest.mark.parametrize("other", [False, True])
@pytest.mark.parametrize("page,new", [(8, 70), (8, 1), (16, 1), (16, 40)])   # pages of 8: the kernel of many rows
def test_paged_one_key_above_many(dev, page, new, other):
    L, Hq, Hkv, D = 8192, 4, 2, 128
    q, k, v = _one_above(L, Hq, Hkv, D, 12.8, 77 if other else L - 1)
    kc, vc, pt, sl, cu, ks, vs = _paged(1, [new], [L], Hkv, D, page, "f16", dev)
    for c, x in ((kc, k), (vc, v)):
        c[pt[0, :L // page].long()] = x.view(L // page, page, Hkv, D).to(dev)
    out = paged_attention(q[-new:].to(dev), kc, vc, pt, sl, cu_seqlens=cu)
    _last(q, k, v, out[-1])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 256])
def test_rows_own_score_of_minus_infinity(dev, dt, D):
    """A key that no query can choose, among them its own: it has no weight, and a
    query that sees nothing else has no result."""
    L, H, at = 300, 2, 200
    q, k, v = (_rows(s, 1, L, H, D, dt=dt) for s in (1, 2, 3))
    q[..., 0] = 1.0
    shut = k.clone()
    for i in (at, 150):
        shut[0, i, :, 0] = -math.inf
    seg = torch.tensor([0] * 150 + [1] * 150)
    out = causal_attention(q.to(dev), shut.to(dev), v.to(dev), segment_ids=seg.to(dev))
    vis = A.visible(L, L, 0, A.starts_of(seg.tolist()))
    vis[:, [150, at]] = False
    for h in range(H):
        ref, _, tol = A.attend(q[0, :, h].double(), k[0, :, h].double(), v[0, :, h].double(), vis, 1.0 / math.sqrt(D), dt)
        ref[150] = math.nan
        _near(out[0, :, h], ref, tol, f"head {h}")
