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


def _grads(dev, q, k, v, do, **kw):
    x = [t.to(dev).detach().requires_grad_(True) for t in (q, k, v)]
    return [g.double().cpu() for g in torch.autograd.grad(causal_attention(*x, **kw), x, do.to(dev))]


def _formula(q, k, v, do):
    """dq, dk, dv of one key head and its group in float64."""
    L, G, D = q.shape
    vis = A.visible(L, L, 0)
    dq, dk, dv = torch.zeros(L, G, D, dtype=torch.float64), 0.0, 0.0
    for g in range(G):
        dq[:, g], a, b = A.attend_grad(q[:, g].double(), k.double(), v.double(), do[:, g].double(), vis, 1.0 / math.sqrt(D), "f16")[:3]
        dk, dv = dk + a, dv + b
    return dq, dk, dv


def _powers(seed, *shape):
    """Cotangents of magnitude 1/2, 1 and 2, which powers of two scale exactly."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 2, shape, generator=g) * 2.0 - 1.0) * 2.0 ** torch.randint(-1, 2, shape, generator=g)


@pytest.mark.parametrize("power", [-10, -13, -17])
@pytest.mark.parametrize("B,L,Hq,Hkv,D", [(1, 2048, 4, 2, 64), (2, 2111, 16, 8, 128), (1, 1000, 2, 2, 256)])
def test_gradients_of_small_cotangents(dev, B, L, Hq, Hkv, D, power):
    """The gradient is linear in the cotangent: a power of two goes through it to
    the rounding of the results (each of the two within 2^-11, and half a step
    next to zero).  And both are as near the formulas, by 2-norms, as four roundings
    (P or dS, the output's, the result's, the sums')."""
    q, k, v = _rows(1, B, L, Hq, D, dt="f16"), _rows(2, B, L, Hkv, D, dt="f16"), _rows(3, B, L, Hkv, D, dt="f16")
    do, f = _powers(4, B, L, Hq, D), 2.0 ** power
    one, small = _grads(dev, q, k, v, do.half()), _grads(dev, q, k, v, (do * f).half())
    u = A.ROUND["f16"]
    for name, a, b in zip(("dq", "dk", "dv"), one, small):
        _near(b, a * f, 2.1 * u * (a * f).abs() + A.TINY["f16"] * (1.0 + f), name)
    G, b = Hq // Hkv, B - 1
    ref = _formula(q[b, :, :G], k[b, :, 0], v[b, :, 0], do[b, :, :G])
    for name, r, x in zip(("dq", "dk", "dv"), ref, (small[0][b, :, :G], small[1][b, :, 0], small[2][b, :, 0])):
        assert (x - r * f).norm() <= 4 * u * (r * f).norm() + A.TINY["f16"] * math.sqrt(r.numel()), name


def test_gradients_of_large_cotangents(dev):
    """dS beyond float16's range, of results that are not."""
    B, L, H, D = 1, 60, 2, 64
    q, k, v = (_rows(s, B, L, H, D, dt="f16") for s in (1, 2, 3))
    do, f, u = _powers(4, B, L, H, D), 2.0 ** 14, A.ROUND["f16"]
    one, large = _grads(dev, q, k, v, do.half(), scale=2.0 ** -7), _grads(dev, q, k, v, (do * f).half(), scale=2.0 ** -7)
    for name, a, b in zip(("dq", "dk"), one, large):
        _near(b, a * f, 2.1 * u * (a * f).abs() + A.TINY["f16"] * (1.0 + f), name)


@pytest.mark.parametrize("small_first", [False, True])
def test_gradients_of_documents_of_different_size(dev, small_first):
    """Cotangents of one document 2^16 below those of its neighbours: each as near
    the formulas as by itself."""
    L, H, D, n = 700, 2, 64, 350
    q, k, v = (_rows(s, 1, L, H, D, dt="f16") for s in (1, 2, 3))
    do, u = _powers(4, 1, L, H, D) * 16.0, A.ROUND["f16"]
    do[:, :n] *= 2.0 ** -16 if small_first else 1.0
    do[:, n:] *= 1.0 if small_first else 2.0 ** -16
    seg = torch.tensor([0] * n + [1] * (L - n), device=dev)
    got = _grads(dev, q, k, v, do.half(), segment_ids=seg)
    for h in range(H):
        for s in (slice(0, n), slice(n, L)):
            ref = _formula(q[0, s, h:h + 1], k[0, s, h], v[0, s, h], do[0, s, h:h + 1])
            for name, r, x in zip(("dq", "dk", "dv"), ref, (got[0][0, s, h:h + 1], got[1][0, s, h], got[2][0, s, h])):
                assert (x - r).norm() <= 4 * u * r.norm() + A.TINY["f16"] * math.sqrt(r.numel()), (name, h, s)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_gradient_of_values_under_one_key_above(dev, D):
    """Every query has the first key about 13 nats above the others: what it leaves
    them, e^-13 each, reaches their values' gradients."""
    L = 1024
    g = torch.Generator().manual_seed(D)
    q, k = torch.zeros(1, L, 1, D), torch.zeros(1, L, 1, D)
    x = math.sqrt(13.0 * math.sqrt(D))
    q[..., 0], k[:, 0, :, 0] = x, x
    k[..., 1:] = torch.randn(1, L, 1, D - 1, generator=g)
    v, do = torch.randn(1, L, 1, D, generator=g), 1.0 + 0.1 * torch.randn(1, L, 1, D, generator=g)
    q, k, v, do = q.half(), k.half(), v.half(), do.half()
    dv = _grads(dev, q, k, v, do)[2]
    ref = _formula(q[0], k[0, :, 0], v[0, :, 0], do[0])[2]
    a, r = dv[0, 1:, 0], ref[1:]
    assert (a - r).norm() <= 4 * A.ROUND["f16"] * r.norm() + A.TINY["f16"] * math.sqrt(r.numel())
