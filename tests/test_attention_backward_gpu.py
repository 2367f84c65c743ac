"""Gradient of causal attention on the GPU against the formulas in float64 and
against differences."""

import math

import pytest
import torch

from deltanet_tpu_amd import causal_attention
from tests import attn_ref as A
from tests.test_attention_gpu import _near, _rows

pytestmark = pytest.mark.gpu


def _grads(dev, q, k, v, do, **kw):
    qd, kd, vd = (t.to(dev).detach().requires_grad_(True) for t in (q, k, v))
    out = causal_attention(qd, kd, vd, **kw)
    return torch.autograd.grad(out, (qd, kd, vd), do.to(dev))


def _check(got, q, k, v, do, dt, starts=None, window=None, scale=None):
    B, L, Hq, D = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u = A.ROUND[dt]
    for x, y in zip(got, (q, k, v)):
        assert x.dtype == y.dtype and x.shape == y.shape
    for b in range(B):
        vis = A.visible(L, L, 0, None if starts is None else starts[b], window)
        for hk in range(Hkv):
            dk = dv = tk = tv = 0.0
            for h in range(hk * G, hk * G + G):
                r = A.attend_grad(q[b, :, h].double(), k[b, :, hk].double(), v[b, :, hk].double(), do[b, :, h].double(), vis, scale, dt)
                _near(got[0][b, :, h], r[0], r[3], f"dq row {b} head {h}")
                dk, dv, tk, tv = dk + r[1], dv + r[2], tk + r[4], tv + r[5]
            _near(got[1][b, :, hk], dk, tk + 1.05 * u * dk.abs() + A.TINY[dt], f"dk row {b} head {hk}")
            _near(got[2][b, :, hk], dv, tv + 1.05 * u * dv.abs() + A.TINY[dt], f"dv row {b} head {hk}")


def _inputs(B, L, Hq, Hkv, D, dt, seed=1):
    return (_rows(seed, B, L, Hq, D, dt=dt), _rows(seed + 1, B, L, Hkv, D, dt=dt), _rows(seed + 2, B, L, Hkv, D, dt=dt),
            _rows(seed + 3, B, L, Hq, D, dt=dt))


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,L,Hq,Hkv,D", [(1, 1, 1, 1, 64), (2, 3, 4, 2, 128), (1, 63, 3, 1, 256), (1, 64, 4, 4, 128),
                                          (2, 129, 8, 2, 64), (1, 300, 6, 1, 128), (1, 257, 4, 2, 256), (1, 515, 2, 2, 128)])
def test_gradients(dev, dt, B, L, Hq, Hkv, D):
    q, k, v, do = _inputs(B, L, Hq, Hkv, D, dt)
    _check(_grads(dev, q, k, v, do), q, k, v, do, dt)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("window", [None, 1, 17, 64, 1000])
@pytest.mark.parametrize("docs", [False, True])
@pytest.mark.parametrize("D", [64, 256])
def test_gradients_windows_and_documents(dev, dt, window, docs, D):
    B, L, Hq, Hkv = 2, 333, 3, 1
    q, k, v, do = _inputs(B, L, Hq, Hkv, D, dt)
    seg = starts = None
    if docs:
        seg = torch.zeros(B, L, dtype=torch.int64)
        for t in (1, 64, 65, 130, 200, 332):
            seg[0, t:] += 1
        seg[1, 100:] = 5
        starts = [A.starts_of(s.tolist()) for s in seg]
    got = _grads(dev, q, k, v, do, segment_ids=None if seg is None else seg.to(dev), window=window)
    _check(got, q, k, v, do, dt, starts, window)


def test_gradients_of_many_documents(dev):
    """A long row: the search for the last query of a key tile takes several steps."""
    B, L, H, D = 1, 4500, 1, 64
    q, k, v, do = _inputs(B, L, H, H, D, "bf16")
    g = torch.Generator().manual_seed(0)
    seg = (torch.rand(L, generator=g) < 0.004).long().cumsum(0)
    _check(_grads(dev, q, k, v, do, segment_ids=seg.to(dev)), q, k, v, do, "bf16", [A.starts_of(seg.tolist())])


def test_gradients_strided_scaled_and_repeatable(dev):
    B, L, Hq, Hkv, D = 2, 150, 4, 2, 128
    x = _rows(4, B, L, Hq + 2 * Hkv, D)
    do = _rows(5, B, L, Hq, D)
    xd = x.to(dev).requires_grad_(True)
    f = lambda: causal_attention(xd[:, :, :Hq], xd[:, :, Hq:Hq + Hkv], xd[:, :, Hq + Hkv:], scale=0.3)
    (dx,) = torch.autograd.grad(f(), xd, do.to(dev))
    got = dx[:, :, :Hq], dx[:, :, Hq:Hq + Hkv], dx[:, :, Hq + Hkv:]
    _check(got, x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:], do, "bf16", scale=0.3)
    assert torch.equal(dx, torch.autograd.grad(f(), xd, do.to(dev))[0])
    # a cotangent that is not contiguous, and a broadcast one
    (dy,) = torch.autograd.grad(f(), xd, do.to(dev).transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(dx, dy)
    (ds,) = torch.autograd.grad(f().sum(), xd)
    (de,) = torch.autograd.grad(f(), xd, torch.ones_like(do).to(dev))
    assert torch.equal(ds, de)


def test_gradient_against_differences(dev):
    """Central differences of a weighted sum along random directions, in float32:
    the sum's rounding (2^-24 of its terms) over the step, and the third
    derivative's step^2, stay under 2e-3 of the slope's scale."""
    B, L, Hq, Hkv, D = 1, 90, 4, 2, 64
    q, k, v, do = (t.to(dev) for t in _inputs(B, L, Hq, Hkv, D, "f32"))
    seg = torch.tensor([0] * 30 + [1] * 60, device=dev)
    f = lambda q, k, v: (causal_attention(q, k, v, segment_ids=seg, window=40).double() * do).sum()
    g = _grads(dev, q, k, v, do, segment_ids=seg, window=40)
    for i, x in enumerate((q, k, v)):
        d = torch.randn(x.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(i))
        step = 1e-2
        args = lambda s: [y + s * d if j == i else y for j, y in enumerate((q, k, v))]
        slope = float((f(*args(step)) - f(*args(-step))) / (2 * step))
        want = float((g[i].double() * d).sum())
        assert abs(slope - want) <= 2e-3 * float((g[i] * d).double().norm()) * math.sqrt(1.0 * L), (i, slope, want)


@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_gradients_hidden_infinities(dev, odd):
    """A document with infinities or NaNs leaves the gradients of its neighbours,
    in the same tiles, as they were."""
    B, L, H, D = 1, 200, 2, 64
    q, k, v, do = _inputs(B, L, H, H, D, "bf16")
    seg = torch.tensor([0] * 40 + [1] * 60 + [2] * 100, device=dev)
    base = _grads(dev, q, k, v, do, segment_ids=seg)
    for which in range(4):
        x = [t.clone() for t in (q, k, v, do)]
        x[which][0, 70, 0, 5] = odd
        got = _grads(dev, *x, segment_ids=seg)
        for a, b in zip(got, base):
            assert torch.equal(a[0, :40], b[0, :40]) and torch.equal(a[0, 100:], b[0, 100:])
            assert torch.equal(a[0, :, 1], b[0, :, 1])
        assert not torch.isfinite(got[2][0, 40:70, 0]).all() or which in (1, 2)
        assert not torch.isfinite(got[0][0, 70, 0]).any()


def test_gradient_of_some_inputs_and_lse(dev):
    q, k, v, do = (t.to(dev) for t in _inputs(1, 50, 2, 1, 64, "bf16"))
    full = _grads(dev, q, k, v, do)
    vr = v.clone().requires_grad_(True)
    out, lse = causal_attention(q, k, vr, return_lse=True)
    assert not lse.requires_grad
    (dv,) = torch.autograd.grad(out, vr, do)
    assert torch.equal(dv, full[2])
    with torch.no_grad():
        assert torch.equal(causal_attention(q, k, vr), out)
    e = torch.zeros(0, 5, 2, 64, device=dev, requires_grad=True)
    causal_attention(e, e, e).sum().backward()
    assert e.grad.shape == e.shape
