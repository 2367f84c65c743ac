"""The forms of the attention kernels that large calls run in (tiles of 128 rows,
one set of waves; the gradient's 32 rows per wave and unsplit keys), a few heads and
rows of each against float64."""

import math

import pytest
import torch

from deltanet_tpu_amd import causal_attention, paged_attention
from tests import attn_ref as A
from tests.test_attention_gpu import _near, _paged, _rows

pytestmark = pytest.mark.gpu
FORMS = [(dt, D) for dt in ("bf16", "f16", "f32") for D in (64, 128, 256)]
B, L, HQ, HKV = 2, 2111, 16, 8   # 2 x 8 heads of 33 tiles of 128 rows: more than 512 workgroups
SLICES = [slice(0, 70), slice(1000, 1080), slice(2030, L)]


def _inputs(dt, D):
    return (_rows(1, B, L, HQ, D, dt=dt), _rows(2, B, L, HKV, D, dt=dt), _rows(3, B, L, HKV, D, dt=dt), _rows(4, B, L, HQ, D, dt=dt))


def _check_some(out, lse, q, k, v, dt, starts=None, window=None, slices=SLICES):
    scale = 1.0 / math.sqrt(q.shape[3])
    vis = A.visible(L, L, 0, starts, window)
    for b, h in ((0, 0), (1, 7), (1, 15)):
        kk, vv = k[b, :, h // 2].double(), v[b, :, h // 2].double()
        for s in slices:
            ref, l, tol = A.attend(q[b, s, h].double(), kk, vv, vis[s], scale, dt)
            _near(out[b, s, h], ref, tol, f"row {b} head {h} {s}")
            if lse is not None:
                _near(lse[b, s, h], l, 4 * A.f32_error(q[b, s, h].double(), kk, scale, torch.zeros(1)) + 1e-6 * l.abs(), "lse")


@pytest.mark.parametrize("dt,D", FORMS)
@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("docs", [False, True])
def test_rows(dev, dt, D, window, docs):
    q, k, v, _ = _inputs(dt, D)
    seg = torch.zeros(L, dtype=torch.int64)
    for t in (1, 64, 65, 1030, 2040, L - 1):
        seg[t:] += 1
    out, lse = causal_attention(q.to(dev), k.to(dev), v.to(dev), window=window, segment_ids=seg.to(dev) if docs else None, return_lse=True)
    _check_some(out, lse, q, k, v, dt, A.starts_of(seg.tolist()) if docs else None, window)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dt,D", FORMS)
def test_rows_scores_far_above_the_own(dev, dt, D):
    """Rows beyond the range of exponents, whose tiles are done again, and rows
    whose largest score grows from tile to tile."""
    q, k, v, _ = _inputs(dt, D)
    for at, size in ((3, 40.0), (70, 80.0), (1900, 160.0)):
        k[:, at] = 0
        k[:, at, :, 0] = size
    q[:, 1000:1010, :, 0], q[:, 2050:2060, :, 0] = 50.0, 100.0
    out, lse = causal_attention(q.to(dev), k.to(dev), v.to(dev), return_lse=True)
    _check_some(out, lse, q, k, v, dt)


@pytest.mark.parametrize("dt,D", FORMS)
@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_rows_hidden_infinities(dev, dt, D, odd):
    """A token whose key and value are not finite reaches its own document alone."""
    q, k, v, _ = _inputs(dt, D)
    seg = torch.tensor([0] * 900 + [1] * 500 + [2] * 711, device=dev)
    base = causal_attention(q.to(dev), k.to(dev), v.to(dev), segment_ids=seg)
    at = 1003
    v[:, at, :, 3] = odd
    out = causal_attention(q.to(dev), k.to(dev), v.to(dev), segment_ids=seg)
    hit = torch.zeros(L, dtype=torch.bool, device=dev)
    hit[at:1400] = True
    assert torch.equal(out[:, ~hit], base[:, ~hit]) and torch.equal(out[:, hit][..., 4:], base[:, hit][..., 4:])
    assert not torch.isfinite(out[:, hit][..., 3]).any()
    k[:, at] = odd
    out = causal_attention(q.to(dev), k.to(dev), v.to(dev), segment_ids=seg)
    assert torch.equal(out[:, ~hit], base[:, ~hit]) and not torch.isfinite(out[:, at]).any()


@pytest.mark.parametrize("dt,D", FORMS)
@pytest.mark.parametrize("window,docs", [(None, False), (300, True)])
def test_gradients(dev, dt, D, window, docs):
    q, k, v, do = _inputs(dt, D)
    seg = torch.zeros(L, dtype=torch.int64)
    for t in (1, 64, 65, 1030, 2040, L - 1):
        seg[t:] += 1
    x = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = causal_attention(*x, window=window, segment_ids=seg.to(dev) if docs else None)
    dq, dk, dv = torch.autograd.grad(out, x, do.to(dev))
    vis = A.visible(L, L, 0, A.starts_of(seg.tolist()) if docs else None, window)
    scale, u = 1.0 / math.sqrt(D), A.ROUND[dt]
    for b, hk in ((0, 0), (1, 7)):
        rk = rv = tk = tv = 0.0
        for h in (2 * hk, 2 * hk + 1):
            r = A.attend_grad(q[b, :, h].double(), k[b, :, hk].double(), v[b, :, hk].double(), do[b, :, h].double(), vis, scale, dt)
            _near(dq[b, :, h], r[0], r[3], f"dq row {b} head {h}")
            rk, rv, tk, tv = rk + r[1], rv + r[2], tk + r[4], tv + r[5]
        _near(dk[b, :, hk], rk, tk + 1.05 * u * rk.abs() + A.TINY[dt], f"dk row {b} head {hk}")
        _near(dv[b, :, hk], rv, tv + 1.05 * u * rv.abs() + A.TINY[dt], f"dv row {b} head {hk}")


@pytest.mark.parametrize("dt,D", FORMS)
@pytest.mark.parametrize("window", [None, 700])
def test_paged(dev, dt, D, window):
    """Prompts over cached tokens: more than 512 workgroups of 128 rows."""
    new, lens = [900, 1, 0, 1150], [1500, 300, 20, 1150]
    Hq, Hkv = 32, 8
    kc, vc, pt, sl, cu, ks, vs = _paged(5, new, lens, Hkv, D, 32, dt, dev)
    q = _rows(6, sum(new), Hq, D, dt=dt)
    out, lse = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu, window=window, return_lse=True)
    at = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        vis = A.visible(n, m, m - n, None, window)
        for h in (0, 13, 31):
            for s in (slice(0, min(n, 50)), slice(n // 2, min(n // 2 + 60, n)), slice(max(n - 40, 0), n)):
                x, kk = q[at:at + n][s, h].double(), ks[b][:, h // 4].double()
                ref, l, tol = A.attend(x, kk, vs[b][:, h // 4].double(), vis[s], 1.0 / math.sqrt(D), dt)
                _near(out[at:at + n][s, h], ref, tol, f"sequence {b} head {h}")
                _near(lse[at:at + n][s, h], l, 4 * A.f32_error(x, kk, 1.0 / math.sqrt(D), torch.zeros(1)) + 1e-6 * l.abs(), "lse")
        at += n
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dt,D", [("bf16", 256), ("f16", 256), ("f32", 128), ("bf16", 128)])
def test_paged_hidden_infinities_and_far_scores(dev, dt, D):
    """In one of many sequences: later tokens that are not finite, and scores
    beyond the range of exponents."""
    new, lens = [600] * 6, [800] * 6
    Hq, Hkv = 32, 8
    kc, vc, pt, sl, cu, ks, vs = _paged(7, new, lens, Hkv, D, 16, dt, dev, junk=math.nan)
    q = _rows(8, sum(new), Hq, D, dt=dt)
    q[700:710, :, 0] = 100.0   # sequence 1, from its 100th new token on
    page, place = int(pt[1, 40 // 16]), 40 % 16
    kc[page, place] = 0
    kc[page, place, :, 0] = 80.0
    ks[1][40] = 0
    ks[1][40, :, 0] = 80.0
    base = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu)
    for h in (0, 31):
        s = slice(90, 130)
        vis = A.visible(600, 800, 200)[s]
        ref, _, tol = A.attend(q[600:1200][s, h].double(), ks[1][:, h // 4].double(), vs[1][:, h // 4].double(), vis, 1.0 / math.sqrt(D), dt)
        _near(base[600:1200][s, h], ref, tol, f"head {h}")
    vc[int(pt[1, 500 // 16]), 500 % 16] = math.inf   # its 301st new token
    out = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu)
    keep = torch.ones(len(q), dtype=torch.bool, device=dev)
    keep[900:1200] = False
    assert torch.equal(out[keep], base[keep]) and not torch.isfinite(out[~keep]).any()
