"""Calls of the attention operators at the edges of what they take."""

import math

import pytest
import torch

from deltanet_tpu_amd import apply_rotary, causal_attention, paged_attention, paged_kv_append, rotary_table
from tests import attn_ref as A
from tests.test_attention_backward_gpu import _grads, _inputs
from tests.test_attention_gpu import _check_paged, _check_rows, _near, _paged, _rows
from tests.test_attention_placement_gpu import _wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_cotangent_off_16_bytes(dev, dt):
    """A concatenation hands its operands slices of one cotangent: contiguous, on
    any element."""
    q, k, v, do = (t.to(dev) for t in _inputs(1, 70, 2, 1, 64, dt))
    want = _grads(dev, q, k, v, do)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = causal_attention(*x)
    whole = torch.cat([torch.zeros(3, dtype=q.dtype, device=dev), out.flatten()])
    got = torch.autograd.grad(whole, x, torch.cat([torch.ones(3, dtype=q.dtype, device=dev), do.flatten()]))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("wide", [False, True])
def test_windows_past_every_key(dev, wide, window):
    """A window that reaches past the first token is no window, for tokens of
    positions below 0 next to others too."""
    new, lens = [30, 1, 6, 1], [12, 700, 3, 0]
    kc, vc, pt, sl, cu, ks, vs = _paged(9, new, lens, 2, 128, 16, "bf16", dev)
    if wide:
        pt = _wide(pt, 16)
    q = _rows(10, sum(new), 8, 128)
    out = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu, window=window)
    _check_paged(out, None, q, ks, vs, new, lens, "bf16")
    assert torch.equal(out, paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu))
    q, k, v, do = (t.to(dev) for t in _inputs(1, 150, 2, 1, 64, "bf16"))
    assert torch.equal(causal_attention(q, k, v, window=window), causal_attention(q, k, v))
    for a, b in zip(_grads(dev, q, k, v, do, window=window), _grads(dev, q, k, v, do)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("wide", [False, True])
def test_window_of_the_capacity(dev, wide):
    """The longest windows that hide something, at the cache's end and one token off."""
    new, lens = [1, 2, 40], [320, 319, 320]
    kc, vc, pt, sl, cu, ks, vs = _paged(9, new, lens, 1, 64, 16, "bf16", dev)
    pt = _wide(pt, 16) if wide else pt[:, :20].contiguous()
    q = _rows(10, sum(new), 4, 64)
    for window in (318, 319, 320, 321):
        _check_paged(paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu, window=window), None, q, ks, vs, new, lens, "bf16", window)
    q, k, v = (_rows(s, 1, 150, 2, 64) for s in (1, 2, 3))
    for window in (148, 149, 150, 151):
        _check_rows(causal_attention(q.to(dev), k.to(dev), v.to(dev), window=window), None, q, k, v, "bf16", None, window)


@pytest.mark.parametrize("before,after", [(0, 9), (3, 0), (40, 700), (1, 1)])
@pytest.mark.parametrize("new,lens", [([1, 2, 1], [900, 30, 2]), ([70, 0, 130], [70, 9, 500]), ([0, 0], [4, 0])])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f32", 64), ("f16", 256)])
def test_tokens_of_no_sequence(dev, dt, D, wide, new, lens, before, after):
    """Tokens in front of cu_seqlens[0] and from cu_seqlens[-1] on get zeros (lse
    -inf) whatever the memory of the result held; the others are what they are."""
    kc, vc, pt, sl, cu, ks, vs = _paged(3, new, lens, 2, D, 16, dt, dev)
    if wide:
        pt = _wide(pt, 16)
    n = sum(new)
    q = _rows(4, before + n + after, 4, D, dt=dt)
    full = lambda: (torch.full(q.shape, math.nan, dtype=q.dtype, device=dev), torch.full(q.shape[:2], math.nan, device=dev))
    del [full()][:]   # (what the allocator hands out next)
    out, lse = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu + before, return_lse=True)
    mid = slice(before, before + n)
    _check_paged(out[mid], lse[mid], q[mid], ks, vs, new, lens, dt)
    for s in (slice(0, before), slice(before + n, None)):
        assert not out[s].any() and (lse[s] == -math.inf).all()


def test_forward_mode_tangents_are_refused(dev):
    """A tangent that would be dropped raises; inputs without one work beside it."""
    import torch.autograd.forward_ad as fwd
    q, k, v, t = (torch.randn(1, 9, 2, 64, device=dev) for _ in range(4))
    table, pos = rotary_table(16, 32, device=dev), torch.arange(9, device=dev)
    kc, vc = (torch.randn(2, 16, 2, 64, device=dev) for _ in range(2))
    pt, sl = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.full((1,), 9, dtype=torch.int32, device=dev)
    want = causal_attention(q, k, v), apply_rotary(q, k, pos, table), paged_attention(q, kc, vc, pt, sl)
    with fwd.dual_level():
        dual = lambda x: fwd.make_dual(x, t)
        for x in ((dual(q), k, v), (q, dual(k), v), (q, k, dual(v))):
            with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                causal_attention(*x)
        for x in ((dual(q), k), (q, dual(k)), (dual(q), None)):
            with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                apply_rotary(*x, pos, table)
        with pytest.raises(ValueError, match="not differentiable"):
            paged_attention(dual(q), kc, vc, pt, sl)
        with pytest.raises(ValueError, match="not differentiable"):
            paged_kv_append(dual(k), v, kc, vc, pt, sl)
        assert torch.equal(causal_attention(q, k, v), want[0])
        assert torch.equal(apply_rotary(q, k, pos, table)[1], want[1][1])
        assert torch.equal(paged_attention(q, kc, vc, pt, sl), want[2])


def test_tangents_of_cotangents_are_refused(dev):
    """Forward over reverse: the gradient of a dual cotangent."""
    import torch.autograd.forward_ad as fwd
    q = torch.randn(1, 9, 2, 64, device=dev, requires_grad=True)
    w, t = torch.randn(1, 9, 2, 64, device=dev), torch.randn(1, 9, 2, 64, device=dev)
    table, pos = rotary_table(16, 32, device=dev), torch.arange(9, device=dev)
    for f in (lambda: causal_attention(q, q, q), lambda: apply_rotary(q, None, pos, table)[0]):
        want, = torch.autograd.grad(f(), q, w)
        with fwd.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError), match="forward"):
                torch.autograd.grad(f(), q, fwd.make_dual(w, t))
            assert torch.equal(torch.autograd.grad(f(), q, w)[0], want)


def test_caches_that_require_grad_are_refused(dev):
    """Attention over a cache that requires grad, or a store in it, would lose it."""
    q, k = torch.randn(1, 4, 64, device=dev), torch.randn(1, 2, 64, device=dev)
    kc, vc = (torch.randn(2, 16, 2, 64, device=dev) for _ in range(2))
    pt, sl = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    g = lambda c: c.clone().requires_grad_(True)
    for caches in ((g(kc), vc), (kc, g(vc))):
        with pytest.raises(ValueError, match="not differentiable"):
            paged_attention(q, *caches, pt, sl)
        with pytest.raises(ValueError, match="not differentiable"):
            paged_kv_append(k, k, *caches, pt, sl)
        with torch.no_grad():
            paged_attention(q, *caches, pt, sl)
            paged_kv_append(k, k, *caches, pt, sl)


def test_caches_with_tangents_are_refused(dev):
    import torch.autograd.forward_ad as fwd
    q, k = torch.randn(1, 4, 64, device=dev), torch.randn(1, 2, 64, device=dev)
    kc, vc = (torch.randn(2, 16, 2, 64, device=dev) for _ in range(2))
    pt, sl = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    with fwd.dual_level():
        dual = fwd.make_dual(kc, torch.ones_like(kc))
        with pytest.raises(ValueError, match="not differentiable"):
            paged_attention(q, dual, vc, pt, sl)
        with pytest.raises(ValueError, match="not differentiable"):
            paged_kv_append(k, k, dual, vc, pt, sl)


def test_append_is_seen_as_a_write(dev):
    """What autograd has kept of a cache is out of date after a store in it; caches
    made in inference mode are stored in too."""
    k = torch.randn(1, 2, 64, device=dev)
    kc, vc = (torch.randn(2, 16, 2, 64, device=dev) for _ in range(2))
    pt, sl = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    w = torch.ones((), device=dev, requires_grad=True)
    for c in (kc, vc):
        y = (c * w).sum()
        paged_kv_append(k, k, kc, vc, pt, sl)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        kc, vc = (torch.zeros(2, 16, 2, 64, device=dev) for _ in range(2))
        paged_kv_append(k, k, kc, vc, pt, sl)
    paged_kv_append(k, 2 * k, kc, vc, pt, sl)
    assert torch.equal(kc[0, 0], k[0]) and torch.equal(vc[0, 0], 2 * k[0])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 5])
def test_keys_that_cannot_be_chosen(dev, dt, n):
    """Scores of -inf have no weight; a query that sees no other key has no result,
    the same in the kernels of few and of many rows, in one workgroup or several."""
    new, lens = [n, n, 1], [40, 1500, 0]
    kc, vc, pt, sl, cu, ks, vs = _paged(3, new, lens, 1, 64, 16, dt, dev)
    q = _rows(4, sum(new), 2, 64, dt=dt)
    q[..., 0] = 1.0
    kc[pt[0, :3].long(), :, :, 0] = -math.inf                     # all of sequence 0
    for at in (3, 700, 1499):                                     # some of sequence 1
        kc[int(pt[1, at // 16]), at % 16, :, 0] = -math.inf
    for table in (pt, _wide(pt, 16)):
        out, lse = paged_attention(q.to(dev), kc, vc, table, sl, cu_seqlens=cu, return_lse=True)
        assert torch.isnan(out[:n]).all() and not torch.isfinite(lse[:n]).any()
        assert not out[2 * n:].any()
        vis = A.visible(n, 1500, 1500 - n)
        vis[:, [3, 700, 1499]] = False
        for h in range(2):
            ref, _, tol = A.attend(q[n:2 * n, h].double(), ks[1][:, 0].double(), vs[1][:, 0].double(), vis, 0.125, dt)
            _near(out[n:2 * n, h], ref, tol, f"head {h}")
    big = torch.full((1, 200, 1, 64), -math.inf, dtype=A.DT[dt], device=dev)   # (every row, whole rows)
    one = torch.ones(1, 200, 2, 64, dtype=A.DT[dt], device=dev)
    assert torch.isnan(causal_attention(one, big, one[:, :, :1])).all()
