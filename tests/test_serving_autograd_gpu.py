"""Normed heads and the serving operators next to autograd: derivatives that would be
dropped are refused, caches count their stores, inference tensors are taken."""

import pytest
import torch
from torch.autograd import forward_ad

from deltanet_tpu_amd import (
    norm_rotary, page_pool, paged_kv_keep, paged_qkv_append, paged_reserve, paged_slots, paged_tree_attention)

pytestmark = pytest.mark.gpu


def _state(dev):
    r = lambda *s: torch.randn(*s, device=dev)
    return dict(q=r(2, 2, 64), k=r(2, 1, 64), v=r(2, 1, 64), kc=r(4, 16, 1, 64), vc=r(4, 16, 1, 64), wq=r(64), wk=r(64),
                slots=torch.arange(2, device=dev), pos=torch.zeros(2, dtype=torch.int32, device=dev),
                pt=torch.arange(2, dtype=torch.int32, device=dev)[:, None].contiguous(), lens=torch.tensor([5, 9], dtype=torch.int32, device=dev),
                vis=torch.ones(2, 1, dtype=torch.int64, device=dev), kept=torch.tensor([[1], [-1]], dtype=torch.int32, device=dev))


def _append(s):
    return paged_qkv_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["pos"], q_weight=s["wq"], k_weight=s["wk"])


def _tree(s):
    return paged_tree_attention(s["q"], s["kc"], s["vc"], s["pt"], s["lens"], s["vis"])


def _keep(s):
    return paged_kv_keep(s["kc"], s["vc"], s["pt"], s["lens"], s["kept"])


CALLS = [(_append, ["q", "k", "v", "kc", "vc", "wq", "wk"]), (_tree, ["q", "kc", "vc"]), (_keep, ["kc", "vc"])]


@pytest.mark.parametrize("call,names", CALLS)
def test_serving_calls_refuse_derivatives(dev, call, names):
    for n in names:
        s = _state(dev)
        s[n] = s[n].requires_grad_(True)
        with pytest.raises(ValueError, match="not differentiable"):
            call(s)
        with torch.no_grad():
            call(s)
        s = _state(dev)
        with forward_ad.dual_level():
            s[n] = forward_ad.make_dual(s[n], torch.ones_like(s[n]))
            with pytest.raises(ValueError, match="not differentiable"):
                call(s)


def test_tangents_of_normed_heads_are_refused(dev):
    s = _state(dev)
    for n in ("q", "wq"):
        with forward_ad.dual_level():
            x = dict(s)
            x[n] = forward_ad.make_dual(x[n], torch.ones_like(x[n]))
            with pytest.raises((RuntimeError, NotImplementedError)):
                norm_rotary(x["q"], None, x["wq"], None)


def test_stores_are_counted(dev):
    s = _state(dev)
    for call in (_append, _keep):
        before = s["kc"]._version, s["vc"]._version
        call(s)
        assert s["kc"]._version > before[0] and s["vc"]._version > before[1]
    pool, held, table = page_pool(5, device=dev), torch.zeros(2, dtype=torch.int32, device=dev), s["pt"]
    before = pool._version, held._version, table._version
    paged_reserve(pool, table, held, s["lens"], page_size=16)
    assert all(t._version > x for t, x in zip((pool, held, table), before))


def test_inference_tensors(dev):
    want = _state(dev)
    with torch.inference_mode():
        s = {n: t.clone() for n, t in want.items()}
        pool, held = page_pool(5, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    for x in (want, s):
        x["out"] = [_append(x), _tree(x), _keep(x)]
    assert all(torch.equal(a, b) for a, b in zip(want["out"], s["out"])) and torch.equal(want["kc"], s["kc"]) and torch.equal(want["vc"], s["vc"])
    assert not paged_reserve(pool, s["pt"], held, s["lens"], page_size=16).any() and int(pool[0]) == 3
    paged_slots(s["pt"], s["lens"], 2, page_size=16)


def test_inputs_changed_before_the_backward(dev):
    """An input that is written between forward and backward is found, as elsewhere."""
    x, w = torch.randn(3, 2, 64, device=dev), torch.ones(64, device=dev, requires_grad=True)
    y, _ = norm_rotary(x, None, w, None)
    x.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_some_leaves_alone(dev):
    """Gradients of the weights with frozen inputs, and of the inputs with frozen weights."""
    x, w, dz = torch.randn(5, 2, 64, device=dev), torch.randn(64, device=dev), torch.randn(5, 2, 64, device=dev)
    full = [t.clone().requires_grad_(True) for t in (x, w)]
    want = torch.autograd.grad(norm_rotary(full[0], None, full[1], None)[0], full, dz)
    for i, (a, b) in enumerate(((full[0], w), (x, full[1]))):
        got, = torch.autograd.grad(norm_rotary(a, None, b, None)[0], full[i], dz)
        assert torch.equal(got, want[i])
