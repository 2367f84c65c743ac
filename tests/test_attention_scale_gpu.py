"""Attention with a scale of 0 and below: the softmax over -|scale| q k and over
equal scores, forward and backward, over rows and over a paged cache."""

import pytest
import torch

from deltanet_tpu_amd import causal_attention, paged_attention
from tests import attn_ref as A
from tests.test_attention_backward_gpu import _check, _grads, _inputs
from tests.test_attention_gpu import _check_paged, _check_rows, _paged, _rows
from tests.test_attention_placement_gpu import _wide

pytestmark = pytest.mark.gpu
SCALES = [0.0, -0.0, -0.125, -1.0, -2.0 ** -100, 714 * 2.0 ** -149]   # float32 numbers, as the kernels take them


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dt,D", [("bf16", 64), ("f16", 128), ("f32", 64), ("bf16", 256)])
def test_rows(dev, dt, D, scale):
    B, L, Hq, Hkv = 2, 150, 4, 2
    q, k, v = _rows(1, B, L, Hq, D, dt=dt), _rows(2, B, L, Hkv, D, dt=dt), _rows(3, B, L, Hkv, D, dt=dt)
    out, lse = causal_attention(q.to(dev), k.to(dev), v.to(dev), scale=scale, return_lse=True)
    _check_rows(out, lse, q, k, v, dt, scale=scale)
    seg = torch.tensor([0] * 40 + [1] * 60 + [2] * 50)
    out = causal_attention(q.to(dev), k.to(dev), v.to(dev), scale=scale, segment_ids=seg.to(dev), window=33)
    _check_rows(out, None, q, k, v, dt, [A.starts_of(seg.tolist())] * B, 33, scale)


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_rows_negative_scale_far_scores(dev, dt):
    """Scores far above and far below a query's own once their sign is turned."""
    B, L, H, D = 1, 300, 2, 64
    q, k, v = (_rows(s, B, L, H, D, dt=dt, scale=4.0 if s < 3 else 1.0) for s in (1, 2, 3))
    out = causal_attention(q.to(dev), k.to(dev), v.to(dev), scale=-1.0)
    _check_rows(out, None, q, k, v, dt, scale=-1.0)


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_paged(dev, dt, wide, scale):
    new, lens = [1, 5, 0, 40, 2], [700, 60, 9, 300, 1]
    kc, vc, pt, sl, cu, ks, vs = _paged(9, new, lens, 2, 128, 16, dt, dev)
    q = _rows(10, sum(new), 4, 128, dt=dt)
    out, lse = paged_attention(q.to(dev), kc, vc, _wide(pt, 16) if wide else pt, sl, cu_seqlens=cu, scale=scale, return_lse=True)
    _check_paged(out, lse, q, ks, vs, new, lens, dt, scale=scale)


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("dt,D", [("bf16", 128), ("f32", 64)])
def test_gradients(dev, dt, D, scale):
    q, k, v, do = _inputs(1, 200, 4, 2, D, dt)
    _check(_grads(dev, q, k, v, do, scale=scale), q, k, v, do, dt, scale=scale)
