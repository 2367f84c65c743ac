"""Positions that the rotary table does not cover, in the call that stores new tokens."""

import pytest
import torch

from deltanet_tpu_amd import paged_qkv_append, rotary_table
from tests.test_attention_gpu import _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,R,normed,pos_dtype", [(128, 64, True, torch.int32), (64, 64, False, torch.int64), (80, 20, True, torch.int64), (6, 2, False, torch.int32)])
def test_positions_past_the_table(dev, dt, D, R, normed, pos_dtype):
    """Not numbers in the rotated channels of query and stored key, the others as they are;
    a negative position is no token at all."""
    N, Hq, Hkv, page, rows = 7, 4, 2, 4, 50
    q, k, v = (_rows(s, N, h, D, dt=dt).to(dev) for s, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    w = dict(q_weight=_rows(4, D, dt=dt).to(dev), k_weight=_rows(5, D, dt=dt).to(dev)) if normed else {}
    table = rotary_table(rows, R, device=dev)
    far = [3, rows - 1, rows, 2 ** 31 - 1, -1, -(2 ** 31), 0]
    if pos_dtype is torch.int64:
        far[3] = 1 << 40
    slots = torch.arange(N, device=dev)
    calls = []
    for pos in (far, [min(max(p, 0), rows - 1) for p in far]):
        kc, vc = (torch.full((2, page, Hkv, D), 9.0, dtype=k.dtype, device=dev) for _ in range(2))
        out = paged_qkv_append(q, k, v, kc, vc, slots, torch.tensor(pos, dtype=pos_dtype, device=dev), table=table, **w)
        calls.append((out, kc.flatten(0, 1)[:N], vc.flatten(0, 1)[:N]))
    (out, kn, vn), (out2, kn2, vn2) = calls
    for i, p in enumerate(far):
        if p < 0:
            assert not out[i].any() and bool((kn[i] == 9.0).all()) and bool((vn[i] == 9.0).all())
            continue
        assert torch.equal(vn[i], v[i]) and torch.equal(vn[i], vn2[i])
        for a, b in ((out[i], out2[i]), (kn[i], kn2[i])):
            assert torch.equal(a[:, R:], b[:, R:])
            assert bool(torch.isnan(a[:, :R]).all()) if p >= rows else torch.equal(a, b)
