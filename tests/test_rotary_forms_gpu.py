"""The rotation and the append on either side of the size from which a thread takes
several heads, against float64."""

import pytest
import torch

from deltanet_tpu_amd import apply_rotary, paged_kv_append, rotary_table
from tests import attn_ref as A
from tests.test_rotary_gpu import _cache, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,inter", [("bf16", False), ("f16", True), ("f32", False), ("f32", True)])
@pytest.mark.parametrize("N,Hq,Hk", [(8192, 12, 4), (8191, 12, 4), (8193, 12, 4), (9001, 14, 1)])   # of 128 channels: 2^24 elements, ...
def test_rotary_at_many_elements(dev, dt, inter, N, Hq, Hk):
    D, R = 128, 64
    g = torch.Generator().manual_seed(N)
    q, k = (torch.randn(1, N, h, D, generator=g).to(A.DT[dt]) for h in (Hq, Hk))
    pos = torch.randint(0, 500, (1, N), generator=g)
    table = rotary_table(500, R, device=dev)
    qd = q.to(dev).requires_grad_(True)
    qo, ko = apply_rotary(qd, k.to(dev), pos.to(dev), table, interleaved=inter)
    for x, y in ((q, qo), (k, ko)):
        x = x[0].double()
        _near(y[0], A.rotate(x, pos[0], table.cpu(), inter), A.rotate_tolerance(x, dt, R))
    (dq,) = torch.autograd.grad(qo, qd, q.to(dev))
    x = q[0].double()
    _near(dq[0], A.rotate(x, pos[0], table.cpu(), inter, -1.0), A.rotate_tolerance(x, dt, R))


@pytest.mark.parametrize("dt,cdt,inter,R,hf", [("bf16", "bf16", False, 128, False), ("f32", "bf16", True, 64, True), ("f16", "f32", False, 0, False),
                                              ("bf16", "f16", True, 128, True), ("f32", "f32", False, 32, False)])
@pytest.mark.parametrize("H,N", [(8, 8200), (4, 16400), (12, 5500), (6, 12000)])   # (heads by four, and not)
def test_append_of_many_tokens(dev, dt, cdt, inter, R, hf, H, N):
    """Four rows (keys, then values) of a token per thread."""
    D, page, B = 128, 16, 3
    new = [N - 5000, 4999, 1]
    old = [7, 0, 100]
    lens = [a + b for a, b in zip(new, old)]
    g = torch.Generator().manual_seed(H)
    k, v = (torch.randn(N, H, D, generator=g).to(A.DT[dt]) for _ in range(2))
    counts = [-(-x // page) for x in lens]
    order = torch.randperm(sum(counts), generator=g).to(torch.int32)
    pt = torch.full((B, max(counts)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        pt[b, :n] = order[at:at + n]
        at += n
    table = rotary_table(max(lens), R, device=dev) if R else None
    kc, vc = (_cache(sum(counts), page, H, D, A.DT[cdt], dev, hf) for _ in range(2))
    cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32)
    paged_kv_append(k.to(dev), v.to(dev), kc, vc, pt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), cu_seqlens=cu.to(dev),
                    table=table, interleaved=inter)
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new))
    pos = torch.cat([torch.arange(o, o + n) for n, o in zip(new, old)])
    pg, place = pt[seq, pos // page].long(), pos % page
    kr = A.rotate(k.double(), pos, table.cpu(), inter) if R else k.to(A.DT[cdt]).double()
    _near(kc[pg.to(dev), place.to(dev)], kr, A.rotate_tolerance(k.double(), cdt, R) if R else torch.zeros(()), "keys")
    assert torch.equal(vc[pg.to(dev), place.to(dev)].cpu(), v.to(A.DT[cdt]))
    rest = torch.ones(sum(counts), page, dtype=torch.bool)
    rest[pg, place] = False
    assert (kc[rest.to(dev)] == 7.0).all() and (vc[rest.to(dev)] == 7.0).all()
