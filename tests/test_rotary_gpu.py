"""Rotary positions and the paged cache's append on the GPU against float64."""

import math

import pytest
import torch

from deltanet_tpu_amd import apply_rotary, paged_kv_append, rotary_table
from tests import attn_ref as A

pytestmark = pytest.mark.gpu


def _near(got, ref, tol, tag=""):
    d = (got.detach().double().cpu() - ref).abs()
    assert bool((d <= tol).all()), f"{tag}: off by {float(d.max()):.3e}, {int((d > tol).sum())} elements outside"


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,R", [(256, 64), (128, 128), (64, 32), (48, 16), (80, 20), (6, 2), (16, 16)])
def test_rotary_matches_float64(dev, dt, inter, D, R):
    B, L, Hq, Hk = 2, 37, 6, 2
    g = torch.Generator().manual_seed(D + R)
    q = torch.randn(B, L, Hq, D, generator=g).to(A.DT[dt])
    k = torch.randn(B, L, Hk, D, generator=g).to(A.DT[dt])
    pos = torch.randint(0, 500, (B, L), generator=g)
    table = rotary_table(500, R, device=dev)
    qo, ko = apply_rotary(q.to(dev), k.to(dev), pos.to(dev), table, interleaved=inter)
    for x, y in ((q, qo), (k, ko)):
        assert y.dtype == x.dtype and y.is_contiguous()
        x = x.double().flatten(0, 1)
        ref = A.rotate(x, pos.flatten(), table.cpu(), inter)
        _near(y.flatten(0, 1), ref, A.rotate_tolerance(x, dt, R), f"D={D} R={R}")
        assert torch.equal(y.flatten(0, 1)[..., R:].cpu().double(), x[..., R:])


def test_rotary_many_tokens_strided_and_shared_positions(dev):
    """Enough tokens for four heads per thread; q and k are slices of one
    projection; one row of positions for every batch row."""
    B, L, Hq, Hk, D, R = 3, 5000, 6, 3, 128, 64
    x = torch.randn(B, L, Hq + 2 * Hk, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    q, k = x[:, :, :Hq], x[:, :, Hq:Hq + Hk]
    pos = torch.arange(L, dtype=torch.int32).flip(0)
    table = rotary_table(L, R, device=dev)
    qo, ko = apply_rotary(q, k, pos.to(dev), table)
    for a, b in ((q, qo), (k, ko)):
        a = a.cpu().double().flatten(0, 1)
        _near(b.flatten(0, 1), A.rotate(a, pos.long().repeat(B), table.cpu()), A.rotate_tolerance(a, "bf16", R))
    # rank 3, batch-strided views, no k, int64 positions with a stride
    pos2 = torch.arange(2 * L, device=dev)[::2] % L
    qo2, none = apply_rotary(q[1], None, pos2, table)
    assert none is None
    a = q[1].cpu().double()
    _near(qo2, A.rotate(a, pos2.cpu(), table.cpu()), A.rotate_tolerance(a, "bf16", R))
    # channels that are not contiguous and rows that are not on 16 bytes
    y = torch.randn(40, 3, D + 1, generator=torch.Generator().manual_seed(2)).to(dev)
    for z in (y[..., 1:], y[..., :D].transpose(1, 2).contiguous().transpose(1, 2)):
        out, _ = apply_rotary(z, None, torch.arange(40, device=dev), table)
        a = z.cpu().double()
        _near(out, A.rotate(a, torch.arange(40), table.cpu()), A.rotate_tolerance(a, "f32", R))


def test_rotary_positions_outside_the_table(dev):
    table = rotary_table(8, 32, device=dev)
    q = torch.randn(4, 2, 64, device=dev)
    out, _ = apply_rotary(q, None, torch.tensor([-1, 0, 7, 8], device=dev), table)
    assert torch.isnan(out[0, :, :32]).all() and torch.isnan(out[3, :, :32]).all()
    assert torch.equal(out[..., 32:], q[..., 32:]) and torch.equal(out[1], q[1])
    assert torch.isfinite(out[2]).all()
    q0 = torch.randn(0, 2, 64, device=dev)
    assert apply_rotary(q0, q0, torch.zeros(0, dtype=torch.int32, device=dev), table)[0].shape == (0, 2, 64)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_rotary_gradient(dev, inter, dt):
    """The gradient is the transposed rotation; and central differences of a
    weighted sum in float32 agree along a random direction."""
    B, L, H, D, R = 2, 9, 2, 64, 48
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(B, L, H, D, generator=g).to(A.DT[dt]) for _ in range(2))
    wq, wk = (torch.randn(B, L, H, D, generator=g).to(A.DT[dt]) for _ in range(2))
    pos = torch.randint(0, 64, (B, L), generator=g)
    table = rotary_table(64, R, device=dev, scaling={"type": "yarn", "factor": 4.0, "original_max_position": 16})
    qd, kd = (t.to(dev).requires_grad_(True) for t in (q, k))
    qo, ko = apply_rotary(qd, kd, pos.to(dev), table, interleaved=inter)
    dq, dk = torch.autograd.grad((qo, ko), (qd, kd), (wq.to(dev), wk.to(dev)))
    for w, d in ((wq, dq), (wk, dk)):
        x = w.double().flatten(0, 1)
        _near(d.flatten(0, 1), A.rotate(x, pos.flatten(), table.cpu(), inter, -1.0), 1.2 * A.rotate_tolerance(x, dt, R))
    # only one of the two outputs used
    (dk2,) = torch.autograd.grad(apply_rotary(qd, kd, pos.to(dev), table, interleaved=inter)[1], kd, wk.to(dev))
    assert torch.equal(dk2, dk)
    if dt == "f32":
        u = torch.randn(B, L, H, D, generator=g).to(dev)
        f = lambda s: (apply_rotary(qd.detach() + s * u, None, pos.to(dev), table, interleaved=inter)[0].double() * wq.to(dev)).sum()
        diff = float((f(0.5) - f(-0.5)))   # linear: the step does not matter
        assert abs(diff - float((dq.double() * u).sum())) <= 1e-5 * float((dq * u).abs().sum())


def test_rotary_table_scaling(dev):
    base = rotary_table(32, 16, device=dev).cpu().double()
    i = torch.arange(0, 16, 2, dtype=torch.float64)
    f = 10000.0 ** (-i / 16)
    p = torch.arange(32, dtype=torch.float64)[:, None]
    assert (base - torch.cat([torch.cos(p * f), torch.sin(p * f)], 1)).abs().max() <= 2.0 ** -24
    lin = rotary_table(32, 16, device=dev, scaling={"type": "linear", "factor": 4}).cpu()
    assert torch.equal(lin[::4], base[:8].float())
    ntk = rotary_table(32, 16, device=dev, scaling={"type": "ntk", "factor": 4}).cpu().double()
    f2 = f * 4.0 ** (-i / 14)   # the fastest kept, the slowest divided by 4
    assert (ntk - torch.cat([torch.cos(p * f2), torch.sin(p * f2)], 1)).abs().max() <= 2.0 ** -24
    yarn = rotary_table(32, 16, device=dev, scaling={"type": "yarn", "factor": 4, "original_max_position": 4096}).cpu().double()
    gain = 0.1 * math.log(4) + 1
    assert (yarn[:, 0] - gain * base[:, 0]).abs().max() <= 1e-6          # turns 652 times: kept
    assert (yarn[:, 7] - gain * torch.cos(p[:, 0] * f[7] / 4)).abs().max() <= 1e-6   # less than once: divided


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def _cache(pages, page, H, D, dtype, dev, heads_first, fill=7.0):
    if heads_first:
        return torch.full((pages, H, page, D), fill, dtype=dtype, device=dev).transpose(1, 2)
    return torch.full((pages, page, H, D), fill, dtype=dtype, device=dev)


@pytest.mark.parametrize("dt,cdt", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("D,R,page,inter,hf", [(128, 128, 16, False, False), (256, 64, 64, True, True), (64, 0, 1, False, False),
                                              (40, 12, 32, True, False), (48, 16, 8, False, True)])
def test_append_ragged(dev, dt, cdt, D, R, page, inter, hf):
    new, old, H = [5, 0, 1, 70, 3], [0, 9, 31, 10, 64], 3
    lens = [a + b for a, b in zip(new, old)]
    N, most = sum(new), max(-(-x // page) for x in lens)
    pages = sum(-(-x // page) for x in lens) + 1
    g = torch.Generator().manual_seed(5)
    order = torch.randperm(pages, generator=g).tolist()
    pt = torch.full((len(new), most), -1, dtype=torch.int32)
    for b, x in enumerate(lens):
        for i in range(-(-x // page)):
            pt[b, i] = order.pop()
    fused = torch.randn(N, 2 * H, D, generator=g).to(A.DT[dt])
    k, v = fused[:, :H], fused[:, H:]
    table = rotary_table(max(lens), R, device=dev) if R else None
    kc, vc = (_cache(pages, page, H, D, A.DT[cdt], dev, hf) for _ in range(2))
    cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32)
    fd = fused.to(dev)
    r = paged_kv_append(fd[:, :H], fd[:, H:], kc, vc, pt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                        cu_seqlens=cu.to(dev), table=table, interleaved=inter)
    assert r[0] is kc and r[1] is vc
    kref, vref = (torch.full((pages, page, H, D), 7.0, dtype=torch.float64) for _ in range(2))
    ktol = torch.zeros_like(kref)
    pos = torch.cat([torch.arange(o, o + n) for n, o in zip(new, old)])
    kr = A.rotate(k.double(), pos, table.cpu(), inter) if R else k.to(A.DT[cdt]).double()
    i = 0
    for b, (n, o) in enumerate(zip(new, old)):
        for t in range(n):
            at = int(pt[b, (o + t) // page]), (o + t) % page
            kref[at], vref[at] = kr[i], v[i].to(A.DT[cdt]).double()
            ktol[at] = A.rotate_tolerance(k[i].double(), cdt, R) if R else 0.0
            i += 1
    _near(kc, kref, ktol, "keys")
    assert torch.equal(vc.cpu().double(), vref)


def test_append_uniform_and_out_of_range(dev):
    """(B, T, H, D) and (B, H, D) without cu_seqlens, batch-strided views; tokens
    that have no place are left out and nothing else is touched."""
    B, T, H, D, page = 3, 4, 2, 64, 4
    x = torch.randn(B, T + 2, H, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(dev)
    k, v = x[:, :T], x[:, 2:]
    pt = torch.tensor([[0, 1], [2, 99], [3, -5]], dtype=torch.int32, device=dev)
    lens = torch.tensor([4, 6, 10], dtype=torch.int32, device=dev)   # row 2: positions 6 .. 9, two pages only
    kc, vc = (_cache(5, page, H, D, torch.bfloat16, dev, False) for _ in range(2))
    paged_kv_append(k, v, kc, vc, pt, lens)
    want = torch.full_like(kc, 7.0)
    want[0, 0:4] = k[0]
    want[2, 2:4] = k[1, 0:2]        # positions 2, 3; 4, 5 are on page 99
    assert torch.equal(kc, want)
    lens0 = torch.tensor([1, 2, 3], dtype=torch.int32, device=dev)   # some positions are negative
    kc.fill_(7.0)
    paged_kv_append(k, v, kc, vc, pt, lens0)
    want.fill_(7.0)
    want[0, 0], want[2, 0:2], want[3, 0:3] = k[0, 3], k[1, 2:], k[2, 1:]
    assert torch.equal(kc, want)
    one = torch.randn(B, H, D, device=dev).to(torch.bfloat16)
    paged_kv_append(one, one, kc, vc, pt, torch.tensor([1, 1, 1], dtype=torch.int32, device=dev))
    assert torch.equal(kc[[0, 2, 3], 0], one) and torch.equal(vc[[0, 2, 3], 0], one)


@pytest.mark.parametrize("parts", ["q", "k", "both", "q alone"])
def test_rotary_gradient_of_some_and_of_the_gradient(dev, parts):
    """A gradient of one result only, and the gradient of the gradient: the rotation
    is linear, so that this is the rotation of what is put in again, to the bit."""
    table = rotary_table(16, 32, device=dev)
    pos = torch.arange(5, device=dev)
    q = torch.randn(2, 5, 3, 64, device=dev, requires_grad=True)
    k = None if parts == "q alone" else torch.randn(2, 5, 1, 64, device=dev, requires_grad=True)
    yq, yk = apply_rotary(q, k, pos, table)
    wq = torch.randn_like(q).requires_grad_(True)
    wk = None if k is None else torch.randn_like(k).requires_grad_(True)
    loss = (yq * wq).sum() if parts != "k" else 0.0
    if parts in ("k", "both"):
        loss = loss + (yk * wk).sum()
    ins = [x for x, on in ((q, parts != "k"), (k, parts in ("k", "both"))) if on]
    ws = [x for x, on in ((wq, parts != "k"), (wk, parts in ("k", "both"))) if on]
    grads = torch.autograd.grad(loss, ins, create_graph=True)
    # sum of grad * c, c given: its gradient in w is the rotation of c
    cs = [torch.randn_like(x) for x in ins]
    second = torch.autograd.grad(sum((g * c).sum() for g, c in zip(grads, cs)), ws)
    for c, got in zip(cs, second):
        assert torch.equal(got, apply_rotary(c, None, pos, table)[0])
