"""Heads whose squares leave float32's range on either side, next to heads whose squares
do not, against float64."""

import pytest
import torch

from deltanet_tpu_amd import norm_rotary, paged_qkv_append, rotary_table
from tests import attn_ref as A
from tests import serving_ref as S
from tests.test_attention_gpu import _near, _rows

pytestmark = pytest.mark.gpu

# powers of two that heads are taken times, in turn: most lie next to others in a wave
POWERS = (0, -80, 66, -130, 0, 110, -66, -48, 59, -100, 63, 0, -125, 120)


def _heads(seed, N, H, D, dt):
    """Heads of these sizes; in some a channel is far larger or smaller than the rest."""
    x = torch.randn(N, H, D, generator=torch.Generator().manual_seed(seed)).double()
    for i in range(N * H):
        p = POWERS[i % len(POWERS)]
        x[i // H, i % H] *= 2.0 ** p
        if i % 3 == 0 and D > 1:
            x[i // H, i % H, i % D] *= 2.0 ** (30 if p < 0 else -30)
    return x.to(A.DT[dt])


# heads of whole groups and others, of every number of lanes
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,R", [(32, 16), (64, 0), (128, 64), (256, 64), (512, 128), (6, 2), (80, 20), (1, 0), (640, 64)])
@pytest.mark.parametrize("N", [45, 5000])
def test_heads_of_every_size(dev, dt, D, R, N):
    if N * D > 5000 * 128:
        N = 5000 * 128 // D   # (enough tokens for the form of two heads a thread, few enough for the reference)
    Hq, Hk = 5, 2
    q, k, wq, wk = _heads(1, N, Hq, D, dt), _heads(2, N, Hk, D, dt), _rows(3, D, dt="f32", scale=0.3), _rows(4, D, dt="f32", scale=0.3)
    pos = torch.arange(N) % 300
    table = rotary_table(300, R, device=dev) if R else None
    args, cpu = ((pos.to(dev), table), table.cpu()) if R else ((), None)
    for eps in (0.0, 1e-35):
        got = norm_rotary(q.to(dev), k.to(dev), wq.to(dev), wk.to(dev), *args, eps=eps, weight_offset=1.0)
        for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
            ref, tol = S.normed(x.double(), w.double(), eps, 1.0, pos, cpu, False, dt)
            _near(y, ref, tol.nan_to_num(0.0), f"eps {eps}")   # (a zero by itself over eps 0 is no number)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("D,R", [(64, 32), (128, 64), (256, 0), (512, 64), (80, 20), (6, 2), (1, 0)])
@pytest.mark.parametrize("power", [-100, -80, -60, 60, 66, 100])
def test_gradients(dev, dt, D, R, power):
    """Every other head of this size.  A head's share of the weights' gradient does not
    depend on its size; its own gradient is as much larger as it is smaller."""
    N, Hq, Hk = 40, 5, 2
    size = lambda H: torch.tensor([2.0 ** (power if i % 2 else 0) for i in range(N * H)], dtype=torch.float64).view(N, H, 1)
    q, k = ((torch.randn(N, H, D, generator=torch.Generator().manual_seed(H)).double() * size(H)).to(A.DT[dt]) for H in (Hq, Hk))
    wq, wk = _rows(3, D, dt="f32", scale=0.3), _rows(4, D, dt="f32", scale=0.3)
    dq, dk = _rows(5, N, Hq, D, dt=dt), _rows(6, N, Hk, D, dt=dt)
    pos = torch.arange(N)
    table = rotary_table(N, R, device=dev) if R else None
    args, cpu = ((pos.to(dev), table), table.cpu()) if R else ((), None)
    xs = [t.to(dev).requires_grad_(True) for t in (q, k, wq, wk)]
    got = norm_rotary(*xs, *args, eps=0.0, weight_offset=1.0)
    grads = torch.autograd.grad(got, xs, (dq.to(dev), dk.to(dev)))
    for i, (x, w, dz) in enumerate(((q, wq, dq), (k, wk, dk))):
        dx, dw, tx, tw = S.normed_grad(x.double(), w.double(), dz.double(), 0.0, 1.0, pos, cpu, False, dt, "f32")
        _near(grads[i], dx, tx, "dx")
        _near(grads[2 + i], dw, tw, "dw")


def test_stored_heads_of_every_size(dev):
    """The form of serving: the bits of norm_rotary."""
    N, Hq, Hkv, D, R, page = 64, 4, 2, 128, 64, 16
    q, k, v = (_heads(s, N, h, D, "bf16").to(dev) for s, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    wq, wk = _rows(4, D).to(dev), _rows(5, D).to(dev)
    table, pos = rotary_table(N, R, device=dev), torch.arange(N, device=dev)
    kc, vc = (torch.zeros(N // page, page, Hkv, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    out = paged_qkv_append(q, k, v, kc, vc, pos, pos, q_weight=wq, k_weight=wk, eps=0.0, table=table)
    qr, kr = norm_rotary(q, k, wq, wk, pos, table, eps=0.0)
    assert torch.equal(out, qr) and torch.equal(kc.flatten(0, 1), kr) and torch.equal(vc.flatten(0, 1), v)
