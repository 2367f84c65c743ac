"""How many roundings to the 16-bit type the results of short documents carry."""

import math

import pytest
import torch

from deltanet_tpu_amd import causal_attention
from tests import attn_ref as A
from tests.test_attention_gpu import _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("L,D,doc,Hq,Hkv", [(400, 64, 16, 16, 16), (400, 128, 25, 8, 2), (400, 256, 40, 8, 8), (2200, 128, 17, 16, 16)])
def test_short_documents(dev, dt, L, D, doc, Hq, Hkv):
    """Independent roundings add in squares: the output has one, its own; each gradient
    two, of dS (dq, dk) or P (dv) and its own.  3 percent more are allowed for what is
    in float32.  (Rounded probabilities in the output make it 1.33 of one, and dq and
    dk, whose row sums read it, 1.12 of two.)"""
    q, k, v, do = (_rows(s, 1, L, h, D, dt=dt) for s, h in ((1, Hq), (2, Hkv), (3, Hkv), (4, Hq)))
    seg = torch.arange(L) // doc
    x = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = causal_attention(*x, segment_ids=seg.to(dev))
    got = (out, *torch.autograd.grad(out, x, do.to(dev)))
    vis = A.visible(L, L, 0, A.starts_of(seg.tolist()))
    ref = [torch.zeros(t.shape, dtype=torch.float64) for t in (q, q, k, v)]
    for h in range(Hq):
        y = [t[0, :, i].double() for t, i in ((q, h), (k, h * Hkv // Hq), (v, h * Hkv // Hq))]
        s = torch.where(vis, (y[0] @ y[1].T) / math.sqrt(D), -math.inf)
        ref[0][0, :, h] = torch.softmax(s, 1) @ y[2]
        g = A.attend_grad(*y, do[0, :, h].double(), vis, 1.0 / math.sqrt(D), dt)
        ref[1][0, :, h] = g[0]
        ref[2][0, :, h * Hkv // Hq] += g[1]
        ref[3][0, :, h * Hkv // Hq] += g[2]
    for name, x, r, n in zip(("out", "dq", "dk", "dv"), got, ref, (1, 2, 2, 2)):
        one = (r.to(A.DT[dt]).double() - r).norm()
        off = (x.detach().double().cpu() - r).norm()
        assert off <= 1.03 * math.sqrt(n) * one, (name, float(off / one))
