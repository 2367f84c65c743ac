"""The gradient of normed heads computes what is asked for: frozen inputs and weights."""

import itertools

import pytest
import torch

from deltanet_tpu_amd import _lib, attention, norm_rotary, rotary_table
from tests.test_attention_gpu import _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,R", [(128, 64), (80, 20)])
def test_frozen_leaves(dev, monkeypatch, D, R):
    """Of every subset of the leaves: the bits of the whole gradient, and no pointer for
    what nobody wants."""
    blocks, call = [], attention._call

    def watched(name, device, *args):
        if name == "dn_norm_rotary_bwd":
            blocks.append(_lib.NormRotaryGrads.from_buffer_copy(args[1]))
        return call(name, device, *args)

    monkeypatch.setattr(attention, "_call", watched)
    q, k, wq, wk = _rows(1, 2, 50, 4, D), _rows(2, 2, 50, 2, D), _rows(3, D), _rows(4, D)
    table, pos = rotary_table(50, R, device=dev), torch.arange(50, device=dev)
    dz = [_rows(5, 2, 50, 4, D).to(dev), _rows(6, 2, 50, 2, D).to(dev)]

    def leaves(wanted):
        return [x.to(dev).requires_grad_(w) for x, w in zip((q, k, wq, wk), wanted)]

    xs = leaves([True] * 4)
    want = torch.autograd.grad(norm_rotary(*xs, pos, table), xs, dz)
    for wanted in itertools.product((True, False), repeat=4):
        if not any(wanted):
            continue
        xs = leaves(wanted)
        out = norm_rotary(*xs, pos, table)
        blocks.clear()
        pairs = [(y, d) for y, d in zip(out, dz) if y.requires_grad]
        torch.autograd.backward([y for y, _ in pairs], [d for _, d in pairs])
        for x, w, g in zip(xs, wanted, want):
            assert torch.equal(x.grad, g) if w else x.grad is None
        b, = blocks
        assert [bool(p) for p in (b.dq, b.dk, b.dq_weight, b.dk_weight)] == list(wanted)
        assert bool(b.d_q) == (wanted[0] or wanted[2]) and bool(b.d_k) == (wanted[1] or wanted[3])
