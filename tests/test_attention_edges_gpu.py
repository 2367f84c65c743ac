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
