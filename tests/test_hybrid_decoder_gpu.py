"""The attention operators and the delta-rule layers together: what a hybrid
decoder gives token by token over a paged cache is what it gives over whole rows."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("hybrid_decoder", os.path.join(ROOT, "examples", "hybrid_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dt,most", [("bf16", 3e-2), ("f32", 2e-4)])
def test_served_tokens_match_whole_rows(dev, example, dt, most):
    """Eight layers, each rounding its result once to the type (2^-8 in bf16) and its
    probabilities once more; float32 forms differ in the order of their sums alone
    (chunked delta rule at precision "bf16" included: split products, 1e-5 a layer)."""
    torch.manual_seed(0)
    model = example.HybridDecoder().to(dev, torch.bfloat16 if dt == "bf16" else torch.float32)
    err = example.serving_error(model, lengths=(130, 64, 1), steps=5)
    print(f"[measured] {dt} {err:.2e}")
    assert err <= most


def test_training_steps_lower_the_loss(dev, example):
    torch.manual_seed(0)
    model = example.HybridDecoder(blocks=1).to(dev)
    losses = example.train_steps(model, steps=6, L=200)
    assert all(x == x for x in losses) and losses[-1] < losses[0] - 0.5
