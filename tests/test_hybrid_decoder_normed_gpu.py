"""The hybrid decoder with normed heads: it runs, every weight has its gradient, and what
it serves over a paged cache is what it gives over whole rows."""

import pytest
import torch

from tests.test_hybrid_decoder_gpu import example  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,most", [("bf16", 3e-2), ("f32", 2e-4)])
def test_served_tokens_match_whole_rows(dev, example, dt, most):  # noqa: F811
    """The bounds of the decoder without norms: they add one rounding fewer than they
    take away (norm and rotation are rounded once)."""
    torch.manual_seed(0)
    model = example.HybridDecoder(normed=True).to(dev, torch.bfloat16 if dt == "bf16" else torch.float32)
    with torch.no_grad():
        for p in model.layers[3].norms:
            p.uniform_(-0.3, 0.3)
    err = example.serving_error(model, lengths=(130, 64, 1), steps=5)
    print(f"[measured] {dt} {err:.2e}")
    assert err <= most


def test_gradients_of_the_norms(dev, example):  # noqa: F811
    """Against differences of the loss in float32: e^2 of its third derivative, and the
    loss's own error, 1e-5 of it, over 2 e, at e = 0.05."""
    torch.manual_seed(0)
    model = example.HybridDecoder(blocks=1, normed=True).to(dev)
    tokens = torch.randint(0, 512, (1, 100), device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    loss = lambda: torch.nn.functional.cross_entropy(model(tokens[:, :-1])[0].double(), tokens[0, 1:])
    loss().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    e = 0.05
    for p in model.layers[3].norms:
        v = p.grad.sign()
        with torch.no_grad():
            p += e * v
            up = float(loss())
            p -= 2 * e * v
            down = float(loss())
            p += e * v
        want = float(p.grad.abs().sum())
        assert want > 0 and abs((up - down) / (2 * e) - want) <= 0.05 * want + 1e-5 * up / e, ((up - down) / (2 * e), want)
