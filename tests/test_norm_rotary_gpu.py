"""Norms of heads with their rotation, and their gradients, against float64 and
against differences."""

import pytest
import torch

from deltanet_tpu_amd import apply_rotary, norm_rotary, rotary_table
from tests import attn_ref as A
from tests import serving_ref as S
from tests.test_attention_gpu import _near, _rows

pytestmark = pytest.mark.gpu


def _case(seed, B, L, Hq, Hk, D, dt, wdt):
    q, k = _rows(seed, B, L, Hq, D, dt=dt), _rows(seed + 1, B, L, Hk, D, dt=dt)
    return q, k, _rows(seed + 2, D, dt=wdt, scale=0.3), _rows(seed + 3, D, dt=wdt, scale=0.3)


def _check(q, k, wq, wk, pos, table, got, dt, eps, offset, inter):
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
        ref, tol = S.normed(x.double().flatten(0, 1), w.double(), eps, offset, pos, table, inter, dt)
        _near(y.flatten(0, 1), ref, tol)


@pytest.mark.parametrize("dt,wdt", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,R", [(256, 64), (128, 128), (64, 32), (96, 32), (192, 64), (512, 128), (32, 16), (128, 0), (80, 20), (6, 2), (1, 0),
                                 (640, 64)])
def test_matches_float64(dev, dt, wdt, inter, D, R):
    B, L, Hq, Hk = 2, 37, 5, 2
    q, k, wq, wk = _case(D + R, B, L, Hq, Hk, D, dt, wdt)
    pos = torch.randint(0, 500, (B, L), generator=torch.Generator().manual_seed(R))
    table = rotary_table(500, R, device=dev) if R else None
    xs = [t.to(dev).requires_grad_(True) for t in (q, k, wq, wk)]
    args = (pos.to(dev), table) if R else ()
    got = norm_rotary(*xs, *args, eps=1e-5, weight_offset=1.0, interleaved=inter)
    cpu = None if table is None else table.cpu()
    _check(q, k, wq, wk, pos.flatten(), cpu, got, dt, 1e-5, 1.0, inter)
    dq, dk = _rows(7, B, L, Hq, D, dt=dt), _rows(8, B, L, Hk, D, dt=dt)
    grads = torch.autograd.grad(got, xs, (dq.to(dev), dk.to(dev)))
    for i, (x, w, dz) in enumerate(((q, wq, dq), (k, wk, dk))):
        dx, dw, tx, tw = S.normed_grad(x.double().flatten(0, 1), w.double(), dz.double().flatten(0, 1), 1e-5, 1.0, pos.flatten(), cpu,
                                       inter, dt, wdt)
        assert grads[i].dtype == x.dtype and grads[2 + i].dtype == w.dtype
        _near(grads[i].flatten(0, 1), dx, tx, "dx")
        _near(grads[2 + i], dw, tw, "dw")
    with torch.no_grad():
        plain = norm_rotary(*xs, *args, eps=1e-5, weight_offset=1.0, interleaved=inter)
    assert torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[1])


@pytest.mark.parametrize("B,L", [(1, 1), (3, 5000)])
def test_one_and_many_tokens_of_a_projection(dev, B, L):
    """Slices of one projection, one row of positions for all; enough tokens for
    several heads per thread; the same bits every time."""
    Hq, Hk, D, R = 7, 3, 128, 64
    x = _rows(1, B, L, Hq + 2 * Hk, D).to(dev).requires_grad_(True)
    wq, wk = (_rows(s, D, scale=0.3).to(dev).requires_grad_(True) for s in (2, 3))
    table, pos = rotary_table(L, R, device=dev), torch.arange(L, device=dev, dtype=torch.int32).flip(0)
    call = lambda: norm_rotary(x[:, :, :Hq], x[:, :, Hq:Hq + Hk], wq, wk, pos, table)
    got = call()
    q, k = x.detach()[:, :, :Hq].cpu(), x.detach()[:, :, Hq:Hq + Hk].cpu()
    at = pos.long().cpu().repeat(B)
    _check(q, k, wq.detach().cpu(), wk.detach().cpu(), at, table.cpu(), got, "bf16", 1e-6, 0.0, False)
    dq, dk = _rows(4, B, L, Hq, D), _rows(5, B, L, Hk, D)
    grads = [torch.autograd.grad(call(), (x, wq, wk), (dq.to(dev), dk.to(dev))) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    for sl, x_, w, dz, dw in ((slice(0, Hq), q, wq, dq, grads[0][1]), (slice(Hq, Hq + Hk), k, wk, dk, grads[0][2])):
        rx, rw, tx, tw = S.normed_grad(x_.double().flatten(0, 1), w.detach().cpu().double(), dz.double().flatten(0, 1), 1e-6, 0.0, at,
                                       table.cpu(), False, "bf16", "bf16")
        _near(grads[0][0][:, :, sl].flatten(0, 1), rx, tx, "dx")
        _near(dw, rw, tw, "dw")
    assert not grads[0][0][:, :, Hq + Hk:].any()


def test_gradient_against_differences(dev):
    """d/de f(x + e v) from two forwards in float32: the step's error, e^2 |f'''| / 6,
    and the roundings', 2^-19 |f| / e per element, at e = 2^-6."""
    B, L, H, D, R = 1, 4, 2, 64, 32
    xs = [_rows(s, *sh, dt="f32").to(dev).requires_grad_(True) for s, sh in ((1, (B, L, H, D)), (2, (B, L, 1, D)), (3, (D,)), (4, (D,)))]
    table, pos = rotary_table(9, R, device=dev), torch.arange(L, device=dev)
    c = [_rows(s, B, L, h, D, dt="f32").to(dev) for s, h in ((5, H), (6, 1))]
    f = lambda *x: sum((y.double() * z).sum() for y, z in zip(norm_rotary(*x, pos, table, eps=1e-3), c))
    grads = torch.autograd.grad(f(*xs), xs)
    e = 2.0 ** -6
    for i, x in enumerate(xs):
        v = _rows(10 + i, *x.shape, dt="f32").to(dev)
        up, down = ([y.detach() + s * e * v if j == i else y.detach() for j, y in enumerate(xs)] for s in (1, -1))
        diff, want = float((f(*up) - f(*down)) / (2 * e)), float((grads[i].double() * v).sum())
        size = float(sum(z.abs().sum() for z in c))
        assert abs(diff - want) <= 2.0 ** -19 * size / e * 4 + e * e * size, (i, diff, want)


def test_sides_and_broadcast(dev):
    """No keys; one side's result unused; a gradient that is one row for all; rank 3;
    channels that are not contiguous and rows off 16 bytes."""
    N, H, D, R = 21, 3, 128, 64
    table, pos = rotary_table(N, R, device=dev), torch.arange(N, device=dev)
    q, k, wq, wk = (t.to(dev) for t in _case(1, 1, N, H, 2, D, "bf16", "bf16"))
    q, k = q[0], k[0]
    a, b = norm_rotary(q, k, wq, wk, pos, table)
    alone, none = norm_rotary(q, None, wq, None, pos, table)
    assert none is None and torch.equal(alone, a)
    off = torch.empty(q.numel() + 3, dtype=q.dtype, device=dev)[3:].view(q.shape)
    off.copy_(q)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    for x in (off, turned):
        y, _ = norm_rotary(x, None, wq, None, pos, table)
        ref, tol = S.normed(q.cpu().double(), wq.cpu().double(), 1e-6, 0.0, pos.cpu(), table.cpu(), False, "bf16")
        _near(y, ref, tol)
    xs = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]
    a, b = norm_rotary(*xs, pos, table)
    gk, gwk = torch.autograd.grad(b, (xs[1], xs[3]), torch.ones_like(b[:1, :1]).expand_as(b), retain_graph=True)
    want = S.normed_grad(k.cpu().double(), wk.cpu().double(), torch.ones(N, 2, D, dtype=torch.float64), 1e-6, 0.0, pos.cpu(), table.cpu(),
                         False, "bf16", "bf16")
    _near(gk, want[0], want[2])
    _near(gwk, want[1], want[3])
    assert torch.autograd.grad(b.sum(), (xs[0], xs[2]), allow_unused=True) == (None, None)


def test_zeros_infinities_and_far_positions(dev):
    """A head of zeros gives zeros; a position outside the table NaN in the rotated
    channels; a head that is not finite changes no other."""
    N, H, D, R = 6, 4, 128, 64
    table = rotary_table(4, R, device=dev)
    q, wq = _rows(1, N, H, D).to(dev), _rows(2, D).to(dev)
    base, _ = norm_rotary(q, None, wq, None, torch.arange(N, device=dev) % 4, table)
    q2 = q.clone()
    q2[0, 1], q2[1, 2, 5], q2[2, 0, 7] = 0.0, float("inf"), float("nan")
    pos = torch.tensor([0, 1, 2, 3, 4, -1], device=dev)
    out, _ = norm_rotary(q2, None, wq, None, pos, table)
    assert not out[0, 1].any() and not torch.isfinite(out[1, 2, 5]) and torch.isnan(out[2, 0]).all()
    hit = torch.zeros(N, H, dtype=torch.bool, device=dev)
    hit[0, 1] = hit[1, 2] = hit[2, 0] = True
    hit[4:] = True
    assert torch.equal(out[~hit], base[~hit])
    assert torch.isnan(out[4:, :, :R]).all() and torch.isfinite(out[4:, :, R:]).all()


def test_empty_calls(dev):
    table, w = rotary_table(4, 32, device=dev), torch.ones(64, device=dev, requires_grad=True)
    q = torch.zeros(2, 0, 3, 64, device=dev, requires_grad=True)
    a, b = norm_rotary(q, q, w, w, torch.arange(0, device=dev), table)
    (a.sum() + b.sum()).backward()
    assert a.shape == q.shape and q.grad.shape == q.shape and not w.grad.any()


def test_a_layer_of_norm_and_rotation_agrees(dev):
    """The same as the norm in float32 and apply_rotary of it, to that one's rounding."""
    B, L, H, D, R = 2, 50, 4, 128, 128
    q, _, w, _ = _case(3, B, L, H, 1, D, "f32", "f32")
    table, pos = rotary_table(L, R, device=dev), torch.arange(L, device=dev)
    a, _ = norm_rotary(q.to(dev), None, w.to(dev), None, pos, table, weight_offset=1.0)
    y = q.to(dev) * torch.rsqrt((q.to(dev) ** 2).mean(-1, keepdim=True) + 1e-6) * (1.0 + w.to(dev))
    b, _ = apply_rotary(y, None, pos, table)
    assert torch.allclose(a, b, rtol=2e-5, atol=2e-5)


def test_captured_backward(dev):
    """Forward and backward in a graph, replayed on new inputs, against eager calls."""
    N, H, D, R = 300, 4, 128, 64
    table, pos = rotary_table(N, R, device=dev), torch.arange(N, device=dev)
    bufs = [_rows(s, *sh).to(dev) for s, sh in ((1, (N, H, D)), (2, (N, 2, D)), (3, (D,)), (4, (D,)), (5, (N, H, D)), (6, (N, 2, D)))]

    def both(q, k, wq, wk, dq, dk):
        xs = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
        y = norm_rotary(*xs, pos, table)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, xs, (dq, dk)))

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(*bufs)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both(*bufs)
    for t in range(4):
        for i, x in enumerate(bufs):
            x.copy_(_rows(100 * t + i, *x.shape))
        g.replay()
        got = [x.clone() for x in out]
        assert all(torch.equal(a, b) for a, b in zip(got, both(*bufs))), t
        torch.cuda.synchronize()


def test_second_derivatives_are_refused(dev):
    x = torch.randn(3, 2, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y, = torch.autograd.grad(norm_rotary(x, None, w, None)[0].sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        y.sum().backward()


@pytest.mark.parametrize("dt,D", [("f32", 128), ("bf16", 64), ("f32", 6)])
def test_heads_whose_squares_are_below_the_normal_numbers(dev, dt, D):
    """Channels of 1 and 1.5 times 2^-66 with eps 0: their squares are whole multiples of
    2^-134, the sum is exact, the mean is rounded to a multiple of 2^-149, half of that of
    2^-132 or more: 2^-18 of it, 2^-19 of the root, 3 times that of the terms of dx: less
    than twice what the tolerance has for the other roundings."""
    g = torch.Generator().manual_seed(D)
    x = (torch.randint(2, 4, (5, 3, D), generator=g) * (2 * torch.randint(0, 2, (5, 3, D), generator=g) - 1)).double() * 2.0 ** -67
    w, dz = _rows(1, D, dt="f32"), _rows(2, 5, 3, D, dt=dt)
    xs = [x.to(dz.dtype).to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)]
    y, _ = norm_rotary(xs[0], None, xs[1], None, eps=0.0)
    ref, tol = S.normed(x, w.double(), 0.0, 0.0, None, None, False, dt)
    _near(y, ref, 3 * tol)
    dx, dw, tx, tw = S.normed_grad(x, w.double(), dz.double(), 0.0, 0.0, None, None, False, dt, "f32")
    gx, gw = torch.autograd.grad(y, xs, dz.to(dev))
    _near(gx, dx, 3 * tx, "dx")
    _near(gw, dw, 3 * tw, "dw")


def test_more_heads_than_a_launch_has_waves(dev):
    """67 million heads of 2 channels: the first and the last tokens as by calls of their own."""
    L, H, D = 1048600, 65, 2
    x = torch.randn(1, L, H, D, device=dev, dtype=torch.bfloat16)
    w = torch.tensor([0.5, 2.0], device=dev)
    y, _ = norm_rotary(x, None, w, None)
    for part in (slice(0, 1000), slice(L // 2, L // 2 + 1000), slice(L - 1000, L)):
        assert torch.equal(y[:, part], norm_rotary(x[:, part], None, w, None)[0])
