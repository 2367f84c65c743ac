"""Softmax attention, its gradient and the rotation in float64 on the CPU, with
how far a result in a given type may be off, from the roundings that it has."""

from __future__ import annotations

import math

import torch

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# largest relative error of one rounding to nearest: 8, 11 and 24 significant bits
ROUND = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
# smallest step of the type, halved: what rounding may cost next to zero
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}


def visible(L, S, off, starts=None, window=None):
    """(L, S) whether query i, at position off + i, sees key j."""
    i = torch.arange(L)[:, None] + off
    j = torch.arange(S)[None]
    m = j <= i
    if window:
        m &= j > i - window
    if starts is not None:
        m &= j >= starts[:, None]
    return m


def starts_of(seg):
    """First token of the run of equal ids that each token is in."""
    s = torch.zeros(len(seg), dtype=torch.int64)
    for i in range(1, len(seg)):
        s[i] = s[i - 1] if seg[i] == seg[i - 1] else i
    return s


def attend(q, k, v, vis, scale, dt):
    """One head: q (L, D), k, v (S, D) float64.  (out, lse, tolerance of out).

    A probability is rounded once to the 16-bit type before the second product
    (a relative error, and its smallest step), the result once more.  float32
    arithmetic: a score is off by D roundings of its products, which its
    exponential turns into a relative error, and the sums over S keys are off by
    as many roundings; twice those bounds are allowed.
    """
    s = (q @ k.T) * scale
    s = torch.where(vis, s, -math.inf)
    any_ = vis.any(1)
    if not vis.shape[1]:
        return torch.zeros_like(q), torch.full((len(q),), -math.inf, dtype=torch.float64), torch.zeros_like(q)
    m = torch.where(any_, s.amax(1), torch.zeros(len(q), dtype=torch.float64))
    e = torch.exp(s - m[:, None])
    z = e.sum(1)
    p = torch.where(any_[:, None], e / torch.where(any_, z, torch.ones_like(z))[:, None], torch.zeros_like(e))
    vz = torch.where(vis.any(0)[:, None], v, torch.zeros_like(v))
    out = p @ vz
    lse = torch.where(any_, m + torch.log(z), torch.full_like(z, -math.inf))
    return out, lse, tolerance(q, k, vz, p, out, s, scale, dt)


def f32_error(q, k, scale, s):
    """Relative error of a probability from float32 scores."""
    D, S = q.shape[1], k.shape[0]
    if not len(q) or not S:
        return 0.0
    top = torch.where(torch.isfinite(s), s.abs(), torch.zeros_like(s)).max()
    dots = (q.abs() @ k.abs().T).max() * abs(scale)
    return 2.0 ** -24 * 2.0 * (math.sqrt(D) * float(dots) + 4.0 * float(top) + math.sqrt(S) + 16.0)


def tolerance(q, k, v, p, out, s, scale, dt):
    u = ROUND[dt]
    mass = p @ v.abs()
    f = f32_error(q, k, scale, s)
    # (the running maximum may lag by 2^8: a probability next to zero is a step of the type off, at most S of them)
    step = 0.0 if dt == "f32" else TINY[dt] * v.abs().sum(0, keepdim=True)
    return (u if dt != "f32" else 0.0) * mass * 1.05 + f * mass + u * 1.05 * out.abs() + step + TINY[dt]


def rotate(x, pos, table, interleaved=False, sign=1.0):
    """x (N, H, D) float64 with its first table.shape[1] channels rotated."""
    R = table.shape[1]
    c, s = table[pos, None, :R // 2].double(), sign * table[pos, None, R // 2:].double()
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        y[..., 0:R:2], y[..., 1:R:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        y[..., :R // 2], y[..., R // 2:R] = a * c - b * s, b * c + a * s
    return y


def rotate_tolerance(x, dt, R):
    """Two products and a sum in float32 (three roundings of values up to |x| +
    |y| of the pair), one rounding of the result."""
    a = x[..., :R].abs()
    top = a.amax(-1, keepdim=True) * 2.0 if R else 0.0
    return top * (2.0 ** -23 + ROUND[dt] * 1.01) + TINY[dt]


def attend_grad(q, k, v, do, vis, scale, dt):
    """One head: (dq, dk, dv, tolerances of the three) from the formulas
    dV = P^T dO, dS = P (dO V^T - rowsum(dO O)), dQ = scale dS K, dK = scale dS^T Q.

    Roundings to the type: P and dS before their products, the output that
    rowsum(dO O) reads (as far off as its tolerance), the results.
    """
    s = torch.where(vis, (q @ k.T) * scale, -math.inf)
    p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
    out = p @ v
    u, f = ROUND[dt], f32_error(q, k, scale, s)
    r = 0.0 if dt == "f32" else u
    dp = do @ v.T
    ds = p * (dp - (do * out).sum(1, keepdim=True))
    off = (do.abs() * tolerance(q, k, v, p, out, s, scale, dt)).sum(1, keepdim=True)
    f32 = f * (do.abs() @ v.abs().T + (do * out).abs().sum(1, keepdim=True))
    eds = 1.05 * (r * ds.abs() + p * (off + f32)) + f * ds.abs() + (0.0 if dt == "f32" else TINY[dt])
    ep = 1.05 * r * p + f * p + (0.0 if dt == "f32" else TINY[dt])
    dq, dk, dv = scale * ds @ k, scale * ds.T @ q, p.T @ do
    sc = abs(scale)
    return dq, dk, dv, sc * eds @ k.abs() + 1.05 * u * dq.abs() + TINY[dt], sc * eds.T @ q.abs(), ep.T @ do.abs()
