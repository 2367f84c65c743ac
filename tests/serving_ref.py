"""Normed heads, page tables and drafted trees in float64 and plain integers on the
CPU, with how far a result in a given type may be off, from the roundings that it has."""

from __future__ import annotations

import torch

from tests import attn_ref as A


def pairs(x, R, inter):
    """|x| plus its partner's in the rotation (itself alone where there is none)."""
    y = x.abs().clone()
    if R:
        a, b = (y[..., 0:R:2].clone(), y[..., 1:R:2].clone()) if inter else (y[..., :R // 2].clone(), y[..., R // 2:R].clone())
        if inter:
            y[..., 0:R:2] = y[..., 1:R:2] = a + b
        else:
            y[..., :R // 2] = y[..., R // 2:R] = a + b
    return y


def normed(x, w, eps, offset, pos, table, inter, dt):
    """x (N, H, D) and w (D,) float64, table (P, R) float32 or None: (z, tolerance).

    Roundings to float32 (2^-24 each): the squares and their sum, 16 + 16 in a row at
    most and halved by the root, 16; the root's reciprocal, 2; offset + weight, two
    products: 21 in all, less than 2^-19 of |y|.  The rotation: two products and a
    sum, 2^-22 of the pair.  Then the one rounding to the type."""
    gain = offset + w
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gain
    R = 0 if table is None else table.shape[1]
    z = A.rotate(y, pos, table, inter) if R else y
    return z, 1.2 * 2.0 ** -19 * pairs(y, R, inter) + 1.01 * A.ROUND[dt] * z.abs() + A.TINY[dt]


def normed_grad(x, w, dz, eps, offset, pos, table, inter, dt, wdt):
    """(dx, dw, tolerances): g = rotation^T(dz), h = g (offset + w), dx = r (h - x r^2
    mean(h x)), dw = sum of g x r.

    Each g is 2^-22 of its pair off, h and r 21 roundings more (2^-19 of it), the mean
    as much of the sum of |h x|; of dw besides the sums over tokens, in float32, one
    after another within a thread, over the threads of a block and over the blocks:
    less than 256 additions in a row here, 2^-16 of the sum of magnitudes."""
    D, R = x.shape[-1], 0 if table is None else table.shape[1]
    g = A.rotate(dz, pos, table, inter, -1.0) if R else dz
    gain, r = offset + w, 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    h, big = g * gain, pairs(dz, R, inter)
    dx = r * (h - x * r * r * (h * x).sum(-1, keepdim=True) / D)
    mean = (big * gain.abs() * x.abs()).sum(-1, keepdim=True) / D
    off = 2.0 ** -18 * r * (big * gain.abs() + x.abs() * r * r * mean)
    dw = (g * x * r).sum((0, 1))
    offw = 2.0 ** -16 * (big * x.abs() * r).sum((0, 1))
    return dx, dw, off + 1.01 * A.ROUND[dt] * dx.abs() + A.TINY[dt], offw + 1.01 * A.ROUND[wdt] * dw.abs() + A.TINY[wdt]


class Pool:
    """The pool as a list, sequence by sequence."""

    def __init__(self, pages):
        self.free = list(range(pages - 1, -1, -1))

    def reserve(self, rows, lens, page, most):
        """rows: each sequence's pages, changed in place; the pages each is short of."""
        need = [-(-max(n, 0) // page) for n in lens]
        for b in reversed(range(len(rows))):
            while len(rows[b]) > need[b]:
                self.free.append(rows[b].pop())
        short, over = [], False
        for b, row in enumerate(rows):
            want = need[b] - len(row)
            if need[b] > most:
                short.append(want)
                continue
            if want > 0 and (over or want > len(self.free)):
                over = True
                short.append(want)
                continue
            for _ in range(want):
                row.append(self.free.pop())
            short.append(0)
        return short


def trees(new, seed, wide=4):
    """Parents of drafted trees of these sizes, not in the order of their levels, and
    truth values (n, n) of what each node sees."""
    g = torch.Generator().manual_seed(seed)
    parents, seen = [], []
    for n in new:
        p, m = [], torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            a = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            if wide and i and int(torch.randint(0, wide, (1,), generator=g)):
                a = i - 1   # long branches too
            p.append(a)
            if a >= 0:
                m[i] = m[a]
            m[i, i] = True
        parents += p
        seen.append(m)
    return parents, seen


def words(seen, count):
    """Truth values (n, n) of each sequence as (sum of n, count) 64-bit words."""
    out = torch.zeros(sum(len(m) for m in seen), count, dtype=torch.int64)
    at = 0
    for m in seen:
        for i in range(len(m)):
            for j in m[i].nonzero().flatten().tolist():
                if j < 64 * count:
                    out[at + i, j // 64] |= (1 << (j % 64)) - (1 << 64 if j % 64 == 63 else 0)
        at += len(m)
    return out


def tree_visible(seen, length, window=None, count=16):
    """(n, length) whether each new token sees each token of its sequence."""
    n = len(seen)
    off = length - n
    m = torch.zeros(n, max(length, 0), dtype=torch.bool)
    if off > 0:
        m[:, :off] = True
    for j in range(min(n, 64 * count)):
        if off + j >= 0:
            m[:, off + j] = seen[:, j]
    if window:
        m &= m.flip(1).cumsum(1).flip(1) <= window
    return m
