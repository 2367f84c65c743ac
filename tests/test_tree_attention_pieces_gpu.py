"""Drafted trees where a workgroup's piece is a long walk over keys: more sequences and
heads than the card has workgroups, all of them over the pages of one text, so that
float64 on the CPU has that one to compute."""

import math

import pytest
import torch

from deltanet_tpu_amd import paged_tree_attention
from tests import attn_ref as A
from tests import serving_ref as S
from tests.test_attention_gpu import _rows

pytestmark = pytest.mark.gpu

HEADS, GROUPS = 8, 512   # GROUPS: workgroups that a launch has at most


def _text(dev, k, v, page):
    """Caches that hold k and v (len, D) for every one of HEADS key heads, and their pages."""
    n, D = k.shape
    pages = -(-n // page) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(n)).to(torch.int32)
    caches = []
    for x in (k, v):
        c = torch.full((pages, page, 1, D), math.nan, dtype=x.dtype)
        rows = torch.cat([x, x.new_full((pages * page - n, D), math.nan)]).view(pages, page, 1, D)
        c[order.long()] = rows
        caches.append(c.to(dev).expand(pages, page, HEADS, D))
    return (*caches, order[:-1].to(dev))


def _run(dev, dt, q, k, v, page, B, lens, seen, window=None, scale=None, tag=""):
    """B sequences with the first lens[b % len(lens)] tokens of the text each, q (n, G, D)
    the queries of every key head: every copy of a result against float64."""
    n, G, D = q.shape
    of = [lens[b % len(lens)] for b in range(B)]
    # 64 keys or more a tile, of 256 rows or fewer: pieces are of this many tiles at least
    assert sum(min(x, (window or x) + n) // 64 for x in of) * HEADS * max(1, n * G // 256) >= 6 * GROUPS
    kc, vc, pt = _text(dev, k, v, page)
    words = S.words([seen], -(-n // 64)).repeat(B, 1).to(dev)
    out, lse = paged_tree_attention(q[None, :, None].expand(B, n, HEADS, G, D).reshape(B, n, HEADS * G, D).to(dev), kc, vc, pt.expand(B, -1),
                                    torch.tensor(of, dtype=torch.int32, device=dev), words, window=window, scale=scale, return_lse=True)
    out, lse = out.view(B, n, HEADS, G, D).double(), lse.view(B, n, HEADS, G).double()
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    for i, length in enumerate(lens):
        vis = S.tree_visible(seen, length, window)
        x, y = k[:length].double(), v[:length].double()
        x = torch.where(vis.any(0)[:, None], x, torch.zeros_like(x))   # (what nobody sees may be NaN)
        for g in range(G):
            ref, l, tol = A.attend(q[:, g].double(), x, y, vis, scale, dt)
            at = f"{tag} length {length} head {g}"
            _same(out[i::len(lens), :, :, g].transpose(1, 2), ref, tol, at)
            _same(lse[i::len(lens), :, :, g].transpose(1, 2), l, 4 * A.f32_error(q[:, g].double(), x, scale, torch.zeros(1)) + 1e-6 * l.abs(), at + " lse")


def _same(got, ref, tol, tag):
    """Every copy, on its device."""
    d = (got - ref.to(got.device)).abs()
    assert bool((d <= tol.to(got.device)).all()), f"{tag}: off by {float(d.nan_to_num(1e9).max()):.3e}, {int((~(d <= tol.to(got.device))).sum())} elements outside"


# new tokens of 4 query heads a key head: 32 to 256 rows, every size of a tile
FORMS = [(dt, D, n) for dt in ("bf16", "f16", "f32") for D in (64, 128, 256) for n in (8, 16, 32, 64)]


def _masks(kind, n):
    ones = torch.ones(n, n, dtype=torch.bool)
    return {"chain": ones.tril(), "all": ones, "tree": S.trees([n], n)[1][0]}[kind]


@pytest.mark.parametrize("dt,D,n", FORMS)
def test_windows_whose_first_key_begins_a_tile(dev, dt, D, n):
    """A row that sees all new tokens has the last of the windows' first keys: tiles in
    front of it are the other rows'.  64 sequences of a length: every workgroup has whole
    tasks.  The tokens before the windows are not finite."""
    k, v, q = _rows(1, 1056, D, dt=dt), _rows(2, 1056, D, dt=dt), _rows(3, n, 4, D, dt=dt)
    k[:400] = v[:400] = math.nan
    for kind in ("chain", "all"):
        for lens in ([1024], [1024, 1056, 1027]):
            _run(dev, dt, q, k, v, 16, 64, lens, _masks(kind, n), window=512, tag=kind)


@pytest.mark.parametrize("dt,D,n", FORMS)
def test_scores_of_every_course(dev, dt, D, n):
    """Scores (natural logarithms) of a piece's first tile, of keys in its middle and of its
    last ones, the trees' own among them, far from each other either way."""
    length = 1024 + n
    for first, peak, last in ((0, 90, 62), (0, 90, 95), (0, 90, 88), (0, 30, 0), (0, 60, 0), (-80, 20, 10), (50, 0, 0)):
        q, k, v = _rows(4, n, 4, D, dt=dt, scale=0.1), _rows(5, length, D, dt=dt), _rows(6, length, D, dt=dt)
        q[..., 0] = 1.0
        k[:, 0] = first
        k[300:700:7, 0] = peak
        k[940:, 0] = last
        for B, lens in ((64, [1024]), (41, [length, 1024, 777])):
            _run(dev, dt, q, k, v, 64, B, lens, _masks("tree", n), scale=1.0, tag=f"{first} {peak} {last}")


@pytest.mark.parametrize("dt,D,n", [f for f in FORMS if f[2] != 16])
def test_scores_that_grow_within_a_piece(dev, dt, D, n):
    """Over pages of 4 tokens, up to 2^170 times the first."""
    length = 1300
    for grow in (12.0, 120.0):
        q, k, v = _rows(7, n, 4, D, dt=dt, scale=0.1), _rows(8, length, D, dt=dt), _rows(9, length, D, dt=dt)
        q[..., 0] = 1.0
        k[:, 0] = torch.linspace(0.0, grow, length).to(A.DT[dt])
        _run(dev, dt, q, k, v, 4, 41, [length, 1000], _masks("tree", n), scale=1.0, tag=f"{grow}")


@pytest.mark.parametrize("dt,D,page", [("bf16", 128, 16), ("f16", 64, 4), ("f32", 128, 16), ("f32", 256, 4), ("bf16", 256, 64)])
@pytest.mark.parametrize("n,G", [(7, 2), (20, 4), (64, 6)])
def test_lengths_past_the_page_table(dev, dt, D, page, n, G):
    """Drafts that the page table has no place for are seen by none, and the others keep
    their places; where the window lies past the table a token sees nothing."""
    room = 320
    k, v, q = _rows(10, room, D, dt=dt), _rows(11, room, D, dt=dt), _rows(12, n, G, D, dt=dt)
    kc, vc, pt = _text(dev, k, v, page)
    lens = [room + x for x in (-3, 0, 1, n // 2, n - 1, n, n + 1, 500, 2 ** 31 - 1 - room)]
    seen = _masks("tree", n)
    words = S.words([seen], 1).repeat(len(lens), 1).to(dev)
    qd = q[None, :, None].expand(len(lens), n, HEADS, G, D).reshape(len(lens), n, HEADS * G, D).to(dev)
    for window in (None, 64, 200, 400):
        out, lse = paged_tree_attention(qd, kc, vc, pt.expand(len(lens), -1), torch.tensor(lens, dtype=torch.int32, device=dev), words,
                                        window=window, return_lse=True)
        out, lse = out.view(-1, n, HEADS, G, D).double(), lse.view(-1, n, HEADS, G).double()
        for b, length in enumerate(lens):
            far = min(length, room + 600)   # (from there on all is context, or all behind the table)
            vis = S.tree_visible(seen, far, window)[:, :room]
            for g in range(G):
                ref, l, tol = A.attend(q[:, g].double(), k[:vis.shape[1]].double(), v[:vis.shape[1]].double(), vis, 1.0 / math.sqrt(D), dt)
                at = f"window {window} length {length} head {g}"
                _same(out[b, :, :, g].transpose(0, 1), ref, tol, at)
                got = lse[b, :, :, g].transpose(0, 1)
                assert torch.equal(got.isneginf().cpu(), l.isneginf().expand_as(got)), at
                _same(torch.where(got.isneginf(), 0.0, got), torch.where(l.isneginf(), 0.0, l), torch.full_like(l, 1e-4), at + " lse")
