"""Softmax attention on the GPU, over whole rows and over a paged cache, against
float64 on the CPU."""

import math

import pytest
import torch

from deltanet_tpu_amd import causal_attention, paged_attention
from tests import attn_ref as A

pytestmark = pytest.mark.gpu


def _near(got, ref, tol, tag=""):
    got = got.detach().double().cpu()
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    d = torch.where(same, torch.zeros_like(ref), (got - ref).abs())
    assert bool((d <= tol).all()), f"{tag}: off by {float(d.nan_to_num(1e9).max()):.3e}, {int((~(d <= tol)).sum())} elements outside"


def _rows(seed, *shape, dt="bf16", scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(A.DT[dt])


def _check_rows(out, lse, q, k, v, dt, starts=None, window=None, scale=None, tag=""):
    B, L, Hq, D = q.shape
    G = Hq // k.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        vis = A.visible(L, L, 0, None if starts is None else starts[b], window)
        for h in range(Hq):
            ref, l, tol = A.attend(q[b, :, h].double(), k[b, :, h // G].double(), v[b, :, h // G].double(), vis, scale, dt)
            _near(out[b, :, h], ref, tol, f"{tag} row {b} head {h}")
            if lse is not None:
                _near(lse[b, :, h], l, 4 * A.f32_error(q[b, :, h].double(), k[b, :, h // G].double(), scale, torch.zeros(1)) + 1e-6 * l.abs(), "lse")


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,L,Hq,Hkv,D", [(1, 1, 1, 1, 64), (2, 3, 4, 2, 128), (1, 63, 3, 1, 256), (1, 64, 4, 4, 128),
                                          (2, 129, 8, 2, 64), (1, 300, 6, 1, 128), (1, 257, 4, 2, 256), (1, 515, 2, 2, 128)])
def test_rows(dev, dt, B, L, Hq, Hkv, D):
    q, k, v = _rows(1, B, L, Hq, D, dt=dt), _rows(2, B, L, Hkv, D, dt=dt), _rows(3, B, L, Hkv, D, dt=dt)
    out, lse = causal_attention(q.to(dev), k.to(dev), v.to(dev), return_lse=True)
    assert out.dtype == q.dtype and out.shape == q.shape
    _check_rows(out, lse, q, k, v, dt)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("window", [None, 1, 17, 64, 1000])
@pytest.mark.parametrize("docs", [False, True])
def test_rows_windows_and_documents(dev, dt, window, docs):
    B, L, Hq, Hkv, D = 2, 333, 4, 2, 128
    q, k, v = _rows(1, B, L, Hq, D, dt=dt), _rows(2, B, L, Hkv, D, dt=dt), _rows(3, B, L, Hkv, D, dt=dt)
    seg = starts = None
    if docs:
        seg = torch.zeros(B, L, dtype=torch.int64)
        for t in (1, 64, 65, 130, 200, 332):
            seg[0, t:] += 1
        seg[0, 210:] = 0   # an id that comes again is another document
        seg[1, 100:] = 5
        starts = [A.starts_of(s.tolist()) for s in seg]
    out = causal_attention(q.to(dev), k.to(dev), v.to(dev), segment_ids=None if seg is None else seg.to(dev), window=window)
    _check_rows(out, None, q, k, v, dt, starts, window)


def test_rows_documents_forms(dev):
    """cu_seqlens, shared 1D ids, int32 ids and 2D ids agree to the bit; a long row
    runs the document scan over several blocks."""
    B, L, H, D = 2, 2500, 2, 64
    q, k, v = (_rows(s, B, L, H, D).to(dev) for s in (1, 2, 3))
    cu = [0, 3, 700, 1024, 1025, 2400, L]
    seg = torch.repeat_interleave(torch.arange(len(cu) - 1), torch.tensor(cu).diff())
    a = causal_attention(q, k, v, cu_seqlens=cu)
    for s in (seg.to(dev), seg.to(torch.int32).to(dev), seg.expand(B, L).to(dev), seg.numpy(), seg.to(torch.int16).to(dev)):
        assert torch.equal(a, causal_attention(q, k, v, segment_ids=s))
    starts = [A.starts_of(seg.tolist())] * B
    _check_rows(a[:, :, :1], None, q[:, :, :1].cpu(), k[:, :, :1].cpu(), v[:, :, :1].cpu(), "bf16", starts)


def test_rows_strides_scale_and_peaked_scores(dev):
    """Slices of one projection, heads before tokens, rows off 16 bytes; a scale of
    its own; scores up to hundreds."""
    B, L, Hq, Hkv, D = 2, 150, 4, 2, 128
    x = _rows(4, B, L, Hq + 2 * Hkv, D, scale=3.0)
    xd = x.to(dev)
    q, k, v = x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:]
    out = causal_attention(xd[:, :, :Hq], xd[:, :, Hq:Hq + Hkv], xd[:, :, Hq + Hkv:], scale=0.5)
    _check_rows(out, None, q, k, v, "bf16", scale=0.5)
    t = lambda y: y.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(out, causal_attention(t(q), t(k), t(v), scale=0.5))
    off = torch.empty(B * L * Hq * D + 3, dtype=torch.bfloat16, device=dev)[3:].view(B, L, Hq, D)
    off.copy_(q.to(dev))
    assert torch.equal(out, causal_attention(off, t(k), t(v), scale=0.5))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("odd", [math.nan, math.inf, -math.inf])
def test_rows_hidden_infinities(dev, dt, odd):
    """A token whose key and value are not finite changes no query that does not
    see it, in its tile or elsewhere, and those that see it as the sums say."""
    B, L, H, D, at = 1, 200, 2, 64, 100
    q, k, v = (_rows(s, B, L, H, D, dt=dt) for s in (1, 2, 3))
    seg = torch.tensor([0] * 40 + [1] * 100 + [2] * 60)
    base = causal_attention(q.to(dev), k.to(dev), v.to(dev), segment_ids=seg.to(dev))
    v2 = v.clone()
    v2[0, at, :, 3] = odd
    out = causal_attention(q.to(dev), k.to(dev), v2.to(dev), segment_ids=seg.to(dev))
    hit = torch.zeros(L, dtype=torch.bool)
    hit[at:140] = True
    assert torch.equal(out[0, ~hit], base[0, ~hit])
    assert torch.equal(out[0, hit][..., 4:], base[0, hit][..., 4:])
    want = torch.full((int(hit.sum()), H), odd)
    got = out[0, hit][..., 3].float().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and (math.isnan(odd) or torch.equal(got, want))
    k2 = k.clone()
    k2[0, at] = odd
    out = causal_attention(q.to(dev), k2.to(dev), v2.to(dev), segment_ids=seg.to(dev))
    assert torch.equal(out[0, ~hit], base[0, ~hit])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_rows_scores_far_above_the_own(dev, dt, D):
    """Queries whose score with themselves is far below another one's: by the
    thousand (the kernel's range of exponents does not reach), and growing from
    tile to tile; other rows of the tile keep their bits."""
    B, L, H = 1, 400, 2
    q, k, v = (_rows(s, B, L, H, D, dt=dt) for s in (1, 2, 3))
    base = causal_attention(q.to(dev), k.to(dev), v.to(dev))
    k2, q2 = k.clone(), q.clone()
    for at, size in ((3, 40.0), (70, 80.0), (200, 160.0)):   # keys along one axis, ever longer
        k2[0, at] = 0
        k2[0, at, :, 0] = size
    q2[0, 100:110, :, 0], q2[0, 300:310, :, 0] = 50.0, 100.0
    out, lse = causal_attention(q2.to(dev), k2.to(dev), v.to(dev), return_lse=True)
    _check_rows(out, None, q2, k2, v, dt)
    assert torch.equal(out[0, :3], base[0, :3])
    # the same keys, with and without rows that go beyond the range
    plain = causal_attention(q.to(dev), k2.to(dev), v.to(dev))
    same = torch.ones(L, dtype=torch.bool)
    same[100:110] = same[300:310] = False
    if dt != "f16":   # (float16's range is narrow enough for other rows to go beyond it as well)
        assert torch.equal(out[0, same], plain[0, same])


# ---------------------------------------------------------------------------
# paged
# ---------------------------------------------------------------------------

def _paged(seed, new, lens, Hkv, D, page, dt, dev, heads_first=False, junk=math.nan):
    """Caches whose unused places hold `junk`, the page table, and the keys and
    values (len, Hkv, D) of each sequence."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-x // page) for x in lens]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=g).tolist()
    pt = torch.full((len(lens), max(max(counts), 1) + 1), 1 << 30, dtype=torch.int32)
    kc, vc = (torch.full((pages, page, Hkv, D), junk, dtype=A.DT[dt]) for _ in range(2))
    ks, vs = [], []
    for b, n in enumerate(lens):
        k, v = (torch.randn(n, Hkv, D, generator=g).to(A.DT[dt]) for _ in range(2))
        for i in range(counts[b]):
            pg = order.pop()
            pt[b, i] = pg
            m = min(page, n - i * page)
            kc[pg, :m], vc[pg, :m] = k[i * page:i * page + m], v[i * page:i * page + m]
        ks.append(k)
        vs.append(v)
    put = lambda c: c.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if heads_first else c.to(dev)
    cu = torch.tensor([0] + list(new), dtype=torch.int32).cumsum(0).to(torch.int32)
    return put(kc), put(vc), pt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), cu.to(dev), ks, vs


def _check_paged(out, lse, q, ks, vs, new, lens, dt, window=None, scale=None):
    G, D = q.shape[1] // ks[0].shape[1], q.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    i = 0
    for b, (n, m) in enumerate(zip(new, lens)):
        vis = A.visible(n, m, m - n, None, window)
        for h in range(q.shape[1]):
            x = q[i:i + n, h].double()
            ref, l, tol = A.attend(x, ks[b][:, h // G].double(), vs[b][:, h // G].double(), vis, scale, dt)
            _near(out[i:i + n, h], ref, tol, f"sequence {b} head {h}")
            if lse is not None:
                _near(lse[i:i + n, h], l, 4 * A.f32_error(x, ks[b][:, h // G].double(), scale, torch.zeros(1)) + 1e-6 * l.abs(), "lse")
        i += n


CASES = [
    # new tokens, sequence lengths
    ([1], [1]), ([1], [1000]), ([1, 1, 1], [5, 64, 65]), ([1] * 9, [3, 2000, 16, 17, 129, 700, 1, 2, 33]),
    ([5, 5, 5], [5, 60, 300]), ([70, 1, 0, 3, 130], [70, 40, 9, 500, 200]), ([0, 0], [4, 0]), ([2, 3], [0, 1]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dt,Hq,Hkv,D,page,hf", [("bf16", 8, 2, 128, 16, False), ("bf16", 4, 1, 256, 64, True), ("f16", 3, 3, 64, 128, False),
                                                 ("f32", 4, 2, 128, 32, False), ("bf16", 20, 1, 128, 1, False), ("f32", 2, 1, 256, 64, True),
                                                 ("f16", 16, 2, 256, 16, False)])
def test_paged(dev, case, dt, Hq, Hkv, D, page, hf):
    new, lens = CASES[case]
    kc, vc, pt, sl, cu, ks, vs = _paged(7, new, lens, Hkv, D, page, dt, dev, hf)
    q = _rows(8, sum(new), Hq, D, dt=dt)
    out, lse = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype
    _check_paged(out, lse, q, ks, vs, new, lens, dt)


@pytest.mark.parametrize("window", [1, 30, 64, 400])
@pytest.mark.parametrize("D,page", [(128, 16), (256, 64)])
def test_paged_window(dev, window, D, page):
    new, lens = [1, 4, 90, 1], [700, 333, 600, 20]
    kc, vc, pt, sl, cu, ks, vs = _paged(9, new, lens, 2, D, page, "bf16", dev)
    q = _rows(10, sum(new), 8, D)
    out = paged_attention(q.to(dev), kc, vc, pt, sl, cu_seqlens=cu, window=window, scale=0.2)
    _check_paged(out, None, q, ks, vs, new, lens, "bf16", window, 0.2)


def test_paged_forms_agree(dev):
    """(B, Hq, D), (B, 1, Hq, D) and cu_seqlens; (B, T, Hq, D); strided queries."""
    B, T = 4, 6
    kc, vc, pt, sl, cu, ks, vs = _paged(11, [T] * B, [6, 100, 257, 900], 2, 128, 16, "bf16", dev)
    x = _rows(12, B, T, 12, 128).to(dev)
    q = x[:, :, :8]
    a = paged_attention(q, kc, vc, pt, sl)
    b = paged_attention(q.reshape(B * T, 8, 128), kc, vc, pt, sl, cu_seqlens=cu)
    assert torch.equal(a.reshape(b.shape), b)
    one = q[:, -1]
    c = paged_attention(one, kc, vc, pt, sl)
    assert torch.equal(c, paged_attention(one[:, None], kc, vc, pt, sl)[:, 0])
    _check_paged(c, None, one.cpu(), ks, vs, [1] * B, [6, 100, 257, 900], "bf16")
    # twice the same call: the same bits
    assert torch.equal(c, paged_attention(one, kc, vc, pt, sl))


def test_paged_matches_rows(dev):
    """A prompt in uneven chunks gives what whole-row attention gives."""
    L, Hq, Hkv, D = 700, 4, 2, 128
    kc, vc, pt, sl, cu, ks, vs = _paged(13, [L], [L], Hkv, D, 32, "bf16", dev)
    q = _rows(14, 1, L, Hq, D).to(dev)
    whole = causal_attention(q, ks[0][None].to(dev), vs[0][None].to(dev))
    at, parts = 0, []
    for n in (1, 250, 3, 400, 46):
        parts.append(paged_attention(q[:, at:at + n], kc, vc, pt, torch.tensor([at + n], dtype=torch.int32, device=dev)))
        at += n
    got = torch.cat(parts, 1)
    _check_rows(got, None, q.cpu(), ks[0][None], vs[0][None], "bf16")
    assert (got.float() - whole.float()).norm() <= 2.0 ** -8 * whole.float().norm()


@pytest.mark.parametrize("odd", [math.nan, math.inf])
def test_paged_hidden_infinities(dev, odd):
    """Later tokens of the same call that are not finite do not reach earlier ones."""
    new, lens = [20], [150]
    kc, vc, pt, sl, cu, ks, vs = _paged(15, new, lens, 1, 128, 16, "bf16", dev, junk=odd)
    q = _rows(16, 20, 4, 128).to(dev)
    base = paged_attention(q, kc, vc, pt, sl, cu_seqlens=cu)
    pg, at = int(pt[0, 140 // 16]), 140 % 16   # the 11th new token
    vc[pg, at] = odd
    out = paged_attention(q, kc, vc, pt, sl, cu_seqlens=cu)
    assert torch.equal(out[:10], base[:10])
    assert not torch.isfinite(out[10:]).any()
