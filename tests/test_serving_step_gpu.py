"""The serving operators as a server runs them: the fused store against its parts, and
whole steps with drafted trees against whole rows, eagerly and out of a graph."""

import pytest
import torch

from deltanet_tpu_amd import (
    apply_rotary, causal_attention, norm_rotary, page_pool, paged_kv_append, paged_kv_keep, paged_qkv_append, paged_reserve,
    paged_slots, paged_tree_attention, rotary_table)
from tests import attn_ref as A
from tests import serving_ref as S
from tests.test_attention_gpu import _near, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,ct", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f32"), ("bf16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("D,R,page,hf,inter", [(128, 128, 16, False, False), (256, 64, 64, True, True), (64, 0, 1, False, False), (80, 20, 8, True, False),
                                               (96, 32, 4, False, True)])
@pytest.mark.parametrize("norm", [False, True])
def test_qkv_append(dev, dt, ct, D, R, page, hf, inter, norm):
    """Queries out, keys and values in the cache, each against float64; slots that are
    none, tokens that are none; nothing else of the cache changes."""
    N, Hq, Hkv, pages = 43, 6, 2, 70
    x = _rows(1, N, Hq + 2 * Hkv, D, dt=dt)
    g = torch.Generator().manual_seed(2)
    slots = torch.randperm(pages * page, generator=g)[:N]
    pos = torch.randint(0, 300, (N,), generator=g)
    slots[3], slots[5], pos[7], pos[8] = -1, pages * page, -1, -9
    wq, wk = _rows(3, D, scale=0.3), _rows(4, D, scale=0.3)
    table = rotary_table(300, R, device=dev) if R else None
    caches = [_rows(s, pages, Hkv, page, D, dt=ct).transpose(1, 2) if hf else _rows(s, pages, page, Hkv, D, dt=ct) for s in (5, 6)]
    kc, vc = (c.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if hf else c.contiguous().to(dev) for c in caches)
    xd = x.to(dev)
    kw = dict(q_weight=wq.to(dev), k_weight=wk.to(dev), weight_offset=1.0) if norm else {}
    got = paged_qkv_append(xd[:, :Hq], xd[:, Hq:Hq + Hkv], xd[:, Hq + Hkv:], kc, vc, slots.to(dev), pos.to(dev, torch.int32), table=table,
                           interleaved=inter, **kw)
    cpu = None if table is None else table.cpu()
    some = pos >= 0
    store = some & (slots >= 0) & (slots < pages * page)

    def ref(part, w, to):
        y = part.double()
        if norm:
            return S.normed(y, w.double(), 1e-6, 1.0, pos.clamp_min(0), cpu, inter, to)
        z = A.rotate(y, pos.clamp_min(0), cpu, inter) if R else y
        return z, 2.0 ** -22 * S.pairs(y, R, inter) + 1.01 * A.ROUND[to] * z.abs() + A.TINY[to]

    q, tol = ref(x[:, :Hq], wq, dt)
    assert got.dtype == x.dtype and got.is_contiguous()
    _near(got[some.to(dev)], q[some], tol[some], "q")
    assert not got[~some.to(dev)].any()
    k, tol = ref(x[:, Hq:Hq + Hkv], wk, ct)
    want, wtol = caches[0].double(), torch.zeros(caches[0].shape, dtype=torch.float64)
    at = (slots[store] // page, slots[store] % page)
    want[at], wtol[at] = k[store], tol[store]
    _near(kc, want, wtol, "k")
    want = caches[1].clone()
    want[at] = x[:, Hq + Hkv:][store].to(A.DT[ct])
    assert torch.equal(vc.cpu(), want)


def test_qkv_append_agrees_with_its_parts(dev):
    """Many tokens, rank 4: the bits of norm_rotary and paged_kv_append."""
    B, T, Hq, Hkv, D, R, page = 3, 2000, 8, 2, 128, 64, 16
    q, k, v = (_rows(s, B, T, h, D).to(dev) for s, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    wq, wk = _rows(4, D).to(dev), _rows(5, D).to(dev)
    table = rotary_table(4000, R, device=dev)
    pages = B * T // page
    pt = torch.randperm(pages, generator=torch.Generator().manual_seed(6)).to(torch.int32).view(B, -1).to(dev)
    lens = torch.full((B,), T, dtype=torch.int32, device=dev)
    pos, slots = paged_slots(pt, lens, B * T, page_size=page)
    a, b = ([torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device=dev) for _ in range(2)] for _ in range(2))
    versions = [c._version for c in a]
    out = paged_qkv_append(q, k, v, *a, slots.view(B, T), pos.view(B, T), q_weight=wq, k_weight=wk, table=table)
    assert all(c._version > x for c, x in zip(a, versions))
    qr, kr = norm_rotary(q, k, wq, wk, pos.view(B, T), table)
    paged_kv_append(kr, v, *b, pt, lens)
    assert torch.equal(out, qr) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    out = paged_qkv_append(q, k, v, *a, slots.view(B, T), pos.view(B, T).long(), table=table)
    qr, kr = apply_rotary(q, k, pos.view(B, T), table)
    paged_kv_append(kr, v, *b, pt, lens)
    assert torch.equal(out, qr) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_far_slots(dev):
    """Slots behind 2^32 elements of a cache."""
    pages, page, H, D = 33000, 128, 4, 256
    kc = torch.empty((pages, page, H, D), dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    x = _rows(1, 2, 3 * H, D).to(dev)
    slots = torch.tensor([pages * page - 1, pages * page], device=dev)
    paged_qkv_append(x[:, :H], x[:, H:2 * H], x[:, 2 * H:], kc, vc, slots, torch.zeros(2, dtype=torch.int64, device=dev))
    assert torch.equal(kc[-1, -1], x[0, H:2 * H]) and torch.equal(vc[-1, -1], x[0, 2 * H:])
    starts = torch.tensor([127], dtype=torch.int32, device=dev)
    vc[5, 0] = 3.0
    kept = torch.tensor([[1]], dtype=torch.int32, device=dev)
    pt = torch.tensor([[pages - 1, 5]], dtype=torch.int32, device=dev)
    assert paged_kv_keep(kc, vc, pt, starts, kept).tolist() == [128]
    assert bool((vc[-1, -1] == 3.0).all())


class _Server:
    """One attention layer of random projections; sequences of given tokens' vectors."""

    def __init__(self, dev, B, layers=2, Hq=8, Hkv=2, D=128, R=64, page=16, pages=400, most=40, dt=torch.float32):
        self.B, self.Hq, self.Hkv, self.D, self.page, self.layers = B, Hq, Hkv, D, page, layers
        self.wq, self.wk = _rows(1, D, dt="f32", scale=0.2).to(dev), _rows(2, D, dt="f32", scale=0.2).to(dev)
        self.rotary = rotary_table(1024, R, device=dev)
        self.kc, self.vc = (torch.zeros(layers, pages, page, Hkv, D, dtype=dt, device=dev) for _ in range(2))
        self.pool = page_pool(pages, device=dev)
        self.table = torch.zeros(B, most, dtype=torch.int32, device=dev)
        self.held = torch.zeros(B, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(B, dtype=torch.int32, device=dev)

    def step(self, x, cu, parents, nodes, kept):
        """Projected tokens x (N, layers, Hq + 2 Hkv, D) as trees; the attention of every
        layer, then the tokens in `kept` alone remain."""
        Hq, Hkv = self.Hq, self.Hkv
        starts = self.lens.clone()
        lens = starts + (cu[1:] - cu[:-1])
        short = paged_reserve(self.pool, self.table, self.held, lens, page_size=self.page)
        pos, slots, visible = paged_slots(self.table, lens, x.shape[0], page_size=self.page, cu_seqlens=cu, held=self.held, parents=parents, nodes=nodes)
        outs = []
        for i in range(self.layers):
            q = paged_qkv_append(x[:, i, :Hq], x[:, i, Hq:Hq + Hkv], x[:, i, Hq + Hkv:], self.kc[i], self.vc[i], slots, pos, q_weight=self.wq,
                                 k_weight=self.wk, weight_offset=1.0, table=self.rotary)
            outs.append(paged_tree_attention(q, self.kc[i], self.vc[i], self.table, lens, visible, cu_seqlens=cu))
        self.lens.copy_(paged_kv_keep(self.kc, self.vc, self.table, starts, kept))
        less = paged_reserve(self.pool, self.table, self.held, self.lens, page_size=self.page)
        return torch.stack(outs, 1), short + less


def _plan(seed, B, T, longest):
    """A step's trees, a path of each that is accepted and its tokens."""
    g = torch.Generator().manual_seed(seed)
    new = [int(torch.randint(1, T + 1, (1,), generator=g)) for _ in range(B)]
    parents, seen = S.trees(new, seed)
    paths = []
    for n, m in zip(new, seen):
        leaf = int(torch.randint(0, n, (1,), generator=g))
        paths.append(m[leaf].nonzero().flatten().tolist()[:longest])
    return new, parents, seen, paths


@pytest.mark.parametrize("graph", [False, True])
def test_steps_of_drafted_trees_match_whole_rows(dev, graph):
    """Prompts, then steps of trees of which a path is kept: every node's output is that
    of causal attention over the row of tokens that it sees, in float32 (2e-5: two
    orders of the same sums, normed keys of length sqrt(D))."""
    B, T, steps, longest = 3, 12, 5, 7
    srv = _Server(dev, B)
    H = srv.Hq + 2 * srv.Hkv
    rows = [[] for _ in range(B)]   # the vectors of the tokens kept

    def pad(paths):
        k = torch.full((B, T), -1, dtype=torch.int32)
        for b, p in enumerate(paths):
            k[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        return k.to(dev)

    bufs = dict(x=torch.zeros(B * T, srv.layers, H, srv.D, device=dev), cu=torch.zeros(B + 1, dtype=torch.int32, device=dev),
                parents=torch.zeros(B * T, dtype=torch.int32, device=dev), kept=pad([[]] * B))
    captured = None
    if graph:
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            srv.step(bufs["x"], bufs["cu"], bufs["parents"], T, bufs["kept"])   # (no token: changes nothing)
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            outs = srv.step(bufs["x"], bufs["cu"], bufs["parents"], T, bufs["kept"])
    for t in range(steps):
        new, parents, seen, paths = _plan(t, B, T, longest)
        N = sum(new)
        x = _rows(200 + t, N, srv.layers, H, srv.D, dt="f32")
        bufs["x"][:N].copy_(x)
        bufs["cu"].copy_(torch.tensor([0] + new).cumsum(0))
        bufs["parents"][:N].copy_(torch.tensor(parents))
        bufs["kept"].copy_(pad(paths))
        if graph:
            captured.replay()
            out, short = outs
        else:
            out, short = srv.step(bufs["x"], bufs["cu"], bufs["parents"], T, bufs["kept"])
        assert not short.any() and not out[N:].any()
        at = 0
        for b in range(B):
            for i in range(new[b]):
                mine = rows[b] + [x[at + j] for j in seen[b][i].nonzero().flatten().tolist()]
                row = torch.stack(mine).to(dev)
                for layer in range(srv.layers):
                    y = row[None, :, layer]
                    q, k = norm_rotary(y[:, :, :srv.Hq], y[:, :, srv.Hq:srv.Hq + srv.Hkv], srv.wq, srv.wk,
                                       torch.arange(len(mine), device=dev), srv.rotary, weight_offset=1.0)
                    want = causal_attention(q, k, y[:, :, srv.Hq + srv.Hkv:].contiguous())[0, -1]
                    d = float((out[at + i, layer] - want).abs().max())
                    assert d <= 2e-5, (t, b, i, layer, d)
            rows[b] += [x[at + j] for j in paths[b]]
            at += new[b]
        assert srv.lens.tolist() == [len(r) for r in rows]
        assert srv.held.tolist() == [-(-len(r) // srv.page) for r in rows]
    srv.lens.zero_()
    paged_reserve(srv.pool, srv.table, srv.held, srv.lens, page_size=srv.page)
    assert int(srv.pool[0]) == 400 and sorted(srv.pool[2:].tolist()) == list(range(400))


def test_another_stream(dev):
    """A whole step on a stream of its own, the default stream busy elsewhere."""
    new, parents, _, paths = _plan(9, 2, 20, 5)
    N = sum(new)
    x = _rows(1, N, 2, 12, 128, dt="f32")
    kept = torch.full((2, 8), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        kept[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    cu, par = torch.tensor([0] + new).cumsum(0).to(torch.int32), torch.tensor(parents, dtype=torch.int32)
    a = _Server(dev, 2)
    want, _ = a.step(x.to(dev), cu.to(dev), par.to(dev), 20, kept.to(dev))
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=dev)
    for _ in range(10):
        busy = busy @ busy * 1e-3
    s = torch.cuda.Stream(dev)
    with torch.cuda.stream(s):
        b = _Server(dev, 2)
        out, _ = b.step(x.to(dev), cu.to(dev), par.to(dev), 20, kept.to(dev))
    s.synchronize()
    assert torch.equal(out, want) and torch.equal(a.kc, b.kc) and torch.equal(a.pool, b.pool) and torch.equal(a.lens, b.lens)
