"""A server whose pool of pages, or whose page table, is too small for its sequences:
steps as ``serving.py`` gives them, and what every sequence has afterwards."""

import pytest
import torch

from deltanet_tpu_amd import (
    causal_attention, norm_rotary, paged_kv_keep, paged_qkv_append, paged_reserve, paged_slots, paged_tree_attention)
from tests import serving_ref as S
from tests.test_attention_gpu import _rows
from tests.test_serving_step_gpu import _plan, _Server

pytestmark = pytest.mark.gpu


class _Held(_Server):
    def step(self, x, cu, parents, nodes, kept):
        Hq, Hkv = self.Hq, self.Hkv
        starts = self.lens.clone()
        lens = starts + (cu[1:] - cu[:-1])
        short = paged_reserve(self.pool, self.table, self.held, lens, page_size=self.page)
        held = self.held.clone()
        pos, slots, visible = paged_slots(self.table, lens, x.shape[0], page_size=self.page, cu_seqlens=cu, held=self.held, parents=parents, nodes=nodes)
        outs = []
        for i in range(self.layers):
            q = paged_qkv_append(x[:, i, :Hq], x[:, i, Hq:Hq + Hkv], x[:, i, Hq + Hkv:], self.kc[i], self.vc[i], slots, pos, q_weight=self.wq,
                                 k_weight=self.wk, weight_offset=1.0, table=self.rotary)
            outs.append(paged_tree_attention(q, self.kc[i], self.vc[i], self.table, lens, visible, cu_seqlens=cu))
        self.lens.copy_(paged_kv_keep(self.kc, self.vc, self.table, starts, kept, held=self.held))
        paged_reserve(self.pool, self.table, self.held, self.lens, page_size=self.page)
        return torch.stack(outs, 1), short, held


def _whole_rows(srv, mine, layer):
    """The last token's output of causal attention over these tokens' vectors."""
    y = torch.stack(mine).to(srv.kc.device)[None, :, layer]
    q, k = norm_rotary(y[:, :, :srv.Hq], y[:, :, srv.Hq:srv.Hq + srv.Hkv], srv.wq, srv.wk, torch.arange(len(mine), device=y.device), srv.rotary, weight_offset=1.0)
    return causal_attention(q, k, y[:, :, srv.Hq + srv.Hkv:].contiguous())[0, -1]


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("pages,most", [(9, 40), (40, 2)])
def test_a_pool_or_table_that_runs_short(dev, graph, pages, most):
    """Every path is accepted, short or not: a sequence keeps what it has pages for, and
    nobody's tokens change.  Outputs as in whole rows, 2e-5 (two orders of the same sums)."""
    B, T, steps = 4, 12, 14
    srv = _Held(dev, B, pages=pages, most=most)
    H = srv.Hq + 2 * srv.Hkv
    bufs = dict(x=torch.zeros(B * T, srv.layers, H, srv.D, device=dev), cu=torch.zeros(B + 1, dtype=torch.int32, device=dev),
                parents=torch.zeros(B * T, dtype=torch.int32, device=dev), kept=torch.full((B, T), -1, dtype=torch.int32, device=dev))
    run = lambda: srv.step(bufs["x"], bufs["cu"], bufs["parents"], T, bufs["kept"])
    if graph:
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()   # (no token: changes nothing)
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            outs = run()
    rows, pool, table, shorts = [[] for _ in range(B)], S.Pool(pages), [[] for _ in range(B)], 0
    for t in range(steps):
        new, parents, seen, paths = _plan(t, B, T, 7)
        if t == steps - 3:   # one ends, the others take its pages
            rows[1] = []
            srv.lens[1] = 0
        N = sum(new)
        x = _rows(300 + t, N, srv.layers, H, srv.D, dt="f32")
        kept = torch.full((B, T), -1, dtype=torch.int32)
        for b, p in enumerate(paths):
            kept[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        bufs["x"][:N].copy_(x)
        bufs["cu"].copy_(torch.tensor([0] + new).cumsum(0))
        bufs["parents"][:N].copy_(torch.tensor(parents))
        bufs["kept"].copy_(kept)
        if graph:
            captured.replay()
            out, short, held = outs
        else:
            out, short, held = run()
        want = pool.reserve(table, [len(r) + n for r, n in zip(rows, new)], srv.page, most)
        assert short.tolist() == want and held.tolist() == [len(r) for r in table], t
        shorts += sum(map(bool, want))
        at = 0
        for b in range(B):
            room = len(table[b]) * srv.page
            for i in range(new[b]):
                if len(rows[b]) + i >= room:
                    break
                mine = rows[b] + [x[at + j] for j in seen[b][i].nonzero().flatten().tolist()]
                for layer in range(srv.layers):
                    d = float((out[at + i, layer] - _whole_rows(srv, mine, layer)).abs().max())
                    assert d <= 2e-5, (t, b, i, layer, d)
            rows[b] = rows[b] + [x[at + j] for j in paths[b] if len(rows[b]) + j < room]
            at += new[b]
        pool.reserve(table, [len(r) for r in rows], srv.page, most)
        assert srv.lens.tolist() == [len(r) for r in rows], t
    assert shorts >= 5   # (of the pool that is too small)


def test_keep_behind_the_pages_held(dev):
    """Pages behind those held are another sequence's: nothing of them moves."""
    page, H, D = 4, 2, 8
    table = torch.tensor([[0, 1, 5, 6], [5, 6, 7, 8], [9, 2, 3, 4], [10, 11, 12, 13]], dtype=torch.int32, device=dev)
    starts = torch.tensor([5, 3, 1, 0], dtype=torch.int32, device=dev)
    kept = torch.tensor([[1, 2, 4, 5, -1], [2, 4, 9, 12, -1], [3, 7, -1, 0, 0], [1, 2, -1, -1, -1]], dtype=torch.int32, device=dev)
    held = torch.tensor([2, 4, 9, -3], dtype=torch.int32, device=dev)
    kc = torch.arange(14 * page * H * D, dtype=torch.float32, device=dev).view(14, page, H, D)
    vc = -kc
    before = kc.clone()
    lens = paged_kv_keep(kc, vc, table, starts, kept, held=held)
    assert lens.tolist() == [7, 7, 3, 0]
    want = before.clone()
    for b, path in ((0, [1, 2]), (1, [2, 4, 9, 12]), (2, [3, 7])):
        s = int(starts[b])
        for i, j in enumerate(path):
            f, t = s + j, s + i
            want[int(table[b, t // page]), t % page] = before[int(table[b, f // page]), f % page]
    assert torch.equal(kc, want) and torch.equal(vc, -want)
