"""Pages, slots and trees of a paged cache, and the accepted tokens' move, against
lists on the CPU: whole numbers and copies, equal to the bit."""

import pytest
import torch

from deltanet_tpu_amd import page_pool, paged_kv_keep, paged_reserve, paged_slots
from tests import attn_ref as A
from tests import serving_ref as S

pytestmark = pytest.mark.gpu


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _rand(seed, lo, hi, n):
    return torch.randint(lo, hi, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("B,page,most,pages", [(1, 1, 3, 2), (1, 64, 40, 30), (7, 16, 12, 40), (64, 16, 40, 1500), (300, 1, 9, 1000), (300, 16, 300, 20000),
                                               (4096, 16, 5, 9000), (1000, 8, 600, 5)])
def test_reserve_follows_the_list(dev, B, page, most, pages):
    """Sequences that grow, shrink, end and come again; a pool that runs short; lengths
    below 0 and past the table."""
    pool, rows, ref = page_pool(pages, device=dev), [[] for _ in range(B)], S.Pool(pages)
    table, held = torch.full((B, most), -5, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    for t in range(8):
        lens = [n if n % 5 else 0 for n in _rand(100 * t + B, -3, (most + 1) * page if t != 3 else max(1, page * most // 4), B)]
        before = table.cpu()
        stale = [r + before[b, len(r):].tolist() for b, r in enumerate(rows)]
        short = paged_reserve(pool, table, held, _i32(lens, dev), page_size=page)
        want = ref.reserve(rows, lens, page, most)
        assert short.tolist() == want, t
        assert held.tolist() == [len(r) for r in rows]
        got = pool.tolist()
        assert got[0] == len(ref.free) and got[1] == 0 and got[2:2 + got[0]] == ref.free, t
        now = table.tolist()
        for b, r in enumerate(rows):
            assert now[b][:len(r)] == r
            assert all(x == y for x, y in zip(now[b][len(r):], stale[b][len(r):]))   # what is not reserved is not written
    assert sorted(ref.free + [x for r in rows for x in r]) == list(range(pages))


def test_growing_and_trimming_leave_the_pool(dev):
    B, page = 100, 16
    pool, held = page_pool(5000, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    table = torch.zeros(B, 40, dtype=torch.int32, device=dev)
    lens = _rand(1, 0, 300, B)
    paged_reserve(pool, table, held, _i32(lens, dev), page_size=page)
    a = pool.clone()
    paged_reserve(pool, table, held, _i32([n + m for n, m in zip(lens, _rand(2, 0, 300, B))], dev), page_size=page)
    assert not torch.equal(a, pool)
    assert not paged_reserve(pool, table, held, _i32(lens, dev), page_size=page).any()
    assert torch.equal(a, pool)


def test_pools_and_tables_that_hold_nonsense(dev):
    """Counts outside their ranges are taken as the nearest inside; nothing is written
    outside pool and table."""
    B, most = 3, 4
    whole = torch.cat([page_pool(6, device=dev), _i32([77] * 4, dev)])
    pool = whole[:8]
    for count, held in ((1 << 30, [0, 9, -4]), (-5, [4, 4, 4]), (6, [4, 4, 4])):
        pool[0] = count
        h, guard = _i32(held, dev), torch.full((B + 2, most + 3), 88, dtype=torch.int32, device=dev)
        table = guard[1:-1, 1:1 + most]
        table.fill_(2)
        paged_reserve(pool, table, h, _i32([20, 1, 0], dev), page_size=16)
        assert all(0 <= x <= most for x in h.tolist()) and 0 <= int(pool[0]) <= 6 and int(pool[1]) == 0
        guard[1:-1, 1:1 + most] = 88
        assert bool((guard == 88).all())
        assert bool((whole[8:] == 77).all())


def _slots_want(table, lens, new, page, held=None):
    pos, slots = [], []
    for b, n in enumerate(new):
        for i in range(n):
            x = lens[b] - n + i
            limit = table.shape[1] if held is None else min(held[b], table.shape[1])
            ok = x >= 0 and x // page < limit and int(table[b, x // page]) >= 0
            pos.append(x)
            slots.append(int(table[b, x // page]) * page + x % page if ok else -1)
    return pos, slots


@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("new,lens", [([1], [1]), ([1] * 70, list(range(1, 71))), ([5, 0, 300, 2], [5, 9, 512, 1]), ([0, 0], [3, 0]), ([3000], [5000])])
def test_slots(dev, page, new, lens):
    B, most = len(new), max(1, max(lens) // page)   # (some lie past the table)
    table = torch.randint(-1, 10 ** 6, (B, most), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    held = _rand(3, 0, most + 3, B)
    N = sum(new)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    for h in (None, held):
        pos, slots = paged_slots(table.to(dev), _i32(lens, dev), N, page_size=page, cu_seqlens=cu.to(dev), held=None if h is None else _i32(h, dev))
        assert (pos.tolist(), slots.tolist()) == _slots_want(table, lens, new, page, h)
    if len(set(new)) == 1:
        pos, slots = paged_slots(table.to(dev), _i32(lens, dev), N, page_size=page)
        assert (pos.tolist(), slots.tolist()) == _slots_want(table, lens, new, page)
    # a batch of fixed size that is not full, tokens in front
    pos, slots = paged_slots(table.to(dev), _i32(lens, dev), N + 9, page_size=page, cu_seqlens=(cu + 4).to(dev))
    want = _slots_want(table, lens, new, page)
    assert pos.tolist() == [-1] * 4 + want[0] + [-1] * 5 and slots.tolist() == [-1] * 4 + want[1] + [-1] * 5


def test_slots_past_32_bits(dev):
    table = torch.tensor([[(1 << 31) - 1]], dtype=torch.int32)
    pos, slots = paged_slots(table.to(dev), _i32([100], dev), 3, page_size=128, cu_seqlens=_i32([0, 3], dev))
    assert pos.tolist() == [97, 98, 99] and slots.tolist() == [((1 << 31) - 1) * 128 + x for x in (97, 98, 99)]


@pytest.mark.parametrize("new,nodes", [([1], 1), ([7, 1, 0, 64, 33], 64), ([65, 3], 65), ([200, 128, 1], 200), ([1024], 1024), ([100, 300], 128)])
@pytest.mark.parametrize("wide", [0, 4])
def test_slots_of_trees(dev, new, nodes, wide):
    """Depths and ancestors; trees longer than `nodes` end there."""
    page = 16
    lens = [n + x for n, x in zip(new, _rand(5, 0, 200, len(new)))]
    table = torch.randint(0, 5000, (len(new), max(lens) // page + 1), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    parents, seen = S.trees(new, 3, wide)
    N, W = sum(new), -(-nodes // 64)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32)
    full = [-7] * 2 + parents + [5] * 3
    pos, slots, visible = paged_slots(table.to(dev), _i32(lens, dev), N + 5, page_size=page, cu_seqlens=(cu + 2).to(dev), parents=_i32(full, dev), nodes=nodes)
    want = _slots_want(table, lens, new, page)
    at, rows, count = [], S.words(seen, W), 0
    for b, n in enumerate(new):
        for i in range(n):
            x = i < 64 * W
            at.append(lens[b] - n + int(seen[b][i].sum()) - 1 if x else -1)
            if not x:
                want[1][count] = -1
                rows[count] = 0
            count += 1
    assert pos.tolist() == [-1] * 2 + at + [-1] * 3
    assert slots.tolist() == [-1] * 2 + want[1] + [-1] * 3
    none = torch.zeros(1, W, dtype=torch.int64)
    assert torch.equal(visible.cpu(), torch.cat([none.expand(2, W), rows, none.expand(3, W)]))


def test_parents_that_are_none(dev):
    """A parent that does not come before its child counts as none: no chain is endless."""
    table = torch.arange(4, dtype=torch.int32, device=dev)[None]
    pos, _, visible = paged_slots(table, _i32([10], dev), 5, page_size=4, cu_seqlens=_i32([0, 5], dev),
                                  parents=_i32([0, 2, 1, 1 << 30, -(1 << 31)], dev), nodes=5)
    assert pos.tolist() == [5, 5, 6, 5, 5] and visible.flatten().tolist() == [1, 2, 6, 8, 16]


@pytest.mark.parametrize("dt,D,heads_first", [("bf16", 128, False), ("f32", 64, True), ("f16", 6, False), ("f32", 5, True), ("bf16", 256, True)])
@pytest.mark.parametrize("layers", [0, 1, 3])
def test_keep(dev, dt, D, heads_first, layers):
    """Every kind of end of a path; what is not kept stays as it was."""
    page, H, most = 4, 3, 70
    starts = [5, 0, 7, 2, 1, 30, 3, -2, 11]
    kept = [[0, 1, 2], [2, 5, 6, 9], [], [3, 3, 4], [0, 2, 1, 5], [1, 90], [4, -1, 6], [0, 1], list(range(1, 140, 2))]
    limit = 40
    g = torch.Generator().manual_seed(1)
    pages = len(starts) * limit
    table = torch.randperm(pages, generator=g).reshape(len(starts), limit).to(torch.int32)
    table[6, 1] = pages + 3   # (its token 4 .. 7: the first move's source)
    shape = (max(layers, 1), pages, page, H, D)
    caches = [torch.randn(shape, generator=g).to(A.DT[dt]) for _ in range(2)]
    want, lens = [c.clone() for c in caches], []
    for b, path in enumerate(kept):
        before, n = -1, 0
        for i, x in enumerate(path):
            if starts[b] < 0 or x <= before or starts[b] + x >= limit * page:
                break
            before, n = x, i + 1
            f, t = starts[b] + x, starts[b] + i
            fp, tp = int(table[b, f // page]), int(table[b, t // page])
            if fp < pages and tp < pages:
                for c, w in zip(caches, want):
                    w[:, tp, t % page] = c[:, fp, f % page]
        lens.append(starts[b] + n)
    put = lambda c: c.transpose(2, 3).contiguous().to(dev).transpose(2, 3) if heads_first else c.to(dev)
    got = [put(c) for c in caches]
    args = got if layers else [c[0] for c in got]
    rows = torch.full((len(kept), most), -1, dtype=torch.int32)
    for b, path in enumerate(kept):
        rows[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
    out = paged_kv_keep(*args, table.to(dev), _i32(starts, dev), rows.to(dev))
    assert out.tolist() == lens
    assert all(torch.equal(c.cpu(), w) for c, w in zip(got, want))


def test_empty_calls(dev):
    z = torch.zeros(0, dtype=torch.int32, device=dev)
    pool = page_pool(0, device=dev)
    assert pool.tolist() == [0, 0]
    assert paged_reserve(pool, z.view(0, 1).new_empty(0, 3), z, z, page_size=16).shape == (0,)
    t = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    assert paged_reserve(pool, t, _i32([0, 0], dev), _i32([0, 17], dev), page_size=16).tolist() == [0, 2]
    assert [x.shape[0] for x in paged_slots(t, _i32([5, 5], dev), 0, page_size=16)] == [0, 0]
    kc = torch.zeros(0, 16, 2, 64, device=dev)
    assert paged_kv_keep(kc, kc, t, _i32([3, 4], dev), _i32([[0], [-1]], dev)).tolist() == [4, 4]
    kc = torch.ones(4, 16, 2, 64, device=dev)
    assert paged_kv_keep(kc, kc.clone(), t, _i32([3, 4], dev), torch.zeros(2, 0, dtype=torch.int32, device=dev)).tolist() == [3, 4]


@pytest.mark.parametrize("tree", [False, True])
def test_slots_of_more_sequences_than_31_bits_of_threads(dev, tree):
    """8.4 million sequences without a new token: all tokens are nobody's."""
    B, N = (1 << 23) + 5, 1000
    extra = {"parents": _i32([-1] * N, dev), "nodes": 3} if tree else {}
    table, lens = torch.zeros(B, 1, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    for at in (0, 400, N):
        cu = torch.full((B + 1,), at, dtype=torch.int32, device=dev)
        got = paged_slots(table, lens, N, page_size=4, cu_seqlens=cu, **extra)
        assert got[0].eq(-1).all() and got[1].eq(-1).all() and not (tree and got[2].any())
