"""The word of a page pool that the kernels count in holds nothing that a call needs."""

import pytest
import torch

from deltanet_tpu_amd import page_pool, paged_reserve
from tests import serving_ref as S

pytestmark = pytest.mark.gpu


# one block; a few; the most, of 1024 threads
@pytest.mark.parametrize("B,most,page", [(7, 20, 16), (200, 64, 16), (64, 1024, 4), (3000, 400, 1)])
def test_a_call_finds_anything_in_the_word(dev, B, most, page):
    pages = B * most // 2
    pool, ref, rows = page_pool(pages, device=dev), S.Pool(pages), [[] for _ in range(B)]
    table, held = torch.zeros(B, most, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    g = torch.Generator().manual_seed(B)
    for t, word in enumerate((1, 7, -1, 31, 255, 1 << 9, (5 << 9) + 3, -(1 << 31), 2 ** 31 - 1, 0)):
        pool[1] = word
        lens = torch.randint(0, most * page + 1, (B,), generator=g).tolist()
        short = paged_reserve(pool, table, held, torch.tensor(lens, dtype=torch.int32, device=dev), page_size=page)
        assert short.tolist() == ref.reserve(rows, lens, page, most), t
        assert held.tolist() == [len(r) for r in rows], t
        got = pool.tolist()
        assert got[0] == len(ref.free) and got[1] == 0 and got[2:2 + got[0]] == ref.free, t
        now = table.tolist()
        assert all(now[b][:len(r)] == r for b, r in enumerate(rows)), t
