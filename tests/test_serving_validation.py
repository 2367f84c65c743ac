"""Refusals of the serving operators and of normed heads: CPU only, nothing is launched."""

import torch

from deltanet_tpu_amd import (
    norm_rotary, page_pool, paged_kv_keep, paged_qkv_append, paged_reserve, paged_slots, paged_tree_attention, rotary_table)
from tests.test_attention_validation import i32, refuses, z


def i64(*s):
    return torch.zeros(*s, dtype=torch.int64)


def test_norm_rotary_refusals():
    t, pos = rotary_table(8, 16, device="cpu"), i64(2, 4)
    q, k, w = z(2, 4, 3, 32), z(2, 4, 1, 32), z(32)
    ok = (q, k, w, w, pos, t)
    sub = lambda i, x: ok[:i] + (x,) + ok[i + 1:]
    refuses("rank 3", norm_rotary, *sub(0, z(4, 32)))
    refuses("float32, bfloat16 or float16", norm_rotary, *sub(0, q.double()))
    refuses("must match q", norm_rotary, *sub(1, k.float()))
    refuses("must match q", norm_rotary, *sub(1, z(2, 5, 1, 32)))
    refuses("goes with", norm_rotary, *sub(1, None))
    refuses("goes with", norm_rotary, *sub(3, None))
    refuses("goes with", norm_rotary, *sub(4, None))
    refuses("norm weights", norm_rotary, *sub(2, z(31)))
    refuses("norm weights", norm_rotary, *sub(2, w.float()))
    refuses("norm weights", norm_rotary, *sub(2, z(64)[::2]))
    refuses("at most the head dimension", norm_rotary, z(2, 4, 3, 8), None, z(8), None, pos, t)
    refuses("int32 or int64", norm_rotary, *sub(4, pos.float()))
    for kw, match in (({"eps": -1.0}, "negative"), ({"eps": float("inf")}, "finite"), ({"eps": "x"}, "concrete float"),
                      ({"weight_offset": float("nan")}, "finite")):
        refuses(match, norm_rotary, *ok, **kw)
    refuses("only on a ROCm GPU", norm_rotary, *ok, error=RuntimeError)


def test_pool_and_reserve_refusals():
    pool = page_pool(5, device="cpu")
    assert pool.tolist() == [5, 0, 4, 3, 2, 1, 0] and page_pool(0, device="cpu").tolist() == [0, 0]
    for x in (-1, 1.5, True, 1 << 31):
        refuses("pages must be", page_pool, x, device="cpu")
    ok = (pool, i32(3, 4), i32(3), i32(3))
    sub = lambda i, x: ok[:i] + (x,) + ok[i + 1:]
    for page in (0, 3, -16, 1.0, True, None):
        refuses("power of two", paged_reserve, *ok, page_size=page)
    call = lambda *a: paged_reserve(*a, page_size=16)
    refuses("page_pool", call, *sub(0, pool.long()))
    refuses("page_pool", call, *sub(0, i32(1)))
    refuses("page_table", call, *sub(1, i64(3, 4)))
    refuses("page_table", call, *sub(1, i32(4, 3).T))
    refuses("have a column", call, *sub(1, i32(3, 0)))
    refuses("held", call, *sub(2, i32(4)))
    refuses("lens", call, *sub(3, i32(6)[::2]))
    refuses("at most 4096", call, pool, i32(4097, 1), i32(4097), i32(4097))
    refuses("only on a ROCm GPU", call, *ok, error=RuntimeError)


def test_slots_refusals():
    pt, lens = i32(3, 4), i32(3)
    call = lambda *a, **k: paged_slots(*a, **{"page_size": 16, **k})
    refuses("power of two", call, pt, lens, 3, page_size=12)
    refuses("tokens must be", call, pt, lens, -3)
    refuses("tokens / B", call, pt, lens, 4)
    refuses("tokens / B", call, i32(0, 4), i32(0), 4)
    refuses("seq_lens", call, pt, i32(4), 3)
    refuses("cu_seqlens", call, pt, lens, 3, cu_seqlens=i32(3))
    refuses("held", call, pt, lens, 3, held=i64(3))
    refuses("goes with nodes", call, pt, lens, 3, parents=i32(3))
    refuses("goes with nodes", call, pt, lens, 3, nodes=3)
    refuses("parents must", call, pt, lens, 3, parents=i32(4), nodes=3)
    for n in (0, 1025, 2.0, True):
        refuses("nodes must", call, pt, lens, 3, parents=i32(3), nodes=n)
    refuses("only on a ROCm GPU", call, pt, lens, 3, error=RuntimeError)


def test_qkv_append_refusals():
    kc, q, k, slots, pos, w = z(4, 16, 2, 64), z(3, 4, 64), z(3, 2, 64), i64(3), i32(3), z(64)
    ok = (q, k, k, kc, kc, slots, pos)
    sub = lambda i, x: ok[:i] + (x,) + ok[i + 1:]
    f = paged_qkv_append
    refuses("pages, page_size", f, *sub(3, z(4, 16, 2)))
    refuses("must match k_cache", f, *sub(4, z(5, 16, 2, 64)))
    refuses("power of two", f, q, k, k, z(4, 12, 2, 64), z(4, 12, 2, 64), slots, pos)
    refuses("q must be", f, *sub(0, z(3, 64)))
    refuses("q must be", f, *sub(0, z(3, 4, 32)))
    refuses("q must be", f, *sub(0, q.double()))
    refuses("k must match", f, *sub(1, z(3, 4, 64)))
    refuses("v must match", f, *sub(2, k.float()))
    refuses("slots must", f, *sub(5, i32(3)))
    refuses("slots must", f, *sub(5, i64(6)[::2]))
    refuses("positions must", f, *sub(6, i32(4)))
    refuses("goes with k_weight", f, *ok, q_weight=w)
    refuses("norm weights", f, *ok, q_weight=w, k_weight=z(32))
    refuses("eps", f, *ok, eps=-1.0)
    refuses("at most the head dimension", f, *ok, table=rotary_table(4, 128, device="cpu"))
    refuses("only on a ROCm GPU", f, *ok, error=RuntimeError)


def test_tree_attention_refusals():
    kc, q, pt, lens, vis = z(4, 16, 2, 64), z(6, 4, 64), i32(2, 3), i32(2), i64(6, 2)
    cu = i32(3)
    ok = (q, kc, kc, pt, lens, vis)
    sub = lambda i, x: ok[:i] + (x,) + ok[i + 1:]
    f = lambda *a, **k: paged_tree_attention(*a, **{"cu_seqlens": cu, **k})
    refuses("channels and type", f, *sub(0, q.float()))
    refuses("power of two", f, q, z(4, 24, 2, 64), z(4, 24, 2, 64), pt, lens, vis)
    refuses("64, 128 or 256", f, z(6, 4, 32), z(4, 16, 2, 32), z(4, 16, 2, 32), pt, lens, vis)
    refuses("divisible", f, z(6, 3, 64), kc, kc, pt, lens, vis)
    refuses("have a column", f, *sub(3, i32(2, 0)))
    refuses("cu_seqlens", f, *ok, cu_seqlens=i32(2))
    for bad in (i32(6, 2), i64(5, 2), i64(6, 0), i64(6, 17), i64(6), i64(6, 4)[:, ::2]):
        refuses("visible must", f, *sub(5, bad))
    refuses("take in the 128", f, *ok, window=127)
    refuses("window", f, *ok, window=0)
    refuses("finite", f, *ok, scale=float("inf"))
    refuses("only on a ROCm GPU", f, *ok, error=RuntimeError)


def test_keep_refusals():
    kc, pt, starts, kept = z(4, 16, 2, 64), i32(2, 3), i32(2), i32(2, 5)
    ok = (kc, kc, pt, starts, kept)
    sub = lambda i, x: ok[:i] + (x,) + ok[i + 1:]
    f = paged_kv_keep
    refuses("pages, page_size", f, *sub(0, z(4, 16, 2)))
    refuses("must match k_cache", f, *sub(1, z(4, 16, 2, 32)))
    refuses("have the layers", f, z(3, 4, 16, 2, 64), z(2, 4, 16, 2, 64), pt, starts, kept)
    refuses("pages, page_size", f, z(3, 4, 16, 2, 64), kc, pt, starts, kept)
    refuses("power of two", f, z(4, 12, 2, 64), z(4, 12, 2, 64), pt, starts, kept)
    refuses("starts must", f, *sub(3, i32(3)))
    refuses("kept must", f, *sub(4, i32(2)))
    refuses("kept must", f, *sub(4, i64(2, 5)))
    refuses("only on a ROCm GPU", f, *ok, error=RuntimeError)




def test_rows_of_a_table_that_overlap_are_refused():
    """Pages are written into the rows: a table with one row for all has no place for them."""
    refuses("overlap", paged_reserve, page_pool(5, device="cpu"), i32(1, 4).expand(3, 4), i32(3), i32(3), page_size=16)
    refuses("overlap", paged_reserve, page_pool(5, device="cpu"), i32(9).as_strided((3, 4), (2, 1)), i32(3), i32(3), page_size=16)
