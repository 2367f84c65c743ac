"""Refusals of the attention entry points: CPU only, nothing is launched."""

import pytest
import torch

from deltanet_tpu_amd import apply_rotary, causal_attention, paged_attention, paged_kv_append, rotary_table

BF = torch.bfloat16


def z(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


def i32(*s):
    return torch.zeros(*s, dtype=torch.int32)


def refuses(match, f, *a, error=ValueError, **k):
    with pytest.raises(error, match=match):
        f(*a, **k)


def test_rotary_table_refusals():
    for kw, match in (({"rotary_dim": 7}, "even"), ({"rotary_dim": 0}, "even"), ({"max_position": 0}, "at least 1"), ({"base": 0.0}, "base"),
                      ({"scaling": {"type": "linear", "factor": 0.5}}, "at least 1"), ({"scaling": {"type": "linear"}}, "at least 1"),
                      ({"scaling": {"type": "other", "factor": 2}}, "'linear', 'ntk' or 'yarn'"),
                      ({"scaling": {"type": "yarn", "factor": 2}}, "original_max_position"),
                      ({"scaling": {"type": "ntk", "factor": 2}, "rotary_dim": 2}, "at least 4"),
                      ({"scaling": {"type": "yarn", "factor": 2, "original_max_position": 8, "beta_fast": 1, "beta_slow": 2}}, "beta_fast")):
        refuses(match, rotary_table, **{"max_position": 4, "rotary_dim": 8, "device": "cpu", **kw})


def test_rotary_refusals():
    t = rotary_table(8, 16, device="cpu")
    pos = torch.zeros(2, 4, dtype=torch.int64)
    q, k = z(2, 4, 3, 32), z(2, 4, 1, 32)
    refuses("rank 3", apply_rotary, z(4, 32), None, pos, t)
    refuses("float32, bfloat16 or float16", apply_rotary, q.double(), None, pos, t)
    refuses("must match q", apply_rotary, q, k.float(), pos, t)
    refuses("must match q", apply_rotary, q, z(2, 4, 1, 64), pos, t)
    refuses("must match q", apply_rotary, q, z(2, 5, 1, 32), pos, t)
    refuses("at most the head dimension", apply_rotary, z(2, 4, 3, 8), None, pos, t)
    refuses("contiguous float32", apply_rotary, q, k, pos, t.double())
    refuses("contiguous float32", apply_rotary, q, k, pos, t.T)
    refuses("int32 or int64", apply_rotary, q, k, pos.float(), t)
    refuses("only on a ROCm GPU", apply_rotary, q, k, pos, t, error=RuntimeError)


def test_append_refusals():
    kc, pt, lens = z(4, 16, 2, 64), i32(3, 2), i32(3)
    k = z(3, 2, 64)
    ok = (k, k, kc, kc, pt, lens)
    sub = lambda i, x: ok[:i] + (x,) + ok[i + 1:]
    refuses("pages, page_size", paged_kv_append, *sub(2, z(4, 16, 2)))
    refuses("contiguous channels", paged_kv_append, *sub(2, z(4, 16, 64, 2).transpose(2, 3)))
    refuses("must match k_cache", paged_kv_append, *sub(3, z(5, 16, 2, 64)))
    refuses("power of two", paged_kv_append, k, k, z(4, 12, 2, 64), z(4, 12, 2, 64), pt, lens)
    refuses("one shape", paged_kv_append, *sub(1, z(3, 2, 32)))
    refuses("one shape", paged_kv_append, *sub(1, k.float()))
    refuses("heads and channels", paged_kv_append, z(3, 4, 64), z(3, 4, 64), kc, kc, pt, lens)
    refuses("only on a ROCm GPU", paged_kv_append, *ok, error=RuntimeError)


def test_attention_refusals():
    q, k = z(1, 8, 4, 128), z(1, 8, 2, 128)
    refuses("4D", causal_attention, z(8, 4, 128), k, k)
    refuses("Key tensor", causal_attention, q, z(1, 7, 2, 128), z(1, 7, 2, 128))
    refuses("Value tensor", causal_attention, q, k, z(1, 8, 4, 128))
    refuses("one type", causal_attention, q, k.float(), k)
    refuses("64, 128 or 256", causal_attention, z(1, 8, 4, 96), z(1, 8, 2, 96), z(1, 8, 2, 96))
    refuses("divisible", causal_attention, q, z(1, 8, 3, 128), z(1, 8, 3, 128))
    refuses("float32, bfloat16 or float16", causal_attention, q.double(), k.double(), k.double())
    for w in (0, -1, 1.5, True):
        refuses("window", causal_attention, q, k, k, window=w)
    refuses("concrete float", causal_attention, q, k, k, scale="x")
    refuses("finite", causal_attention, q, k, k, scale=float("nan"))
    refuses("only on a ROCm GPU", causal_attention, q, k, k, error=RuntimeError)
    kc = z(4, 16, 2, 128)
    refuses("channels and type", paged_attention, z(3, 4, 64), kc, kc, i32(3, 2), i32(3))
    refuses("channels and type", paged_attention, z(3, 4, 128).float(), kc, kc, i32(3, 2), i32(3))
    refuses("power of two", paged_attention, z(3, 4, 128), z(4, 24, 2, 128), z(4, 24, 2, 128), i32(3, 2), i32(3))


def test_page_arguments():
    from deltanet_tpu_amd.attention import _check_pages
    x, pt, lens = z(3, 4, 128), i32(3, 2), i32(3)
    assert _check_pages(pt, lens, None, x, "q") == (3, 3, 512, 512)
    assert _check_pages(pt, lens, None, z(3, 5, 4, 128), "q") == (3, 15, 2560, 512)
    assert _check_pages(pt, lens, i32(4), z(9, 4, 128), "q") == (3, 9, 512, 512)
    refuses("page_table", _check_pages, pt.long(), lens, None, x, "q")
    refuses("page_table", _check_pages, i32(2, 3).T, lens, None, x, "q")
    refuses("seq_lens", _check_pages, pt, i32(4), None, x, "q")
    refuses("seq_lens", _check_pages, pt, lens.long(), None, x, "q")
    refuses("one token per sequence", _check_pages, pt, lens, None, z(4, 4, 128), "q")
    refuses("cu_seqlens must be", _check_pages, pt, lens, i32(3), z(9, 4, 128), "q")
    refuses("goes with", _check_pages, pt, lens, i32(4), z(3, 5, 4, 128), "q")
    refuses("batch dimension", _check_pages, pt, lens, None, z(2, 5, 4, 128), "q")
    refuses("rank 3", _check_pages, pt, lens, None, z(3, 4), "q")
