"""Refusals of the attention entry points and the layout of their argument blocks:
CPU only, nothing is launched."""

import ctypes
import os
import subprocess

import pytest
import torch

from deltanet_tpu_amd import _lib, apply_rotary, causal_attention, paged_attention, paged_kv_append, rotary_table

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
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


def test_argument_blocks_match_the_header(tmp_path):
    fields = {"dn_rotary_args": _lib.RotaryArgs, "dn_kv_append_args": _lib.KvAppendArgs,
              "dn_paged_attention_args": _lib.PagedAttentionArgs, "dn_attention_args": _lib.AttentionArgs}
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "deltanet_amd.h"', "int main(void){"]
    for cname, cls in fields.items():
        src.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        src += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(src + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, f, n = line.split()
        cls = fields[cname]
        assert (ctypes.sizeof(cls) if f == "size" else getattr(cls, f).offset) == int(n), line


def test_packed_blocks_match_the_structs():
    """The packed bytes are the struct's, field by field."""
    for cls, pack in ((_lib.RotaryArgs, _lib.ROTARY_PACK), (_lib.KvAppendArgs, _lib.KV_APPEND_PACK),
                      (_lib.PagedAttentionArgs, _lib.PAGED_ATTENTION_PACK), (_lib.AttentionArgs, _lib.ATTENTION_PACK)):
        a, values = cls(), []
        for f, t in cls._fields_:
            n = getattr(t, "_length_", 0)
            v = [len(values) + i + 1 for i in range(max(n, 1))]
            values += v
            setattr(a, f, t(*v) if n else v[0])
        assert pack(*values) == bytes(a), cls


def _set(a, **k):
    for f, v in k.items():
        setattr(a, f, type(getattr(a, f))(*v) if isinstance(v, tuple) else v)
    return a


def test_c_entries_refuse_before_any_launch():
    lib = _lib.load_library()
    err = lambda: lib.dn_last_error()
    P = _lib.packed_call
    r = _set(_lib.RotaryArgs(), abi_version=_lib.DN_ABI_VERSION, B=1, L=1, Hq=1, D=8, R=3, rows=1, dtype=1, pos_dtype=3)
    assert P("dn_rotary")(bytes(r), None) == -1 and b"even" in err()
    r.R = 4
    assert P("dn_rotary")(bytes(r), None) == -1 and b"missing" in err()
    r.L = 0
    assert P("dn_rotary")(bytes(r), None) == 0
    r.abi_version = 9
    assert P("dn_rotary")(bytes(r), None) == -4
    a = _set(_lib.KvAppendArgs(), abi_version=_lib.DN_ABI_VERSION, N=3, B=2, H=1, D=8, dtype=1, cache_dtype=1, pages=1, page_size=3, max_pages=1)
    assert P("dn_kv_append")(bytes(a), None) == -1 and b"power of two" in err()
    a.page_size = 4
    assert P("dn_kv_append")(bytes(a), None) == -1 and b"N / B" in err()
    a.N = 4
    assert P("dn_kv_append")(bytes(a), None) == -1 and b"missing" in err()
    p = _set(_lib.PagedAttentionArgs(), abi_version=_lib.DN_ABI_VERSION, N=2, B=2, Hq=4, Hkv=2, D=96, dtype=1, pages=1, page_size=16, max_pages=4, scale=1.0)
    call = lambda: P("dn_paged_attention")(bytes(p), None, 0, None)
    size = lambda: P("dn_paged_attention_workspace_size")(bytes(p))
    assert call() == -1 and b"head dimension" in err() and size() == 0
    p.D = 128
    assert call() == -1 and b"missing" in err()
    for f in ("q", "k_cache", "v_cache", "out", "page_table", "seq_lens"):
        setattr(p, f, 0x1000)
    p.Hkv = 3
    assert call() == -1 and b"multiple" in err()
    p.Hkv = 2
    p.q_strides[1] = 4
    assert call() == -1 and b"16 bytes" in err()
    p.q_strides[1] = 512
    assert size() > 0 and call() == -2 and b"workspace" in err()
    p.window = -1
    assert call() == -1 and b"window" in err()
    t = _set(_lib.AttentionArgs(), abi_version=_lib.DN_ABI_VERSION, B=1, L=8, Hq=4, Hkv=2, D=128, dtype=1, scale=1.0)
    assert P("dn_attention_fwd")(bytes(t), None) == -1 and b"missing" in err()
    for f in ("q", "k", "v", "out"):
        setattr(t, f, 0x1000)
    bwd = lambda *x: P("dn_attention_bwd")(bytes(t), *x)
    assert bwd(0x1000, 0x1000, 0x1000, 0x1000, None, 0, None) == -1 and b"missing" in err()   # no lse
    t.lse = 0x1000
    assert bwd(0x1000, 0x1000, 0x1001, 0x1000, None, 0, None) == -1 and b"16 bytes" in err()
    assert bwd(0x1000, 0x1000, 0x1000, 0x1000, None, 0, None) == -2
    assert P("dn_attention_bwd_workspace_size")(bytes(t)) >= 8 * 4 * 4
    t.scale = float("inf")
    assert P("dn_attention_fwd")(bytes(t), None) == -1 and b"scale" in err()
    assert lib.dn_document_starts(None, 0, 1, 1, 1, None, None) == -1
    assert lib.dn_document_starts(None, 3, 1, 0, 1, None, None) == 0
