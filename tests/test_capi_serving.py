"""The serving entries' argument blocks have the C layout, packed or as structs, and the
C entries refuse bad ones before any launch.  CPU only."""

import ctypes
import os
import subprocess

from deltanet_tpu_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCKS = {"dn_norm_rotary_args": (_lib.NormRotaryArgs, _lib.NORM_ROTARY_PACK), "dn_norm_rotary_grads": (_lib.NormRotaryGrads, _lib.NORM_ROTARY_GRADS_PACK),
          "dn_qkv_append_args": (_lib.QkvAppendArgs, _lib.QKV_APPEND_PACK), "dn_paged_reserve_args": (_lib.PagedReserveArgs, _lib.PAGED_RESERVE_PACK), "dn_paged_slots_args": (_lib.PagedSlotsArgs, _lib.PAGED_SLOTS_PACK),
          "dn_kv_keep_args": (_lib.KvKeepArgs, _lib.KV_KEEP_PACK)}


def test_argument_blocks_match_the_header(tmp_path):
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "deltanet_amd.h"', "int main(void){"]
    for cname, (cls, _) in BLOCKS.items():
        src.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        src += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src.append('printf("most sequences %d\\n", DN_MAX_SEQUENCES);')
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(src + ["return 0;}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, f, n = line.split()
        if cname == "most":
            assert int(n) == _lib.MAX_SEQUENCES
            continue
        cls = BLOCKS[cname][0]
        assert (ctypes.sizeof(cls) if f == "size" else getattr(cls, f).offset) == int(n), line


def test_packed_blocks_match_the_structs():
    for cls, pack in BLOCKS.values():
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
    err, P = lib.dn_last_error, _lib.packed_call
    V = _lib.DN_ABI_VERSION
    n = _set(_lib.NormRotaryArgs(), abi_version=V, B=1, L=1, Hq=1, D=8, R=3, dtype=1, weight_dtype=1, pos_dtype=3)
    refused = lambda match: P("dn_norm_rotary")(bytes(n), None) == -1 and match in err()
    assert refused(b"even")
    n.R = 0
    assert refused(b"missing")
    n.eps = -1.0
    assert refused(b"eps")
    n.eps, n.weight_dtype = 0.0, 3
    assert refused(b"dtype")
    n.weight_dtype, n.Hq = 1, 20000
    assert refused(b"heads")
    n.Hq, n.q, n.q_weight = 1, 0x1000, 0x1000
    g = _lib.NormRotaryGrads()
    need = P("dn_norm_rotary_bwd_workspace_size")(bytes(n))
    assert need > 0
    assert P("dn_norm_rotary_bwd")(bytes(n), bytes(g), None, need, None) == -1 and b"missing" in err()
    g.d_q = g.dq = 0x1000
    assert P("dn_norm_rotary_bwd")(bytes(n), bytes(g), 0x1000, need - 1, None) == -2
    n.L = 0
    assert P("dn_norm_rotary")(bytes(n), None) == 0 and P("dn_norm_rotary_bwd_workspace_size")(bytes(n)) == 0
    n.abi_version = 9
    assert P("dn_norm_rotary")(bytes(n), None) == -4

    a = _set(_lib.QkvAppendArgs(), abi_version=V, B=1, L=1, Hq=1, Hkv=1, D=64, dtype=1, cache_dtype=1, weight_dtype=1, pos_dtype=3, pages=1, page_size=3)
    assert P("dn_qkv_append")(bytes(a), None) == -1 and b"power of two" in err()
    a.page_size = 4
    assert P("dn_qkv_append")(bytes(a), None) == -1 and b"missing" in err()
    for f in ("q", "k", "v", "q_out", "k_cache", "v_cache", "slots", "pos", "q_weight"):
        setattr(a, f, 0x1000)
    assert P("dn_qkv_append")(bytes(a), None) == -1 and b"none" in err()
    a.B = 0
    assert P("dn_qkv_append")(bytes(a), None) == 0

    ok = dict(abi_version=V, capacity=5, B=2, page_size=16, max_pages=4, pool=0x1000, page_table=0x1000, held=0x1000, lens=0x1000, short_of=0x1000)
    r = lambda **k: P("dn_paged_reserve")(bytes(_set(_lib.PagedReserveArgs(), **{**ok, **k})), None)
    assert r(B=5000) == -1 and b"4096" in err()
    assert r(page_size=12) == -1 and b"power of two" in err()
    assert r(max_pages=1 << 30) == -1 and b"too many pages" in err()
    assert r(pool=None) == -1 and b"missing" in err()
    assert r(B=0) == 0 and r(abi_version=9) == -4

    s = _set(_lib.PagedSlotsArgs(), abi_version=V, N=3, B=2, page_size=16, max_pages=4)
    assert P("dn_paged_slots")(bytes(s), None) == -1 and b"N / B" in err()
    s.N, s.words = 4, 1
    assert P("dn_paged_slots")(bytes(s), None) == -1 and b"words" in err()
    s.parents, s.words = 0x1000, 17
    assert P("dn_paged_slots")(bytes(s), None) == -1 and b"words" in err()
    s.words = 2
    assert P("dn_paged_slots")(bytes(s), None) == -1 and b"missing" in err()

    t = _set(_lib.PagedAttentionArgs(), abi_version=V, N=4, B=2, Hq=2, Hkv=1, D=64, dtype=1, scale=1.0, pages=4, page_size=16, max_pages=4, q=0x1000,
             k_cache=0x1000, v_cache=0x1000, out=0x1000, page_table=0x1000, seq_lens=0x1000)
    tree = lambda words, vis=0x1000: P("dn_paged_tree_attention")(bytes(t), vis, words, None, 0, None)
    assert tree(0) == -1 and tree(17) == -1 and b"words" in err()
    assert tree(1, None) == -1 and b"missing" in err()
    assert tree(1) == -2 and P("dn_paged_tree_attention_workspace_size")(bytes(t), 1) > 0
    t.window = 63
    assert tree(1) == -1 and b"window" in err()
    t.window, t.max_pages, t.N, t.Hkv, t.Hq = 0, 1 << 26, 1 << 20, 8, 64
    assert tree(1) == -1 and b"too many rows" in err()

    k = _set(_lib.KvKeepArgs(), abi_version=V, layers=1, B=1, H=1, D=64, most=2, dtype=1, pages=1, page_size=16, max_pages=1)
    assert P("dn_kv_keep")(bytes(k), None) == -1 and b"missing" in err()
    k.dtype = 3
    assert P("dn_kv_keep")(bytes(k), None) == -1 and b"dtype" in err()
    k.dtype, k.B = 1, 70000
    assert P("dn_kv_keep")(bytes(k), None) == -1 and b"sizes" in err()
    k.B = 0
    assert P("dn_kv_keep")(bytes(k), None) == 0


def test_c_entries_refuse_overlapping_rows_and_too_many_sequences():
    lib = _lib.load_library()
    err, P, V = lib.dn_last_error, _lib.packed_call, _lib.DN_ABI_VERSION
    r = _set(_lib.PagedReserveArgs(), abi_version=V, B=2, page_size=4, max_pages=3, page_table_stride=2, pool=0x1000,
             page_table=0x1000, held=0x1000, lens=0x1000, short_of=0x1000)
    assert P("dn_paged_reserve")(bytes(r), None) == -1 and b"overlap" in err()
    s = _set(_lib.PagedSlotsArgs(), abi_version=V, N=1, B=1 << 24, page_size=4, max_pages=3, cu_seqlens=0x1000)
    assert P("dn_paged_slots")(bytes(s), None) == -1 and b"too many sequences" in err()
