"""The attention entries' argument blocks have the C layout, packed or as structs,
and the C entries refuse bad ones before any launch.  CPU only."""

import ctypes
import os
import subprocess

from deltanet_tpu_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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
    p = _set(_lib.PagedAttentionArgs(), abi_version=_lib.DN_ABI_VERSION, N=2, B=2, Hq=4, Hkv=2, D=96, dtype=1, pages=1, page_size=16, max_pages=64, scale=1.0)
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
