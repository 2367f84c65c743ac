"""Refusals of the pages that sequences have, in the call that moves accepted tokens: CPU only."""

import ctypes

from deltanet_tpu_amd import _lib, paged_kv_keep
from tests.test_attention_validation import i32, refuses, z


def test_keep_refuses_other_pages_held():
    kc, pt, starts, kept = z(4, 16, 2, 64), i32(2, 3), i32(2), i32(2, 5)
    for held in (i32(3), i32(2, 1), i32(2).long(), i32(4)[::2]):
        refuses("held must", paged_kv_keep, kc, kc, pt, starts, kept, held=held)
    refuses("only on a ROCm GPU", paged_kv_keep, kc, kc, pt, starts, kept, held=i32(2), error=RuntimeError)


def test_the_block_ends_with_the_pages_held():
    """Callers built for the block without them are refused by its version."""
    assert _lib.KvKeepArgs.held.offset == ctypes.sizeof(_lib.KvKeepArgs) - 8
    k = _lib.KvKeepArgs()
    k.abi_version, k.layers, k.B, k.H, k.D, k.most, k.dtype, k.pages, k.page_size, k.max_pages = 2, 1, 1, 1, 64, 2, 1, 1, 16, 1
    assert _lib.packed_call("dn_kv_keep")(bytes(k), None) == -4
