"""Arguments of the attention entries near the ends of their types: CPU only,
nothing is launched."""

import pytest
import torch

from deltanet_tpu_amd import _lib, causal_attention, paged_attention


def _block(cls, **k):
    a = cls()
    a.abi_version = _lib.DN_ABI_VERSION
    for f, v in k.items():
        setattr(a, f, v)
    return a


def _refused(entry, a, match):
    rc = _lib.packed_call(entry)(bytes(a), *([None] if entry == "dn_attention_fwd" else [None, 0, None]))
    assert rc == -1 and match in _lib.load_library().dn_last_error(), (rc, _lib.load_library().dn_last_error())


def test_scales_past_float32():
    x = torch.zeros(1, 4, 2, 64)
    for scale in (1e39, -1e300, float("inf"), float("nan"), 3.4e38):
        with pytest.raises(ValueError, match="finite"):
            causal_attention(x, x, x, scale=scale)
    a = _block(_lib.AttentionArgs, B=1, L=1, Hq=1, Hkv=1, D=64, scale=3.4e38)
    _refused("dn_attention_fwd", a, b"scale")


def test_counts_next_to_32_bits():
    """Sequences, rows and documents whose last step would pass 2^31 are refused;
    windows up to there are not, and change no plan."""
    ptr = dict(q=0x1000, k_cache=0x1000, v_cache=0x1000, out=0x1000, page_table=0x1000, seq_lens=0x1000)
    a = _block(_lib.PagedAttentionArgs, N=2, B=2, Hq=4, Hkv=2, D=128, dtype=1, scale=1.0, pages=64, page_size=64, max_pages=(1 << 25) - 8, **ptr)
    _refused("dn_paged_attention", a, b"2^31 - 1024 tokens")
    a.max_pages = 64
    size = lambda: _lib.packed_call("dn_paged_attention_workspace_size")(bytes(a))
    plain = size()
    assert plain > 0
    for a.window in (4096, 4097, (1 << 31) - 1):
        assert size() == plain
    t = _block(_lib.AttentionArgs, B=1, L=(1 << 31) - 1024, Hq=1, Hkv=1, D=64, scale=1.0)
    _refused("dn_attention_fwd", t, b"too many query rows")
    lib = _lib.load_library()
    assert lib.dn_document_starts(0x1000, _lib.DN_I32, 0, 1, (1 << 31) - 1024, 0x1000, None) == -1


def test_windows_of_any_size_pack():
    from deltanet_tpu_amd.attention import _window
    assert [_window(w) for w in (None, 1, 2 ** 31 - 1, 2 ** 31, 2 ** 40)] == [0, 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]
