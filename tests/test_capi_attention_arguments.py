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
