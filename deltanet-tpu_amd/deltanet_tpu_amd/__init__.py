"""deltanet_tpu_amd: MI355X-native (gfx950 HIP) drop-in for the forward
delta-rule recurrence core of maelie-labs/deltanet-tpu (chunk_gdn2,
gdn2_decode_step and their variants).  See ``gdn2.py`` for the API, and
``attention.py`` and ``serving.py`` for the softmax-attention layers of a hybrid
model."""

from .attention import apply_rotary, causal_attention, norm_rotary, paged_attention, paged_kv_append, rotary_table
from .gdn2 import chunk_gdn2, gdn2_decode_step, gdn2_decode_steps
from .serving import page_pool, paged_kv_keep, paged_qkv_append, paged_reserve, paged_slots, paged_tree_attention
from .variants import (
    chunk_delta_rule,
    chunk_gdn,
    chunk_gla,
    chunk_kda,
    delta_rule_decode_step,
    gdn_decode_step,
    gla_decode_step,
    kda_decode_step,
)

__version__ = "0.3.0+mi355x.1"

__all__ = [
    "chunk_gdn2",
    "gdn2_decode_step",
    "gdn2_decode_steps",
    "chunk_gdn",
    "gdn_decode_step",
    "chunk_kda",
    "kda_decode_step",
    "chunk_gla",
    "gla_decode_step",
    "chunk_delta_rule",
    "delta_rule_decode_step",
    "rotary_table",
    "apply_rotary",
    "norm_rotary",
    "paged_kv_append",
    "paged_attention",
    "causal_attention",
    "page_pool",
    "paged_reserve",
    "paged_slots",
    "paged_qkv_append",
    "paged_tree_attention",
    "paged_kv_keep",
    "__version__",
]
