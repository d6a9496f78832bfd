"""MI355X (gfx950)-native video-DiT attention hot path.

Hand-written HIP kernels (``csrc/``) behind the C ABI in ``include/avattn.h``
(``libavattn.so``), with host modules that mirror the reference's Python
interfaces:

* :mod:`avgen_amd.attention` — ``attention`` / ``key_padding_mask`` (drop-in
  for ``avgen.models.attention``), the fused ``rotary_attention``, and
  ``scored_attention`` (scores capped by a tanh or biased by distance, with
  document, causal and prefix windows, also for a few queries on a cache);
* :mod:`avgen_amd.rope` — 3D RoPE tables and rotation (``avgen.models.rope``),
  and the rotation of token sequences by integer positions;
* :mod:`avgen_amd.layers` — a block's q/k norm with rotation, and its residual
  addition with the RMS norm behind it (also to e4m3, or gated and modulated);
* :mod:`avgen_amd.cache` — a paged key/value cache for serving, bf16 or e4m3:
  ``append_paged`` (rotating on the way) and ``paged_attention``;
* :mod:`avgen_amd.ring` — ring local step, LSE merger, emulated ring;
* :mod:`avgen_amd.context` — contiguous context-parallel shard rules;
* :mod:`avgen_amd.ops`, :mod:`avgen_amd.scored_ops`, :mod:`avgen_amd.block_ops`,
  :mod:`avgen_amd.gated_ops`, :mod:`avgen_amd.cache_ops` — the ``torch.library``
  ops over the C ABI.
"""

from . import attention, block_ops, cache, cache_ops, context, gated_ops, layers, ops, ring, rope, scored_ops
from .attention import attention as attention_fn
from .attention import document_windows, key_padding_mask, rotary_attention, scored_attention
from .cache import PagedCache, append_paged, paged_attention
from .layers import add_rms_norm, add_rms_norm_fp8, gated_add_rms_norm
from .ring import SDPAMerger, flash_attention_backward_op, flash_attention_op, ring_attention
from .rope import (
    PositionScaling,
    RotaryEmbedding,
    RotaryTables,
    apply_rotary,
    build_position_tables,
    build_rotary_tables,
    rope_axis_pairs,
    rotate_heads,
    rotate_query_key,
)

__all__ = [
    "PagedCache",
    "PositionScaling",
    "RotaryEmbedding",
    "RotaryTables",
    "SDPAMerger",
    "add_rms_norm",
    "add_rms_norm_fp8",
    "append_paged",
    "apply_rotary",
    "attention",
    "attention_fn",
    "block_ops",
    "build_position_tables",
    "build_rotary_tables",
    "cache",
    "cache_ops",
    "context",
    "document_windows",
    "flash_attention_backward_op",
    "flash_attention_op",
    "gated_add_rms_norm",
    "gated_ops",
    "key_padding_mask",
    "layers",
    "ops",
    "paged_attention",
    "ring",
    "ring_attention",
    "rope",
    "rope_axis_pairs",
    "rotary_attention",
    "rotate_heads",
    "rotate_query_key",
    "scored_attention",
    "scored_ops",
]
