"""The attention section of ``SelfAttention.forward`` on the gfx950 kernels
(src/avgen/models/layers.py:530-545): everything between the q/k/v
projections and ``out_proj``.

The reference splits heads with ``unflatten(-1, (-1, head_dim)).transpose(1,
2)`` (:496-504), normalises q and k (``q_norm``/``k_norm``, RMSNorm with a
bf16 gain, :106-118), rotates them (``apply_rotary``, :535-536), runs
attention, and flattens ``out.transpose(1, 2)`` for ``out_proj`` (:545) —
a copy, since SDPA's output is ``(batch, heads, seq, dim)``.

Here the head split stays a strided view of the projection output
``(batch, seq, heads*dim)``, the norm and rotation are one HBM pass
(:func:`avgen_amd.ops.qk_norm_rope`) whose output keeps that
``(batch, seq, heads, dim)`` layout, and the attention kernel, which takes
and produces any such layout, writes its output in it too, so the final
``transpose(1, 2).flatten(2)`` is a view: no copy on either side of the
kernel, forward or backward.

:func:`add_rms_norm` is the step between two such sections: the residual
addition with the norm that follows it, in one pass; :func:`gated_add_rms_norm`
is the same with a gate, a norm behind the section and a modulated norm.
"""

from __future__ import annotations

import torch

from . import attention as _attention
from . import block_ops, gated_ops, ops
from .rope import RotaryTables

__all__ = [
    "add_rms_norm",
    "add_rms_norm_fp8",
    "gated_add_rms_norm",
    "qk_norm_rope",
    "self_attention_core",
    "split_heads",
]


def split_heads(projected: torch.Tensor, head_dim: int) -> torch.Tensor:
    """``(batch, seq, heads*head_dim)`` -> ``(batch, heads, seq, head_dim)``
    view (src/avgen/models/layers.py:496-504), no copy."""
    return projected.unflatten(-1, (-1, head_dim)).transpose(1, 2)


def qk_norm_rope(
    x: torch.Tensor, weight: torch.Tensor | None, *, eps: float = 1e-6, tables: RotaryTables | None = None
) -> torch.Tensor:
    """``apply_rotary(rms_norm(x) * weight, tables)`` in one pass
    (src/avgen/models/layers.py:530-536); ``weight`` None: no gain (the
    rotation alone when ``tables`` is also None is :func:`avgen_amd.rope.apply_rotary`).
    Differentiable in ``x`` and ``weight``; the output keeps ``x``'s layout."""
    cos = sin = None
    if tables is not None:
        cos, sin = tables.cos, tables.sin
    return ops.qk_norm_rope(x, weight, float(eps), cos, sin)


def _prepare(x: torch.Tensor, weight, eps, tables):
    if weight is None and tables is None:
        return x
    if weight is None:
        return ops.rope_apply(x, tables.cos, tables.sin, False)
    return qk_norm_rope(x, weight, eps=eps, tables=tables)


def self_attention_core(
    q_proj: torch.Tensor,
    k_proj: torch.Tensor,
    v_proj: torch.Tensor,
    *,
    head_dim: int,
    q_norm_weight: torch.Tensor | None = None,
    k_norm_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    rope: RotaryTables | None = None,
    key_mask: torch.Tensor | None = None,
) -> torch.Tensor:
    """src/avgen/models/layers.py:530-545 between the projections and
    ``out_proj``: split heads, RMSNorm q and k (gains ``q_norm_weight`` /
    ``k_norm_weight``; None = the reference's ``qk_norm=False`` identity),
    rotate both with ``rope``, attend (``key_mask`` as built by
    :func:`avgen_amd.attention.key_padding_mask`; grouped-query when k has
    fewer heads), and flatten the heads back.

    Args:
        q_proj: ``(batch, seq, heads*head_dim)`` bf16 output of ``q_proj``.
        k_proj, v_proj: ``(batch, seq, kv_heads*head_dim)``.

    Returns:
        ``(batch, seq, heads*head_dim)``, ready for ``out_proj`` — a view of
        the attention kernel's output, which is written in that layout.
    """
    q = _prepare(split_heads(q_proj, head_dim), q_norm_weight, eps, rope)
    k = _prepare(split_heads(k_proj, head_dim), k_norm_weight, eps, rope)
    v = split_heads(v_proj, head_dim)
    out = _attention.attention(q, k, v, attn_mask=key_mask, enable_gqa=q.shape[1] != k.shape[1])
    return out.transpose(1, 2).flatten(2)


def add_rms_norm(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(rms_norm(x + residual) * weight, x + residual)`` over the last
    dimension in one pass: a block's residual addition and the norm that
    follows it (src/avgen/models/blocks.py:173-227, layers.py:106-118).

    ``x`` and ``residual`` are bf16 or float32 of one shape ``(..., width)``,
    any width; ``weight (width,)`` in their dtype or float32.  The norm is
    that of the unrounded fp32 sum; both results are rounded once.
    Differentiable in all three (the addends share one gradient)."""
    return block_ops.add_rms_norm(x, residual, weight, float(eps))


def add_rms_norm_fp8(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`add_rms_norm` with the norm in e4m3 for an fp8 projection:
    ``(codes, scale, x + residual)``, ``codes`` float8_e4m3fn and ``scale``
    float32 ``(...)`` with ``norm ~ codes * scale[..., None]``; ``scale`` is the
    row's largest magnitude / 448 (1 for a row of zeros).  For sampling: not
    differentiable."""
    return block_ops.add_rms_norm_fp8(x, residual, weight, float(eps))


def _one_modulation(shape, *given):
    """gate, scale and shift with one shape: a row for each group of consecutive
    rows of ``shape``."""
    first = next((t for t in given if t is not None), None)
    if first is None:
        return given
    if first.ndim == 3 == len(shape) and first.shape[-2] == 1 and first.shape[0] == shape[0]:
        # A row per sample, as a modulation's projection has it.
        if first.shape[-1] == shape[-1] and all(t is None or t.shape == first.shape for t in given):
            return given
    lead = tuple(shape[:-1])
    groups = 0  # leading sizes of x that some of them has a row for each of
    for t in given:
        if t is None:
            continue
        if t.ndim < 1 or t.ndim > len(shape) or t.shape[-1] != shape[-1]:
            raise ValueError(f"gate, scale and shift must broadcast to {tuple(shape)}; got {tuple(t.shape)}")
        skip = len(shape) - t.ndim
        for d, n in enumerate(t.shape[:-1], skip):
            if n != 1 and n != lead[d]:
                raise ValueError(f"gate, scale and shift must broadcast to {tuple(shape)}; got {tuple(t.shape)}")
            if n != 1:
                groups = max(groups, d + 1)
    want = lead[:groups] + (1,) * (len(lead) - groups) + (shape[-1],)
    return tuple(t if t is None or t.shape == want or (groups == 0 and t.numel() == shape[-1] and
                                                       t.shape == first.shape)
                 else t.expand(want) for t in given)


def gated_add_rms_norm(
    x: torch.Tensor,
    residual: torch.Tensor,
    weight: torch.Tensor | None = None,
    *,
    gate: torch.Tensor | None = None,
    scale: torch.Tensor | None = None,
    shift: torch.Tensor | None = None,
    post_weight: torch.Tensor | None = None,
    residual_scale: float = 1.0,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The step between two sections of a block in one pass: with ``h =
    residual_scale * residual + gate * y``, ``y`` being ``x`` or with
    ``post_weight`` ``rms_norm(x) * post_weight``, returns ``(rms_norm(h) *
    weight * (1 + scale) + shift, h)`` (src/avgen/models/blocks.py:173-227: the
    gated residual addition of one branch and the modulated norm of the next).

    ``x`` and ``residual`` are bf16 or float32 of one shape ``(..., width)``, any
    width.  ``weight`` and ``post_weight`` ``(width,)``, in their dtype or
    float32; ``gate``, ``scale`` and ``shift`` broadcast to them, for instance
    ``(width,)``, ``(batch, 1, width)`` (pieces of a modulation's projection, read
    in place) or ``(batch, seq, width)``, all in their dtype or all float32.
    What is None leaves its step out.  The norm is that of the unrounded fp32
    ``h``; both results are rounded once.  Differentiable in every tensor; the
    backward forms ``h`` again from ``x`` and ``residual``, which it keeps.

    Raises:
        ValueError: shapes that do not fit, a negative eps.
        TypeError: other types.
        RuntimeError: a tensor not on the GPU, or not on the same one.
    """
    gate, scale, shift = _one_modulation(x.shape, gate, scale, shift)
    return gated_ops.gated_add_rms_norm(x, residual, weight, post_weight, gate, scale, shift, float(residual_scale),
                                        float(eps))
