"""Ops of attention with changed scores: capped by a tanh, biased by distance.

``flash_fwd_scored`` / ``flash_bwd_scored`` (namespace ``avgen_amd``) extend
``flash_fwd(_windowed)`` of :mod:`avgen_amd.ops` with ``softcap``, ``slopes`` and
the queries' offset; checks, strides, workspaces, streams and errors are those
of that module.  bf16 and float32; differentiable in q, k and v.
"""

from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .block_ops import _on, _one_device
from .ops import (
    _alloc_bwd_workspace,
    _check_qkv,
    _check_windows,
    _direct,
    _ds_budget,
    _f32_ready,
    _grad_direct,
    _kernel_ready,
    _normalise_mask,
    _one_pass_workspace,
    _out_or_new,
    _ptr,
    _require_gpu,
    _stream,
    _strides3,
    _workspace,
    compact_ds_table,
    ds_bytes_per_pair,
    f32_ds_bytes_per_pair,
)

__all__ = ["MAX_OFFSET", "MAX_SLOPE_GROUP", "MAX_SOFTCAP_BF16", "flash_bwd_scored", "flash_fwd_scored"]

#: Largest magnitude of a query offset, and most query heads per kv head with
#: slopes (``avattn_fwd_scored``).
MAX_OFFSET = 1 << 30
MAX_SLOPE_GROUP = 64
#: Largest cap of bfloat16 calls (float32: any).
MAX_SOFTCAP_BF16 = 1024.0

# Largest row stride of k and v the kernels for few query rows address.
_MAX_ROW_STRIDE = 1 << 23


def _check_scored(name, q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset):
    """The arguments both directions share: (lo, hi, window stride, mask, mask
    stride, slopes, offsets)."""
    _check_qkv(name, q, k, v, allow_f32=True)
    B, Hq, Lq, _ = q.shape
    if not (math.isfinite(scale) and scale > 0.0):
        raise ValueError(f"{name}: scale must be positive and finite; got {scale}")
    if not (math.isfinite(softcap) and softcap >= 0.0):
        raise ValueError(f"{name}: softcap must be finite and >= 0 (0: none); got {softcap}")
    if q.dtype is torch.bfloat16 and softcap > MAX_SOFTCAP_BF16:
        raise ValueError(f"{name}: softcap {softcap} exceeds {MAX_SOFTCAP_BF16} (bfloat16)")
    if abs(offset) > MAX_OFFSET:
        raise ValueError(f"{name}: query offset {offset} exceeds {MAX_OFFSET}")
    if slopes is not None:
        if slopes.shape != (Hq,):
            raise ValueError(f"{name}: slopes must have one entry per query head ({Hq},); got {tuple(slopes.shape)}")
        if slopes.dtype is not torch.float32:
            raise TypeError(f"{name}: slopes must be float32; got {slopes.dtype}")
        if Hq // k.shape[1] > MAX_SLOPE_GROUP:
            raise ValueError(f"{name}: slopes take at most {MAX_SLOPE_GROUP} query heads per key head; got "
                             f"{Hq // k.shape[1]}")
        slopes = slopes.contiguous()
    if offsets is not None:
        if offsets.shape != (B,):
            raise ValueError(f"{name}: query offsets must be ({B},); got {tuple(offsets.shape)}")
        if offsets.dtype is not torch.int32:
            raise TypeError(f"{name}: query offsets must be int32; got {offsets.dtype}")
        offsets = offsets.contiguous()
    lo = hi = None
    wsb = 0
    if window_lo is not None or window_hi is not None:
        lo, hi, wsb = _check_windows(name, window_lo, window_hi, B, Lq)
    mask, msb = _normalise_mask(name, key_mask, B, k.shape[2])
    _require_gpu(name, q, k, v)
    _one_device(name, q, k, v, lo, hi, mask, slopes, offsets)
    return lo, hi, wsb, mask, msb, slopes, offsets


def _ready(t: torch.Tensor) -> torch.Tensor:
    return _f32_ready(t) if t.dtype is torch.float32 else _kernel_ready(t)


def _fwd_impl(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone):
    name = "avgen_amd.flash_fwd_scored"
    lo, hi, wsb, mask, msb, slopes, offsets = _check_scored(
        name, q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset)
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    f32 = q.dtype is torch.float32
    q, k, v = _ready(q), _ready(k), _ready(v)
    k, v = (t if t.stride(2) < _MAX_ROW_STRIDE else t.contiguous() for t in (k, v))
    out = _ready(torch.empty_like(q, memory_format=torch.preserve_format))
    lse = torch.empty((B, Hq, Lq), device=q.device, dtype=torch.float32)
    lib = _lib.load()
    ws = _workspace(lib.avattn_fwd_scored_workspace_size(B, Hq, Hkv, Lq, Lk, D, int(f32)), q.device)
    with _on(q.device):
        st = lib.avattn_fwd_scored(
            _ptr(q), _ptr(k), _ptr(v), _strides3(q), _strides3(k), _strides3(v),
            B, Hq, Hkv, Lq, Lk, D, int(f32),
            _ptr(mask), msb, _ptr(lo), _ptr(hi), wsb,
            float(scale), float(softcap), _ptr(slopes), _ptr(offsets), int(offset),
            _lib.SCORED_SORTED_WINDOWS if monotone else 0,
            _ptr(out), _strides3(out), _ptr(lse),
            _ptr(ws), ws.numel(), _stream(q.device))
    _lib.check(st, name)
    return out, lse


def _staged_workspace(B, Hq, Hkv, Lq, Lk, D, f32, windowed, device) -> torch.Tensor:
    """The backward's workspace with (dense) staged dS: as many (batch, kv
    head) pairs per pass as the budget and the allocator have, at least one;
    with all of them in one pass also room for a split grid."""
    lib = _lib.load()
    total = B * Hkv
    per = (f32_ds_bytes_per_pair if f32 else ds_bytes_per_pair)(Hq // Hkv, Lq, Lk)
    pairs = max(1, min(total, _ds_budget(device) // per))
    pairs = -(-total // -(-total // pairs))
    while True:
        if f32:
            staged = lib.avattn_bwd_f32_staged_workspace_size(B, Hq, Hkv, Lq, Lk, int(pairs))
        else:
            staged = lib.avattn_bwd_staged_workspace_size(B, Hq, Hkv, Lq, Lk, D, int(pairs))
        try:
            if pairs == total:
                split = lib.avattn_bwd_scored_workspace_size(B, Hq, Hkv, Lq, Lk, D, int(f32), int(windowed))
                return _one_pass_workspace(split, staged, int(pairs) * per, device)
            return _workspace(staged, device)
        except torch.OutOfMemoryError:
            if pairs == 1:
                raise
            pairs = (pairs + 1) // 2


def _bwd_impl(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
              monotone):
    """``monotone``: the caller guarantees windows non-decreasing in the row
    (otherwise checked here, one host synchronisation).  With windows dS is
    staged densely where all of it fits the budget (no synchronisation), else
    compactly (one, for its size)."""
    name = "avgen_amd.flash_bwd_scored"
    lo, hi, wsb, mask, msb, slopes, offsets = _check_scored(
        name, q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset)
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    f32 = q.dtype is torch.float32
    for label, t in (("grad_out", dout), ("out", out)):
        if t.shape != q.shape or t.dtype is not q.dtype:
            raise ValueError(f"{name}: {label} must be {q.dtype} {tuple(q.shape)}")
    if lse.shape != (B, Hq, Lq) or lse.dtype is not torch.float32:
        raise ValueError(f"{name}: logsumexp must be float32 (batch, heads, queries)")
    _one_device(name, q, dout, out, lse)
    if lo is not None and not monotone and Lq > 1:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{name}: a captured backward cannot check the windows' order; pass monotone=True")
        if bool(((lo[..., 1:] < lo[..., :-1]) | (hi[..., 1:] < hi[..., :-1])).any()):
            raise ValueError(f"{name}: the backward needs window_lo and window_hi non-decreasing along the queries")
    dout, q, k, v, out = (_ready(t) for t in (dout, q, k, v, out))
    lse = lse.contiguous()
    if f32:
        dq, dk, dv = (_f32_ready(torch.empty_like(t)) for t in (q, k, v))
    else:
        dq, dk, dv = (_out_or_new(None, t, name, "gradient") for t in (q, k, v))
    lib = _lib.load()
    table, tsb, units = None, 0, 0
    if 0 in (B, Hq, Lq, Lk):
        ws = _workspace(0, q.device)
    elif (not f32 and lo is not None and B * Hkv * ds_bytes_per_pair(Hq // Hkv, Lq, Lk) > _ds_budget(q.device)
            and not torch.cuda.is_current_stream_capturing()):
        table, units = compact_ds_table(lo, hi, Lq, Lk)
        tsb = 0 if table.shape[0] == 1 else table.shape[1]
        ws = _alloc_bwd_workspace(B, Hq, Hkv, Lq, Lk, D, q.device, stage_ds=True, ds_units=units)
    else:
        ws = _staged_workspace(B, Hq, Hkv, Lq, Lk, D, f32, lo is not None, q.device)
    with _on(q.device):
        st = lib.avattn_bwd_scored(
            _ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse),
            _strides3(dout), _strides3(q), _strides3(k), _strides3(v), _strides3(out),
            B, Hq, Hkv, Lq, Lk, D, int(f32),
            _ptr(mask), msb, _ptr(lo), _ptr(hi), wsb,
            _ptr(table), tsb, units,
            float(scale), float(softcap), _ptr(slopes), _ptr(offsets), int(offset),
            _ptr(dq), _strides3(dq), _ptr(dk), _strides3(dk), _ptr(dv), _strides3(dv),
            _ptr(ws), ws.numel(), _stream(q.device))
    _lib.check(st, name)
    return dq, dk, dv


@torch.library.custom_op("avgen_amd::flash_fwd_scored", mutates_args=())
def _fwd_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window_lo: Optional[torch.Tensor],
    window_hi: Optional[torch.Tensor], key_mask: Optional[torch.Tensor], slopes: Optional[torch.Tensor],
    offsets: Optional[torch.Tensor], scale: float, softcap: float, offset: int, monotone: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Forward of attention with changed scores: ``(out, lse)``."""
    return _fwd_impl(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone)


@_fwd_op.register_fake
def _(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone=False):
    return torch.empty_like(q), q.new_empty((q.shape[0], q.shape[1], q.shape[2]), dtype=torch.float32)


@torch.library.custom_op("avgen_amd::flash_bwd_scored", mutates_args=())
def _bwd_op(
    dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
    window_lo: Optional[torch.Tensor], window_hi: Optional[torch.Tensor], key_mask: Optional[torch.Tensor],
    slopes: Optional[torch.Tensor], offsets: Optional[torch.Tensor], scale: float, softcap: float, offset: int,
    monotone: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward of ``flash_fwd_scored``: ``(dq, dk, dv)``."""
    return _bwd_impl(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
                     monotone)


@_bwd_op.register_fake
def _(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
      monotone=False):
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)


def flash_fwd_scored(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
                     monotone=False) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention whose scores ``s = scale q.k`` become ``softcap tanh(s /
    softcap)`` (0: none), lose ``slopes[h] |i + offset - j|`` (None: nothing;
    ``offsets`` int32 per batch row in place of ``offset``) and are masked by
    key windows and ``key_mask`` (each may be None): ``(out, lse)``."""
    return _direct(_FlashFwdScored, _fwd_op, _fwd_impl,
                   (q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone),
                   (q, k, v, window_lo, window_hi, key_mask, slopes, offsets))


def flash_bwd_scored(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
                     monotone=False):
    """``(dq, dk, dv)`` of :func:`flash_fwd_scored` (windows non-decreasing in
    the row; checked unless ``monotone``)."""
    args = (dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone)
    if _grad_direct(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets):
        return _bwd_impl(*args)
    return _bwd_op(*args)


def _setup(ctx, inputs, output):
    q, k, v, lo, hi, mask, slopes, offsets, ctx.scale, ctx.softcap, ctx.offset, ctx.monotone = inputs
    out, lse = output
    ctx.save_for_backward(q, k, v, out, lse, lo, hi, mask, slopes, offsets)
    ctx.mark_non_differentiable(lse)


def _backward(ctx, dout, _dlse):
    q, k, v, out, lse, lo, hi, mask, slopes, offsets = ctx.saved_tensors
    grads = flash_bwd_scored(dout, q, k, v, out, lse, lo, hi, mask, slopes, offsets, ctx.scale, ctx.softcap,
                             ctx.offset, ctx.monotone)
    return (*grads,) + (None,) * 9


torch.library.register_autograd("avgen_amd::flash_fwd_scored", _backward, setup_context=_setup)


class _FlashFwdScored(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        result = _fwd_impl(*args)
        ctx.set_materialize_grads(False)
        _setup(ctx, args, result)
        return result

    @staticmethod
    def backward(ctx, dout, _dlse):
        return (None,) * 12 if dout is None else _backward(ctx, dout, None)
