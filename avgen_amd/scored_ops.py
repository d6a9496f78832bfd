"""Ops of attention with changed scores: capped by a tanh, biased by distance.

``flash_fwd_scored`` / ``flash_bwd_scored`` (namespace ``avgen_amd``) extend
``flash_fwd(_windowed)`` of :mod:`avgen_amd.ops` with ``softcap``, ``slopes`` and
the queries' offset; checks, strides, workspaces, streams and errors are those
of that module.  bf16 and float32; differentiable in q, k and v.

With slopes the backward starts from ``row_lse``, the logsumexp without the
constant ``slope * distance`` that the kernels leave out of a row's scores
(``avattn_fwd_scored``): ``lse`` holds that only as float32 does.
``flash_fwd_scored_rows`` is ``flash_fwd_scored`` with it as a third result.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .block_ops import _on, _one_device
from .ops import (
    SUPPORTED_HEAD_DIMS,
    _alloc_bwd_workspace,
    _check_qkv,
    _check_windows,
    _direct,
    _ds_budget,
    _f32_ready,
    _grad_direct,
    _kernel_ready,
    _normalise_mask,
    _ptr,
    _stream,
    _Strides3,
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

_DTYPES = (torch.bfloat16, torch.float32)

# Bound of the row strides of k and v that the kernels for few query rows
# address.
_MAX_ROW_STRIDE = 1 << 23


def _check_scored(name, q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset):
    """The arguments both directions share: (lo, hi, window stride, mask, mask
    stride, slopes, offsets)."""
    shape, kshape, dtype = q.shape, k.shape, q.dtype
    if not (len(shape) == 4 and len(kshape) == 4 and kshape == v.shape and shape[0] == kshape[0]
            and shape[3] == kshape[3] and shape[3] in SUPPORTED_HEAD_DIMS and kshape[1] and shape[1] % kshape[1] == 0
            and dtype in _DTYPES and k.dtype is dtype and v.dtype is dtype):
        _check_qkv(name, q, k, v, allow_f32=True)  # says what is wrong
    B, Hq, Lq, _ = shape
    if not (math.isfinite(scale) and scale > 0.0):
        raise ValueError(f"{name}: scale must be positive and finite; got {scale}")
    if not (math.isfinite(softcap) and softcap >= 0.0):
        raise ValueError(f"{name}: softcap must be finite and >= 0 (0: none); got {softcap}")
    if dtype is torch.bfloat16 and softcap > MAX_SOFTCAP_BF16:
        raise ValueError(f"{name}: softcap {softcap} exceeds {MAX_SOFTCAP_BF16} (bfloat16)")
    if abs(offset) > MAX_OFFSET:
        raise ValueError(f"{name}: query offset {offset} exceeds {MAX_OFFSET}")
    if slopes is not None:
        if slopes.shape != (Hq,):
            raise ValueError(f"{name}: slopes must have one entry per query head ({Hq},); got {tuple(slopes.shape)}")
        if slopes.dtype is not torch.float32:
            raise TypeError(f"{name}: slopes must be float32; got {slopes.dtype}")
        if Hq // kshape[1] > MAX_SLOPE_GROUP:
            raise ValueError(f"{name}: slopes take at most {MAX_SLOPE_GROUP} query heads per key head; got "
                             f"{Hq // kshape[1]}")
        slopes = slopes.contiguous()
    if offsets is not None:
        if offsets.shape != (B,):
            raise ValueError(f"{name}: query offsets must be ({B},); got {tuple(offsets.shape)}")
        if offsets.dtype is not torch.int32:
            raise TypeError(f"{name}: query offsets must be int32; got {offsets.dtype}")
        offsets = offsets.contiguous()
    lo, hi, wsb, mask, msb = _masks(name, window_lo, window_hi, key_mask, B, Lq, kshape[2])
    _one_device(name, q, k, v, lo, hi, mask, slopes, offsets)
    return lo, hi, wsb, mask, msb, slopes, offsets


def _masks(name, window_lo, window_hi, key_mask, B, Lq, Lk):
    lo = hi = None
    wsb = 0
    if window_lo is not None or window_hi is not None:
        lo, hi, wsb = _check_windows(name, window_lo, window_hi, B, Lq)
    return (lo, hi, wsb, *_normalise_mask(name, key_mask, B, Lk))


def _laid_out(t: torch.Tensor, f32: bool):
    """``t`` as the kernels read it, and its strides for the C call."""
    s0, s1, s2, s3 = t.stride()
    if s3 != 1 or (s0 | s1 | s2) % (4 if f32 else 8) or t.data_ptr() % 16:
        t = _f32_ready(t) if f32 else _kernel_ready(t)
        return t, _strides3(t)
    return t, _Strides3(s0, s1, s2)


def _new_like(t: torch.Tensor, laid: torch.Tensor, strides, f32: bool):
    """An output in the layout that the op promises, ``empty_like`` of its input
    ``t`` (read as ``laid``, with these strides): the output, what the kernels
    write (the output, or where they cannot write its layout a tensor to copy from,
    see :func:`_deliver`), and its strides for the C call."""
    o = torch.empty_like(t)
    if t is laid and o.stride() == t.stride():
        return o, o, strides
    written, strides = _laid_out(o, f32)
    return o, written, strides


def _deliver(*outputs):
    """The outputs of ``(output, written, strides)`` triples, as written."""
    for o, written, _ in outputs:
        if written is not o:
            o.copy_(written)
    return tuple(o for o, _, _ in outputs)


# Workspace sizes: functions of a call's sizes alone.
@lru_cache(maxsize=256)
def _fwd_workspace_size(*sizes: int) -> int:
    return _lib.load().avattn_fwd_scored_workspace_size(*sizes)


@lru_cache(maxsize=256)
def _bwd_workspace_size(*sizes: int) -> int:
    return _lib.load().avattn_bwd_scored_workspace_size(*sizes)


@lru_cache(maxsize=256)
def _staged_workspace_size(B, Hq, Hkv, Lq, Lk, D, f32, pairs) -> int:
    lib = _lib.load()
    if f32:
        return lib.avattn_bwd_f32_staged_workspace_size(B, Hq, Hkv, Lq, Lk, pairs)
    return lib.avattn_bwd_staged_workspace_size(B, Hq, Hkv, Lq, Lk, D, pairs)


def _fwd_impl(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone,
              rows=False):
    """``(out, lse)``; with ``rows`` ``(out, lse, row_lse)``, ``row_lse`` being
    ``lse`` itself without slopes."""
    name = "avgen_amd.flash_fwd_scored"
    lo, hi, wsb, mask, msb, slopes, offsets = _check_scored(
        name, q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset)
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    f32 = q.dtype is torch.float32
    given = q
    (q, qs), (k, ks), (v, vs) = _laid_out(q, f32), _laid_out(k, f32), _laid_out(v, f32)
    if ks[2] >= _MAX_ROW_STRIDE or vs[2] >= _MAX_ROW_STRIDE:
        (k, ks), (v, vs) = (_laid_out(t.clone(memory_format=torch.contiguous_format), f32) for t in (k, v))
    o = _new_like(given, q, qs, f32)
    device = q.device
    row_lse = lse = torch.empty((B, Hq, Lq) if slopes is None or not rows else (2, B, Hq, Lq), device=device,
                                dtype=torch.float32)
    flags = _lib.SCORED_SORTED_WINDOWS if monotone else 0
    if lse.ndim == 4:
        flags |= _lib.SCORED_ROW_LSE
        lse, row_lse = lse[0], lse[1]
    ws = _workspace(_fwd_workspace_size(B, Hq, Hkv, Lq, Lk, D, f32), device)
    with _on(device):
        st = _lib.load().avattn_fwd_scored(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), qs, ks, vs, B, Hq, Hkv, Lq, Lk, D, f32,
            _ptr(mask), msb, _ptr(lo), _ptr(hi), wsb,
            scale, softcap, _ptr(slopes), _ptr(offsets), offset, flags,
            o[1].data_ptr(), o[2], lse.data_ptr(), ws.data_ptr(), ws.numel(), _stream(device))
    _lib.check(st, name)
    (out,) = _deliver(o)
    return (out, lse, row_lse) if rows else (out, lse)


@lru_cache(maxsize=256)
def _staged_plan(B, Hq, Hkv, Lq, Lk, D, f32, windowed, budget) -> tuple[int, int]:
    """Of the backward with (dense) staged dS: its (batch, kv head) pairs per
    pass, as many as the budget has, at least one, and its workspace's bytes:
    with all of them in one pass also room for a split grid, if the budget
    covers the parts."""
    total = B * Hkv
    per = (f32_ds_bytes_per_pair if f32 else ds_bytes_per_pair)(Hq // Hkv, Lq, Lk)
    pairs = max(1, min(total, budget // per))
    pairs = -(-total // -(-total // pairs))
    staged = _staged_workspace_size(B, Hq, Hkv, Lq, Lk, D, f32, pairs)
    if pairs == total:
        split = _bwd_workspace_size(B, Hq, Hkv, Lq, Lk, D, f32, windowed)
        if pairs * per + split - staged <= budget:
            return pairs, split
    return pairs, staged


def _staged_workspace(B, Hq, Hkv, Lq, Lk, D, f32, windowed, device) -> torch.Tensor:
    """The workspace of :func:`_staged_plan`; where the allocator has not got
    it, without the room for a split grid, then in passes of half the pairs."""
    pairs, nbytes = _staged_plan(B, Hq, Hkv, Lq, Lk, D, f32, windowed, _ds_budget(device))
    while True:
        try:
            return _workspace(nbytes, device)
        except torch.OutOfMemoryError:
            staged = _staged_workspace_size(B, Hq, Hkv, Lq, Lk, D, f32, pairs)
            if staged >= nbytes:
                if pairs == 1:
                    raise
                pairs = (pairs + 1) // 2
                staged = _staged_workspace_size(B, Hq, Hkv, Lq, Lk, D, f32, pairs)
            nbytes = staged


def _bwd_impl(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
              monotone, row_lse=None, from_forward=False):
    """``row_lse`` (see the module docstring): in place of ``lse``.  ``monotone``: the caller guarantees windows non-decreasing in the row
    (otherwise checked here, one host synchronisation).  With windows dS is
    staged densely where all of it fits the budget (no synchronisation), else
    compactly (one, for its size).  ``from_forward``: the arguments passed the
    forward's checks (the backward of a small call is bound by this function,
    at half speed on autograd's own thread)."""
    name = "avgen_amd.flash_bwd_scored"
    B, Hq, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    f32 = q.dtype is torch.float32
    if from_forward:
        lo, hi, wsb, mask, msb = _masks(name, window_lo, window_hi, key_mask, B, Lq, Lk)
        slopes, offsets = (None if t is None else t.contiguous() for t in (slopes, offsets))
    else:
        lo, hi, wsb, mask, msb, slopes, offsets = _check_scored(
            name, q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset)
        for label, t in (("grad_out", dout), ("out", out)):
            if t.shape != q.shape or t.dtype is not q.dtype:
                raise ValueError(f"{name}: {label} must be {q.dtype} {tuple(q.shape)}")
        for t in (lse, row_lse):
            if t is not None and (t.shape != (B, Hq, Lq) or t.dtype is not torch.float32):
                raise ValueError(f"{name}: logsumexp must be float32 (batch, heads, queries)")
    _one_device(name, q, k, v, dout, out, lse, row_lse, lo, hi, mask, slopes, offsets)
    if lo is not None and not monotone and Lq > 1:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{name}: a captured backward cannot check the windows' order; pass monotone=True")
        if bool(((lo[..., 1:] < lo[..., :-1]) | (hi[..., 1:] < hi[..., :-1])).any()):
            raise ValueError(f"{name}: the backward needs window_lo and window_hi non-decreasing along the queries")
    given = (q, k, v)
    (dout, dos), (q, qs), (k, ks) = _laid_out(dout, f32), _laid_out(q, f32), _laid_out(k, f32)
    (v, vs), (out, os) = _laid_out(v, f32), _laid_out(out, f32)
    stat = (lse if row_lse is None else row_lse).contiguous()
    dq, dk, dv = (_new_like(*t, f32) for t in zip(given, (q, k, v), (qs, ks, vs)))
    device = q.device
    table, tsb, units = None, 0, 0
    if 0 in (B, Hq, Lq, Lk):
        ws = _workspace(0, device)
    elif (not f32 and lo is not None and B * Hkv * ds_bytes_per_pair(Hq // Hkv, Lq, Lk) > _ds_budget(device)
            and not torch.cuda.is_current_stream_capturing()):
        table, units = compact_ds_table(lo, hi, Lq, Lk)
        tsb = 0 if table.shape[0] == 1 else table.shape[1]
        ws = _alloc_bwd_workspace(B, Hq, Hkv, Lq, Lk, D, device, stage_ds=True, ds_units=units)
    else:
        ws = _staged_workspace(B, Hq, Hkv, Lq, Lk, D, f32, lo is not None, device)
    lib = _lib.load()
    with _on(device):
        st = (lib.avattn_bwd_scored if row_lse is None else lib.avattn_bwd_scored_row_lse)(
            dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), stat.data_ptr(),
            dos, qs, ks, vs, os, B, Hq, Hkv, Lq, Lk, D, f32,
            _ptr(mask), msb, _ptr(lo), _ptr(hi), wsb, _ptr(table), tsb, units,
            scale, softcap, _ptr(slopes), _ptr(offsets), offset,
            dq[1].data_ptr(), dq[2], dk[1].data_ptr(), dk[2], dv[1].data_ptr(), dv[2],
            ws.data_ptr(), ws.numel(), _stream(device))
    _lib.check(st, name)
    return _deliver(dq, dk, dv)


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


@torch.library.custom_op("avgen_amd::flash_fwd_scored_rows", mutates_args=())
def _fwd_rows_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window_lo: Optional[torch.Tensor],
    window_hi: Optional[torch.Tensor], key_mask: Optional[torch.Tensor], slopes: torch.Tensor,
    offsets: Optional[torch.Tensor], scale: float, softcap: float, offset: int, monotone: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``flash_fwd_scored`` with slopes: ``(out, lse, row_lse)``."""
    out, lse, row_lse = _fwd_impl(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
                                  monotone, True)
    return out, lse.clone(), row_lse.clone()  # an op's results share no memory


@_fwd_rows_op.register_fake
def _(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone=False):
    row = (q.shape[0], q.shape[1], q.shape[2])
    return torch.empty_like(q), q.new_empty(row, dtype=torch.float32), q.new_empty(row, dtype=torch.float32)


@torch.library.custom_op("avgen_amd::flash_bwd_scored", mutates_args=())
def _bwd_op(
    dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
    window_lo: Optional[torch.Tensor], window_hi: Optional[torch.Tensor], key_mask: Optional[torch.Tensor],
    slopes: Optional[torch.Tensor], offsets: Optional[torch.Tensor], scale: float, softcap: float, offset: int,
    monotone: bool = False, row_lse: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward of ``flash_fwd_scored``: ``(dq, dk, dv)``."""
    return _bwd_impl(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
                     monotone, row_lse)


@_bwd_op.register_fake
def _(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
      monotone=False, row_lse=None):
    return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)


def _fwd_of_rows(*args):
    return _fwd_rows_op(*args)[:2]


def flash_fwd_scored(q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
                     monotone=False) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention whose scores ``s = scale q.k`` become ``softcap tanh(s /
    softcap)`` (0: none), lose ``slopes[h] |i + offset - j|`` (None: nothing;
    ``offsets`` int32 per batch row in place of ``offset``) and are masked by
    key windows and ``key_mask`` (each may be None): ``(out, lse)``."""
    return _direct(_FlashFwdScored, _fwd_op if slopes is None else _fwd_of_rows, _fwd_impl,
                   (q, k, v, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone),
                   (q, k, v, window_lo, window_hi, key_mask, slopes, offsets))


def flash_bwd_scored(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset,
                     monotone=False, row_lse=None):
    """``(dq, dk, dv)`` of :func:`flash_fwd_scored` (windows non-decreasing in
    the row; checked unless ``monotone``).  With slopes and without ``row_lse``
    (of ``flash_fwd_scored_rows``) probabilities are as exact as ``lse``: off by
    up to ``|lse| 2^-24`` relatively."""
    args = (dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, scale, softcap, offset, monotone,
            row_lse)
    if _grad_direct(dout, q, k, v, out, lse, window_lo, window_hi, key_mask, slopes, offsets, row_lse):
        return _bwd_impl(*args)
    return _bwd_op(*args)


def _setup(ctx, inputs, output):
    q, k, v, lo, hi, mask, slopes, offsets, ctx.scale, ctx.softcap, ctx.offset, ctx.monotone = inputs
    out, lse, *rows = output
    ctx.save_for_backward(q, k, v, out, rows[0] if rows else lse, lo, hi, mask, slopes, offsets)
    ctx.has_rows = bool(rows)
    ctx.mark_non_differentiable(lse, *rows)


def _backward(ctx, dout, *_):
    q, k, v, out, stat, lo, hi, mask, slopes, offsets = ctx.saved_tensors
    grads = flash_bwd_scored(dout, q, k, v, out, stat, lo, hi, mask, slopes, offsets, ctx.scale, ctx.softcap,
                             ctx.offset, ctx.monotone, stat if ctx.has_rows else None)
    return (*grads,) + (None,) * 9


torch.library.register_autograd("avgen_amd::flash_fwd_scored", _backward, setup_context=_setup)
torch.library.register_autograd("avgen_amd::flash_fwd_scored_rows", _backward, setup_context=_setup)


class _FlashFwdScored(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        out, lse, row_lse = _fwd_impl(*args, True)
        ctx.set_materialize_grads(False)
        q, k, v, lo, hi, mask, slopes, offsets, ctx.scale, ctx.softcap, ctx.offset, ctx.monotone = args
        ctx.save_for_backward(q, k, v, out, row_lse, lo, hi, mask, slopes, offsets)
        ctx.has_rows = True
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, dout, _dlse):
        if dout is None:
            return (None,) * 12
        if not _grad_direct(dout):
            return _backward(ctx, dout)
        # The forward was a plain call: so is this one.
        q, k, v, out, stat, lo, hi, mask, slopes, offsets = ctx.saved_tensors
        grads = _bwd_impl(dout, q, k, v, out, stat, lo, hi, mask, slopes, offsets, ctx.scale, ctx.softcap, ctx.offset,
                          ctx.monotone, stat, True)
        return (*grads,) + (None,) * 9
