"""Ops of the gated residual step between two sections of a block: the norm
behind a section, its gate, the residual addition and the modulated norm in
front of the next section.

Registered like those of :mod:`avgen_amd.block_ops` (same checks, streams,
workspaces and errors).  Ops (namespace ``avgen_amd``):

* ``gated_add_rms_norm(x, residual, weight, post_weight, gate, scale, shift,
  residual_scale, eps) -> (norm, sum, stats)``, differentiable in the tensors;
* ``gated_add_rms_norm_bwd``, which takes the stats, two float32 factors a row.

``gate``, ``scale`` and ``shift`` have a row of ``width`` for each of the groups
of consecutive rows that their leading sizes divide ``x`` into, all of them
alike.  Tensors are bf16 or float32, on one device, of any width, stride and
alignment; each vector may be float32 beside bf16 rows.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .block_ops import _FLOATS, _on, _one_device, _rows
from .ops import _grad_direct, _ptr, _stream, _workspace

__all__ = ["gated_add_rms_norm", "gated_add_rms_norm_bwd"]

_NAME = "avgen_amd.gated_add_rms_norm"


def _check_vectors(name, x, weight, post_weight, gate, scale, shift, eps, factor):
    """Types and shapes: the rows, and those of a group."""
    shape, dtype = x.shape, x.dtype
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"{name}: rows of at least one value expected; got {tuple(shape)}")
    if dtype not in _FLOATS:
        raise TypeError(f"{name}: input must be bfloat16 or float32; got {dtype}")
    W = shape[-1]
    for label, t in (("weight", weight), ("post_weight", post_weight)):
        if t is None:
            continue
        if t.shape != (W,):
            raise ValueError(f"{name}: {label} must be ({W},); got {tuple(t.shape)}")
        if t.dtype is not dtype and t.dtype is not torch.float32:
            raise TypeError(f"{name}: {label} must be {dtype} or float32; got {t.dtype}")
    rows = x.numel() // W
    first = gate if gate is not None else scale if scale is not None else shift
    if first is not None:
        if first.ndim < 1 or first.shape[-1] != W:
            raise ValueError(f"{name}: gate, scale and shift must have rows of {W}; got {tuple(first.shape)}")
        if first.dtype is not dtype and first.dtype is not torch.float32:
            raise TypeError(f"{name}: gate, scale and shift must be {dtype} or float32; got {first.dtype}")
        if rows and (first.numel() == 0 or rows % (first.numel() // W)):
            raise ValueError(f"{name}: {tuple(first.shape)} does not divide {tuple(shape)} into groups of rows")
        for t in (scale, shift):
            if t is None or t is first:
                continue
            if t.shape != first.shape:
                raise ValueError(f"{name}: gate, scale and shift must have one shape; got {tuple(first.shape)} and "
                                 f"{tuple(t.shape)}")
            if t.dtype is not first.dtype:
                raise TypeError(f"{name}: gate, scale and shift must have one type; got {first.dtype} and {t.dtype}")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"{name}: eps must be finite and >= 0; got {eps}")
    if not math.isfinite(factor):
        raise ValueError(f"{name}: residual_scale must be finite; got {factor}")
    return rows, rows if first is None or not rows else rows * W // first.numel()


def _row_of(t: Optional[torch.Tensor]):
    """A vector's or modulation's tensor to read (held by the caller until the
    launch), pointer and row stride."""
    if t is None:
        return None, None, 0
    stride = t.stride()
    if stride[-1] == 1 and t.numel() == t.shape[0] * t.shape[-1]:  # rows along the first dimension
        return t, t.data_ptr(), stride[0]
    t, stride = _rows(t)
    return t, t.data_ptr(), stride


def _vectors(weight, post_weight, gate, scale, shift):
    """The C arguments of the vectors, and the tensors to hold until the launch."""
    w, wp, _ = _row_of(weight)
    p, pp, _ = _row_of(post_weight)
    g, gp, gs = _row_of(gate)
    s, sp, ss = _row_of(scale)
    t, tp, ts = _row_of(shift)
    f32 = torch.float32
    first = g if g is not None else s if s is not None else t
    return (wp, w is not None and w.dtype is f32, pp, p is not None and p.dtype is f32, gp, gs, sp, ss, tp, ts,
            first is not None and first.dtype is f32), (w, p, g, s, t)


def _impl(x, residual, weight, post_weight, gate, scale, shift, residual_scale, eps):
    rows, group = _check_vectors(_NAME, x, weight, post_weight, gate, scale, shift, eps, residual_scale)
    shape, dtype, device = x.shape, x.dtype, x.device
    if residual is not x:
        if residual.shape != shape:
            raise ValueError(f"{_NAME}: residual {tuple(residual.shape)} must have the input's shape {tuple(shape)}")
        if residual.dtype is not dtype:
            raise TypeError(f"{_NAME}: residual must be {dtype} like the input; got {residual.dtype}")
    _one_device(_NAME, x, residual, weight, post_weight, gate, scale, shift)
    total = torch.empty(shape, dtype=dtype, device=device)
    norm = torch.empty(shape, dtype=dtype, device=device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=device)
    if rows:
        vectors, _held = _vectors(weight, post_weight, gate, scale, shift)
        (x, xs), (residual, rs) = _rows(x), _rows(residual)
        with _on(device):
            st = _lib.load().avattn_gated_add_rms_norm(
                x.data_ptr(), xs, residual.data_ptr(), rs, *vectors, rows, shape[-1], group,
                dtype is torch.float32, residual_scale, eps, total.data_ptr(), norm.data_ptr(), stats.data_ptr(),
                _stream(device))
        _lib.check(st, _NAME)
    return norm, total, stats


@lru_cache(maxsize=256)
def _bwd_workspace_size(rows: int, width: int, group: int, modulated: bool) -> int:
    return _lib.load().avattn_gated_add_rms_norm_bwd_workspace_size(rows, width, group, modulated)


def _alike(post_weight, gate, residual_scale) -> bool:
    """Whether x and the residual have one gradient."""
    return gate is None and post_weight is None and residual_scale == 1.0


def _bwd_impl(dnorm, dsum, x, residual, stats, weight, post_weight, gate, scale, shift, residual_scale, eps):
    """``(dx, dresidual, dweight, dpost_weight, dgate, dscale, dshift)``; None for
    what is not there, and dresidual is dx where the two are alike."""
    name = _NAME + "_bwd"
    rows, group = _check_vectors(name, x, weight, post_weight, gate, scale, shift, eps, residual_scale)
    shape, dtype, device = x.shape, x.dtype, x.device
    for label, t in (("norm gradient", dnorm), ("sum gradient", dsum), ("residual", residual)):
        if t is not None and (t.shape != shape or t.dtype is not dtype):
            raise ValueError(f"{name}: {label} must be {dtype} {tuple(shape)}")
    if stats.shape != (rows, 2) or stats.dtype is not torch.float32:
        raise ValueError(f"{name}: stats must be float32 ({rows}, 2)")
    _one_device(name, x, residual, stats, dnorm, dsum, weight, post_weight, gate, scale, shift)
    stats = stats.contiguous()
    W = shape[-1]
    dx = torch.empty(shape, dtype=dtype, device=device)
    dr = dx if _alike(post_weight, gate, residual_scale) else torch.empty(shape, dtype=dtype, device=device)
    new = torch.empty if rows else torch.zeros
    grads = [None if t is None else new(t.shape, dtype=t.dtype, device=device)
             for t in (weight, post_weight, gate, scale, shift)]
    if rows:
        vectors, _held = _vectors(weight, post_weight, gate, scale, shift)
        (dnorm, dns), (x, xs), (residual, rs) = _rows(dnorm), _rows(x), _rows(residual)
        dhs = 0
        if dsum is not None:
            dsum, dhs = _rows(dsum)
        modulated = gate is not None or scale is not None or shift is not None
        ws = _workspace(_bwd_workspace_size(rows, W, group, modulated), device)
        with _on(device):
            st = _lib.load().avattn_gated_add_rms_norm_bwd(
                dnorm.data_ptr(), dns, _ptr(dsum), dhs, x.data_ptr(), xs, residual.data_ptr(), rs, stats.data_ptr(),
                *vectors, rows, W, group, dtype is torch.float32, residual_scale, eps, dx.data_ptr(),
                None if dr is dx else dr.data_ptr(), *(_ptr(t) for t in grads), ws.data_ptr(), ws.numel(),
                _stream(device))
        _lib.check(st, name)
    return (dx, dr, *grads)


@torch.library.custom_op("avgen_amd::gated_add_rms_norm", mutates_args=())
def _op(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
        gate: Optional[torch.Tensor], scale: Optional[torch.Tensor], shift: Optional[torch.Tensor],
        residual_scale: float, eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(norm, sum, stats)``; see the module docstring."""
    return _impl(x, residual, weight, post_weight, gate, scale, shift, residual_scale, eps)


@_op.register_fake
def _(x, residual, weight, post_weight, gate, scale, shift, residual_scale, eps):
    rows = x.numel() // x.shape[-1]
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty((rows, 2), dtype=torch.float32)


@torch.library.custom_op("avgen_amd::gated_add_rms_norm_bwd", mutates_args=())
def _bwd_op(dnorm: torch.Tensor, dsum: Optional[torch.Tensor], x: torch.Tensor, residual: torch.Tensor,
            stats: torch.Tensor, weight: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
            gate: Optional[torch.Tensor], scale: Optional[torch.Tensor], shift: Optional[torch.Tensor],
            residual_scale: float, eps: float
            ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                       torch.Tensor]:
    """The gradients of all inputs, without elements for what is not there and
    for a residual's that is x's."""
    dx, dr, *grads = _bwd_impl(dnorm, dsum, x, residual, stats, weight, post_weight, gate, scale, shift,
                               residual_scale, eps)
    none = [x.new_empty(0) for _ in range(6)]
    return (dx, none[0] if dr is dx else dr, *(none[i + 1] if g is None else g for i, g in enumerate(grads)))


@_bwd_op.register_fake
def _(dnorm, dsum, x, residual, stats, weight, post_weight, gate, scale, shift, residual_scale, eps):
    dr = x.new_empty(0 if _alike(post_weight, gate, residual_scale) else x.shape)
    return (x.new_empty(x.shape), dr,
            *(x.new_empty(0) if t is None else t.new_empty(t.shape)
              for t in (weight, post_weight, gate, scale, shift)))


def gated_add_rms_norm(x, residual, weight, post_weight, gate, scale, shift, residual_scale: float,
                       eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, sum)`` of the gated residual step; differentiable."""
    args = (x, residual, weight, post_weight, gate, scale, shift, residual_scale, eps)
    calls = _lib.direct_calls(x)
    if calls is not None:
        out = calls.gated_add_rms_norm(*args)
        if out is not NotImplemented:
            return out
    return _op(*args)[:2]


def gated_add_rms_norm_bwd(dnorm, dsum, x, residual, stats, weight, post_weight, gate, scale, shift,
                           residual_scale: float, eps: float):
    """The gradients of ``gated_add_rms_norm`` from its inputs and stats: ``(dx,
    dresidual, dweight, dpost_weight, dgate, dscale, dshift)``, None for what is
    not there."""
    args = (dnorm, dsum, x, residual, stats, weight, post_weight, gate, scale, shift, residual_scale, eps)
    if _grad_direct(dnorm, dsum, x, residual, stats, weight, post_weight, gate, scale, shift):
        return _bwd_impl(*args)
    dx, dr, *grads = _bwd_op(*args)
    if _alike(post_weight, gate, residual_scale):
        dr = dx
    return (dx, dr, *(None if t is None else g for t, g in zip((weight, post_weight, gate, scale, shift), grads)))


def _setup(ctx, inputs, output):
    *tensors, ctx.residual_scale, ctx.eps = inputs
    stats = output[2]
    ctx.save_for_backward(tensors[0], tensors[1], stats, *tensors[2:])
    ctx.mark_non_differentiable(stats)


def _backward(ctx, dnorm, dsum, _dstats=None):
    saved = ctx.saved_tensors
    if dnorm is None:
        if dsum is None:
            return (None,) * 9
        dnorm = torch.zeros_like(saved[0])  # the sum alone was used
    grads = gated_add_rms_norm_bwd(dnorm, dsum, *saved, ctx.residual_scale, ctx.eps)
    return (*grads, None, None)


torch.library.register_autograd("avgen_amd::gated_add_rms_norm", _backward, setup_context=_setup)
