"""Ops of the gated residual step between two sections of a block: the norm
behind a section, its gate, the residual addition and the modulated norm in
front of the next section.

Registered like those of :mod:`avgen_amd.block_ops` (same checks, streams,
workspaces and errors).  Ops (namespace ``avgen_amd``):

* ``gated_add_rms_norm(x, residual, weight, post_weight, gate, scale, shift,
  residual_scale, eps) -> (norm, sum)``, differentiable in the tensors;
* ``gated_add_rms_norm_bwd``.

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
from .ops import _direct, _grad_direct, _ptr, _stream, _workspace

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
    first = None
    for label, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is None:
            continue
        if t.ndim < 1 or t.shape[-1] != W:
            raise ValueError(f"{name}: {label} must have rows of {W}; got {tuple(t.shape)}")
        if first is None:
            first = t
            if t.dtype is not dtype and t.dtype is not torch.float32:
                raise TypeError(f"{name}: {label} must be {dtype} or float32; got {t.dtype}")
            if rows and (t.numel() == 0 or rows % (t.numel() // W)):
                raise ValueError(f"{name}: {label} {tuple(t.shape)} does not divide {tuple(shape)} into groups of rows")
        elif t.shape != first.shape:
            raise ValueError(f"{name}: gate, scale and shift must have one shape; got {tuple(first.shape)} and "
                             f"{tuple(t.shape)}")
        elif t.dtype is not first.dtype:
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
    t, stride = _rows(t)
    return t, t.data_ptr(), stride


def _vectors(weight, post_weight, gate, scale, shift):
    """The C arguments of the vectors, and the tensors to hold until the launch."""
    held = [_row_of(t) for t in (weight, post_weight, gate, scale, shift)]
    f32 = [t is not None and t.dtype is torch.float32 for t in (weight, post_weight)]
    (_, w, _), (_, p, _), (_, g, gs), (_, s, ss), (_, t, ts) = held
    m32 = any(x is not None and x.dtype is torch.float32 for x in (gate, scale, shift))
    return (w, f32[0], p, f32[1], g, gs, s, ss, t, ts, m32), held


def _impl(x, residual, weight, post_weight, gate, scale, shift, residual_scale, eps):
    rows, group = _check_vectors(_NAME, x, weight, post_weight, gate, scale, shift, eps, residual_scale)
    shape, dtype, device = x.shape, x.dtype, x.device
    if residual is not x:
        if residual.shape != shape:
            raise ValueError(f"{_NAME}: residual {tuple(residual.shape)} must have the input's shape {tuple(shape)}")
        if residual.dtype is not dtype:
            raise TypeError(f"{_NAME}: residual must be {dtype} like the input; got {residual.dtype}")
    _one_device(_NAME, x, residual, weight, post_weight, gate, scale, shift)
    total = torch.empty_like(x, memory_format=torch.contiguous_format)
    norm = torch.empty_like(total)
    if rows:
        vectors, _held = _vectors(weight, post_weight, gate, scale, shift)
        (x, xs), (residual, rs) = _rows(x), _rows(residual)
        with _on(device):
            st = _lib.load().avattn_gated_add_rms_norm(
                x.data_ptr(), xs, residual.data_ptr(), rs, *vectors, rows, shape[-1], group,
                dtype is torch.float32, residual_scale, eps, total.data_ptr(), norm.data_ptr(), _stream(device))
        _lib.check(st, _NAME)
    return norm, total


@lru_cache(maxsize=256)
def _bwd_workspace_size(rows: int, width: int, group: int, modulated: bool) -> int:
    return _lib.load().avattn_gated_add_rms_norm_bwd_workspace_size(rows, width, group, modulated)


def _alike(post_weight, gate, residual_scale) -> bool:
    """Whether x and the residual have one gradient."""
    return gate is None and post_weight is None and residual_scale == 1.0


def _bwd_impl(dnorm, dsum, x, total, weight, post_weight, gate, scale, shift, residual_scale, eps):
    """``(dx, dresidual, dweight, dpost_weight, dgate, dscale, dshift)``; None for
    what is not there, and dresidual is dx where the two are alike."""
    name = _NAME + "_bwd"
    rows, group = _check_vectors(name, total, weight, post_weight, gate, scale, shift, eps, residual_scale)
    needs_x = gate is not None or post_weight is not None
    for label, t in (("norm gradient", dnorm), ("sum gradient", dsum), ("input", x)):
        if t is None and (label == "sum gradient" or (label == "input" and not needs_x)):
            continue
        if t is None or t.shape != total.shape or t.dtype is not total.dtype:
            raise ValueError(f"{name}: {label} must be {total.dtype} {tuple(total.shape)}")
    _one_device(name, total, dnorm, dsum, x, weight, post_weight, gate, scale, shift)
    W, device = total.shape[-1], total.device
    dx = torch.empty_like(total, memory_format=torch.contiguous_format)
    dr = dx if _alike(post_weight, gate, residual_scale) else torch.empty_like(dx)
    new = torch.empty if rows else torch.zeros
    grads = [None if t is None else new(t.shape, dtype=t.dtype, device=device)
             for t in (weight, post_weight, gate, scale, shift)]
    if rows:
        vectors, _held = _vectors(weight, post_weight, gate, scale, shift)
        (dnorm, dns), (total, hs) = _rows(dnorm), _rows(total)
        dhs = xs = 0
        if dsum is not None:
            dsum, dhs = _rows(dsum)
        if needs_x:
            x, xs = _rows(x)
        modulated = gate is not None or scale is not None or shift is not None
        ws = _workspace(_bwd_workspace_size(rows, W, group, modulated), device)
        with _on(device):
            st = _lib.load().avattn_gated_add_rms_norm_bwd(
                dnorm.data_ptr(), dns, _ptr(dsum), dhs, x.data_ptr() if needs_x else None, xs, total.data_ptr(), hs,
                *vectors, rows, W, group, total.dtype is torch.float32, residual_scale, eps, dx.data_ptr(),
                None if dr is dx else dr.data_ptr(), *(_ptr(t) for t in grads), ws.data_ptr(), ws.numel(),
                _stream(device))
        _lib.check(st, name)
    return (dx, dr, *grads)


@torch.library.custom_op("avgen_amd::gated_add_rms_norm", mutates_args=())
def _op(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
        gate: Optional[torch.Tensor], scale: Optional[torch.Tensor], shift: Optional[torch.Tensor],
        residual_scale: float, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, sum)``; see the module docstring."""
    return _impl(x, residual, weight, post_weight, gate, scale, shift, residual_scale, eps)


@_op.register_fake
def _(x, residual, weight, post_weight, gate, scale, shift, residual_scale, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape)


@torch.library.custom_op("avgen_amd::gated_add_rms_norm_bwd", mutates_args=())
def _bwd_op(dnorm: torch.Tensor, dsum: Optional[torch.Tensor], x: Optional[torch.Tensor], total: torch.Tensor,
            weight: Optional[torch.Tensor], post_weight: Optional[torch.Tensor], gate: Optional[torch.Tensor],
            scale: Optional[torch.Tensor], shift: Optional[torch.Tensor], residual_scale: float, eps: float
            ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                       torch.Tensor]:
    """The gradients of all inputs, without elements for what is not there and
    for a residual's that is x's."""
    dx, dr, *grads = _bwd_impl(dnorm, dsum, x, total, weight, post_weight, gate, scale, shift, residual_scale, eps)
    none = [total.new_empty(0) for _ in range(6)]
    return (dx, none[0] if dr is dx else dr, *(none[i + 1] if g is None else g for i, g in enumerate(grads)))


@_bwd_op.register_fake
def _(dnorm, dsum, x, total, weight, post_weight, gate, scale, shift, residual_scale, eps):
    dr = total.new_empty(0 if _alike(post_weight, gate, residual_scale) else total.shape)
    return (total.new_empty(total.shape), dr,
            *(total.new_empty(0) if t is None else t.new_empty(t.shape)
              for t in (weight, post_weight, gate, scale, shift)))


def gated_add_rms_norm(x, residual, weight, post_weight, gate, scale, shift, residual_scale: float,
                       eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, sum)`` of the gated residual step; differentiable."""
    tensors = (x, residual, weight, post_weight, gate, scale, shift)
    return _direct(_GatedAddRmsNorm, _op, _impl, (*tensors, residual_scale, eps), tensors)


def gated_add_rms_norm_bwd(dnorm, dsum, x, total, weight, post_weight, gate, scale, shift, residual_scale: float,
                           eps: float):
    """The gradients of ``gated_add_rms_norm`` from its stored sum (``x`` None
    without gate and post_weight): ``(dx, dresidual, dweight, dpost_weight, dgate,
    dscale, dshift)``, None for what is not there."""
    args = (dnorm, dsum, x, total, weight, post_weight, gate, scale, shift, residual_scale, eps)
    if _grad_direct(dnorm, dsum, x, total, weight, post_weight, gate, scale, shift):
        return _bwd_impl(*args)
    dx, dr, *grads = _bwd_op(*args)
    if _alike(post_weight, gate, residual_scale):
        dr = dx
    return (dx, dr, *(None if t is None else g for t, g in zip((weight, post_weight, gate, scale, shift), grads)))


def _setup(ctx, inputs, output):
    x, _residual, weight, post_weight, gate, scale, shift, ctx.residual_scale, ctx.eps = inputs
    ctx.save_for_backward(None if gate is None and post_weight is None else x, output[1], weight, post_weight, gate,
                          scale, shift)


def _backward(ctx, dnorm, dsum):
    x, total, weight, post_weight, gate, scale, shift = ctx.saved_tensors
    if dnorm is None:
        if dsum is None:
            return (None,) * 9
        dnorm = torch.zeros_like(total)  # the sum alone was used
    grads = gated_add_rms_norm_bwd(dnorm, dsum, x, total, weight, post_weight, gate, scale, shift, ctx.residual_scale,
                                   ctx.eps)
    return (*grads, None, None)


torch.library.register_autograd("avgen_amd::gated_add_rms_norm", _backward, setup_context=_setup)


class _GatedAddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        result = _impl(*args)
        ctx.set_materialize_grads(False)
        _setup(ctx, args, result)
        return result

    @staticmethod
    def backward(ctx, dnorm, dsum):
        return _backward(ctx, dnorm, dsum)
