"""Ops of the steps around attention in a block: the rotation of part of each
head by sequence positions, and the residual addition with its RMS norm.

Registered as ``torch.library`` ops like those of :mod:`avgen_amd.ops`
(same checks, streams, workspaces and errors; plain eager calls skip the
dispatcher's Python layers).  Ops (namespace ``avgen_amd``):

* ``rotate(x, cos, sin, start, half, inverse)`` and ``rotate_pair(q, k, ...)``
  (one launch for both), differentiable in the tensors;
* ``add_rms_norm(x, residual, weight, eps) -> (norm, sum)``, differentiable,
  with ``add_rms_norm_bwd``;
* ``add_rms_norm_fp8(x, residual, weight, eps) -> (codes, scale, sum)``.

Tensors are bf16 or float32, on one device; unlike the attention ops these
take any width, stride and alignment.
"""

from __future__ import annotations

import ctypes
import math
from contextlib import nullcontext
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .ops import _direct, _grad_direct, _ptr, _require_gpu, _stream, _Strides3, _workspace

__all__ = [
    "MAX_TABLE_PAIRS",
    "add_rms_norm",
    "add_rms_norm_bwd",
    "add_rms_norm_fp8",
    "position_tables",
    "rotate",
    "rotate_pair",
]

#: Most pairs of one position table (``avattn_position_tables``).
MAX_TABLE_PAIRS = 256

_FLOATS = (torch.bfloat16, torch.float32)


def _one_device(name: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    """All tensors on one GPU: the GPU."""
    device = first.device
    if device.type != "cuda":
        _require_gpu(name, first)
    for t in others:
        if t is not None and t.device != device:
            _require_gpu(name, t)
            raise RuntimeError(f"{name}: tensors on different devices: {device} and {t.device}")
    return device


_here = nullcontext()


def _on(device: torch.device):
    """Launches on ``device``, whichever is current."""
    index = device.index
    if index is None or index == torch._C._cuda_getDevice():
        return _here
    return torch.cuda.device(device)


def _packed_last(t: torch.Tensor) -> torch.Tensor:
    """``t`` with a contiguous last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


# ---------------------------------------------------------------------------
# Rotation
# ---------------------------------------------------------------------------


def position_tables(positions: torch.Tensor, frequencies: list[float], amplitude: float):
    """cos/sin tables ``(B, 1, L, pairs)`` float32 of integer ``positions``
    ``(B, L)``: ``amplitude * cos(position * frequency)``, the angle in
    double."""
    name = "avgen_amd.position_tables"
    if positions.ndim != 2:
        raise ValueError(f"{name}: positions must be (batch, length); got {tuple(positions.shape)}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: positions must be int32 or int64; got {positions.dtype}")
    P = len(frequencies)
    if not 1 <= P <= MAX_TABLE_PAIRS:
        raise ValueError(f"{name}: 1 to {MAX_TABLE_PAIRS} pairs; got {P}")
    _require_gpu(name, positions)
    positions = _packed_last(positions)
    B, L = positions.shape
    stride = positions.stride(0) if B > 1 else 0
    if 0 < stride < L or stride < 0:
        positions = positions.contiguous()
        stride = L
    cos = torch.empty((B, 1, L, P), device=positions.device, dtype=torch.float32)
    sin = torch.empty_like(cos)
    freq = (ctypes.c_double * P)(*frequencies)
    with _on(positions.device):
        st = _lib.load().avattn_position_tables(
            _ptr(positions), int(positions.dtype is torch.int64), stride, B, L, P,
            ctypes.cast(freq, ctypes.c_void_p), float(amplitude), _ptr(cos), _ptr(sin), _stream(positions.device))
    _lib.check(st, name)
    return cos, sin


def _check_rotation(name, tensors, cos, sin, start):
    """Shapes and dtypes; the tables contiguous, with their batch stride."""
    x = tensors[0]
    dtype, shape = x.dtype, x.shape
    if len(shape) != 4:
        raise ValueError(f"{name}: rotary input must be (batch, heads, length, head_dim); got {tuple(shape)}")
    B, _, L, D = shape
    for t in tensors:
        if t.dtype not in _FLOATS or t.dtype is not dtype:
            raise TypeError(f"{name}: inputs must all be bfloat16 or all float32; got {t.dtype}")
        if t is not x:
            s = t.shape
            if len(s) != 4 or s[0] != B or s[2] != L or s[3] != D:
                raise ValueError(f"{name}: {tuple(shape)} and {tuple(s)} differ in more than their heads")
    table = cos.shape
    if len(table) != 4 or table != sin.shape:
        raise ValueError(f"{name}: rotary tables must be (batch, 1, length, pairs) and agree")
    if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise TypeError(f"{name}: rotary tables must be float32")
    TB, TH, TL, P = table
    if P < 1 or start < 0 or start + 2 * P > D:
        raise ValueError(f"{name}: channels [{start}, {start + 2 * P}) do not lie in a head of {D}")
    if TL != L:
        raise ValueError(f"{name}: sequence length {L} does not match rotary tables built for length {TL}")
    if TB not in (1, B) or TH != 1:
        raise ValueError(f"{name}: rotary tables batch {TB} does not broadcast to {B}")
    _one_device(name, *tensors, cos, sin)
    return cos.contiguous(), sin.contiguous(), (0 if TB == 1 else L * P)


def _rotate_launch(name, q, k, cos, sin, start, half, inverse):
    cos, sin, tsb = _check_rotation(name, (q,) if k is None else (q, k), cos, sin, start)
    return _rotate_run(name, q, k, cos, sin, tsb, start, half, inverse)


def _rotate_run(name, q, k, cos, sin, tsb, start, half, inverse):
    """The rotation of checked arguments."""
    B, _, L, D = q.shape
    outs = []
    written = []
    args = []
    read = []  # held until the launch: copies among them belong to nobody else
    for t in (q, k):
        if t is None:
            args += (None, None, 0, None, None)
            continue
        # The layout that the op promises; written elsewhere and copied where
        # its channels are not next to each other.
        o = w = torch.empty_like(t)
        outs.append(o)
        t = _packed_last(t)
        read.append(t)
        strides, wstrides = t.stride(), o.stride()
        if wstrides[3] != 1 and D > 1:
            w = torch.empty(t.shape, dtype=t.dtype, device=t.device)
            wstrides = w.stride()
        written.append(w)
        s = _Strides3(*strides[:3])
        args += (t.data_ptr(), s, t.shape[1], w.data_ptr(), s if wstrides == strides else _Strides3(*wstrides[:3]))
    device = q.device
    with _on(device):
        st = _lib.load().avattn_rotate(
            *args, B, L, D, cos.shape[-1], start, half, q.dtype is torch.float32,
            cos.data_ptr(), sin.data_ptr(), tsb, inverse, _stream(device))
    _lib.check(st, name)
    for o, w in zip(outs, written):
        if w is not o:
            o.copy_(w)
    return outs


def _rotate_impl(x, cos, sin, start, half, inverse):
    return _rotate_launch("avgen_amd.rotate", x, None, cos, sin, start, half, inverse)[0]


def _rotate_pair_impl(q, k, cos, sin, start, half, inverse):
    return tuple(_rotate_launch("avgen_amd.rotate_pair", q, k, cos, sin, start, half, inverse))


@torch.library.custom_op("avgen_amd::rotate", mutates_args=())
def _rotate_op(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, start: int, half: bool,
               inverse: bool) -> torch.Tensor:
    """Rotation (or its transpose) of channels [start, start + 2 pairs)."""
    return _rotate_impl(x, cos, sin, start, half, inverse)


@_rotate_op.register_fake
def _(x, cos, sin, start, half, inverse):
    return torch.empty_like(x)


@torch.library.custom_op("avgen_amd::rotate_pair", mutates_args=())
def _rotate_pair_op(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, start: int, half: bool,
                    inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """``rotate`` of a query and a key by the same tables, in one launch."""
    return _rotate_pair_impl(q, k, cos, sin, start, half, inverse)


@_rotate_pair_op.register_fake
def _(q, k, cos, sin, start, half, inverse):
    return torch.empty_like(q), torch.empty_like(k)


def rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, start: int, half: bool,
           inverse: bool) -> torch.Tensor:
    """Rotation (or its transpose) of channels [start, start + 2 pairs)."""
    return _direct(_Rotate, _rotate_op, _rotate_impl, (x, cos, sin, start, half, inverse), (x, cos, sin))


def rotate_pair(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, start: int, half: bool,
                inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """``rotate`` of a query and a key by the same tables, in one launch."""
    return _direct(_RotatePair, _rotate_pair_op, _rotate_pair_impl, (q, k, cos, sin, start, half, inverse),
                   (q, k, cos, sin))


def _rotate_setup(ctx, inputs, output):
    _x, cos, sin, ctx.start, ctx.half, ctx.inverse = inputs
    ctx.save_for_backward(cos, sin)


def _rotate_backward(ctx, grad):
    cos, sin = ctx.saved_tensors
    return rotate(grad, cos, sin, ctx.start, ctx.half, not ctx.inverse), None, None, None, None, None


def _rotate_pair_setup(ctx, inputs, output):
    _q, _k, cos, sin, ctx.start, ctx.half, ctx.inverse = inputs
    ctx.save_for_backward(cos, sin)


def _rotate_pair_backward(ctx, gq, gk):
    cos, sin = ctx.saved_tensors
    how = (cos, sin, ctx.start, ctx.half, not ctx.inverse)
    if gq is not None and gk is not None:
        gq, gk = rotate_pair(gq, gk, *how)
    else:
        gq, gk = (None if g is None else rotate(g, *how) for g in (gq, gk))
    return gq, gk, None, None, None, None, None


torch.library.register_autograd("avgen_amd::rotate", _rotate_backward, setup_context=_rotate_setup)
torch.library.register_autograd("avgen_amd::rotate_pair", _rotate_pair_backward, setup_context=_rotate_pair_setup)


# Plain eager calls.  Their backward, a plain call itself, takes the arguments
# that the forward has checked: small calls are bound by this Python, which runs
# at half speed on autograd's own thread.
class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        result = _rotate_impl(*args)
        ctx.set_materialize_grads(False)
        _rotate_setup(ctx, args, result)
        return result

    @staticmethod
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 6
        if not _grad_direct(grad):
            return _rotate_backward(ctx, grad)
        return _rotate_grads(ctx, "avgen_amd.rotate", grad)[0], None, None, None, None, None


class _RotatePair(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        result = _rotate_pair_impl(*args)
        ctx.set_materialize_grads(False)
        _rotate_pair_setup(ctx, args, result)
        return result

    @staticmethod
    def backward(ctx, gq, gk):
        if gq is None or gk is None or not _grad_direct(gq, gk):
            return _rotate_pair_backward(ctx, gq, gk)
        return (*_rotate_grads(ctx, "avgen_amd.rotate_pair", gq, gk), None, None, None, None, None)


def _rotate_grads(ctx, name, gq, gk=None):
    cos, sin = ctx.saved_tensors
    cos, sin = cos.contiguous(), sin.contiguous()
    tsb = 0 if cos.shape[0] == 1 else cos.shape[2] * cos.shape[3]
    return _rotate_run(name, gq, gk, cos, sin, tsb, ctx.start, ctx.half, not ctx.inverse)


# ---------------------------------------------------------------------------
# Residual + RMS norm
# ---------------------------------------------------------------------------


def _rows(t: torch.Tensor):
    """``t (..., W)`` as rows of ``W`` contiguous values: the tensor to read
    and its row stride."""
    W = t.shape[-1]
    if t.is_contiguous():
        return t, W
    t = _packed_last(t)
    if t.ndim == 1 or t.numel() <= W:
        return t, W
    # The leading dimensions must collapse into one stride.
    stride = expect = None
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if stride is None:
            stride = s
        elif s != expect:
            return t.contiguous(), W
        expect = s * n
    if stride < 0:
        return t.contiguous(), W
    return t, stride


def _check_norm(name, x, residual, weight, eps):
    shape, dtype = x.shape, x.dtype
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"{name}: rows of at least one value expected; got {tuple(shape)}")
    if dtype not in _FLOATS:
        raise TypeError(f"{name}: input must be bfloat16 or float32; got {dtype}")
    if residual is not x:
        if residual.shape != shape:
            raise ValueError(f"{name}: residual {tuple(residual.shape)} must have the input's shape {tuple(shape)}")
        if residual.dtype is not dtype:
            raise TypeError(f"{name}: residual must be {dtype} like the input; got {residual.dtype}")
    if weight.shape != shape[-1:]:
        raise ValueError(f"{name}: weight must be ({shape[-1]},); got {tuple(weight.shape)}")
    if weight.dtype is not dtype and weight.dtype is not torch.float32:
        raise TypeError(f"{name}: weight must be {dtype} or float32; got {weight.dtype}")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"{name}: eps must be finite and >= 0; got {eps}")
    _one_device(name, x, residual, weight)
    return weight.contiguous()


def _norm_launch(name, x, residual, weight, eps, fp8):
    w = _check_norm(name, x, residual, weight, eps)
    shape, dtype, device = x.shape, x.dtype, x.device
    W = shape[-1]
    rows = x.numel() // W
    total = torch.empty_like(x, memory_format=torch.contiguous_format)
    norm = torch.empty_like(x, memory_format=torch.contiguous_format, dtype=torch.float8_e4m3fn if fp8 else dtype)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=device) if fp8 else None
    (x, xs), (residual, rs) = _rows(x), _rows(residual)
    if rows:
        with _on(device):
            st = _lib.load().avattn_add_rms_norm(
                x.data_ptr(), xs, residual.data_ptr(), rs, w.data_ptr(), w.dtype is torch.float32, rows, W,
                dtype is torch.float32, eps, total.data_ptr(), norm.data_ptr(), _ptr(scale), _stream(device))
        _lib.check(st, name)
    return norm, scale, total


def _add_rms_norm_impl(x, residual, weight, eps):
    norm, _, total = _norm_launch("avgen_amd.add_rms_norm", x, residual, weight, eps, False)
    return norm, total


def _add_rms_norm_fp8_impl(x, residual, weight, eps):
    return _norm_launch("avgen_amd.add_rms_norm_fp8", x, residual, weight, eps, True)


@lru_cache(maxsize=256)
def _norm_workspace_size(rows: int, width: int) -> int:
    return _lib.load().avattn_add_rms_norm_bwd_workspace_size(rows, width)


def _add_rms_norm_bwd_impl(dnorm, dsum, total, weight, eps):
    name = "avgen_amd.add_rms_norm_bwd"
    w = _check_norm(name, total, total, weight, eps)
    for label, t in (("norm gradient", dnorm), ("sum gradient", dsum)):
        if t is not None and (t.shape != total.shape or t.dtype is not total.dtype):
            raise ValueError(f"{name}: {label} must be {total.dtype} {tuple(total.shape)}")
    _one_device(name, dnorm, dsum, total)
    return _add_rms_norm_bwd_run(name, dnorm, dsum, total, w, eps)


def _add_rms_norm_bwd_run(name, dnorm, dsum, total, w, eps):
    """The backward of checked arguments."""
    W = total.shape[-1]
    rows = total.numel() // W
    dx = torch.empty(total.shape, dtype=total.dtype, device=total.device)
    dw = torch.empty((W,), dtype=w.dtype, device=w.device)
    (dnorm, dns), (total, hs) = _rows(dnorm), _rows(total)
    dhs = 0
    if dsum is not None:
        dsum, dhs = _rows(dsum)
    device = total.device
    ws = _workspace(_norm_workspace_size(rows, W), device)
    with _on(device):
        st = _lib.load().avattn_add_rms_norm_bwd(
            dnorm.data_ptr(), dns, _ptr(dsum), dhs, total.data_ptr(), hs, w.data_ptr(), w.dtype is torch.float32,
            rows, W, total.dtype is torch.float32, eps, dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), ws.numel(),
            _stream(device))
    _lib.check(st, name)
    return dx, dw


@torch.library.custom_op("avgen_amd::add_rms_norm", mutates_args=())
def _add_rms_norm_op(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                     eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, sum)`` of ``x + residual``; see the module docstring."""
    return _add_rms_norm_impl(x, residual, weight, eps)


@_add_rms_norm_op.register_fake
def _(x, residual, weight, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape)


@torch.library.custom_op("avgen_amd::add_rms_norm_bwd", mutates_args=())
def _add_rms_norm_bwd_op(dnorm: torch.Tensor, dsum: Optional[torch.Tensor], total: torch.Tensor,
                         weight: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(dx, dweight)``: the gradient of both addends, and of the gain."""
    return _add_rms_norm_bwd_impl(dnorm, dsum, total, weight, eps)


@_add_rms_norm_bwd_op.register_fake
def _(dnorm, dsum, total, weight, eps):
    return total.new_empty(total.shape), weight.new_empty(weight.shape)


@torch.library.custom_op("avgen_amd::add_rms_norm_fp8", mutates_args=())
def _add_rms_norm_fp8_op(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                         eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(codes, scale, sum)``: the norm as e4m3 with a scale per row."""
    return _add_rms_norm_fp8_impl(x, residual, weight, eps)


@_add_rms_norm_fp8_op.register_fake
def _(x, residual, weight, eps):
    return (x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(x.shape[:-1], dtype=torch.float32),
            x.new_empty(x.shape))


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                 eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``(norm, sum)`` of ``x + residual``; differentiable."""
    return _direct(_AddRmsNorm, _add_rms_norm_op, _add_rms_norm_impl, (x, residual, weight, eps),
                   (x, residual, weight))


def add_rms_norm_bwd(dnorm, dsum, total, weight, eps):
    """``(dx, dweight)`` of ``add_rms_norm`` from its stored sum."""
    if _grad_direct(dnorm, dsum, total, weight):
        return _add_rms_norm_bwd_impl(dnorm, dsum, total, weight, eps)
    return _add_rms_norm_bwd_op(dnorm, dsum, total, weight, eps)


def add_rms_norm_fp8(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor,
                     eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(codes, scale, sum)``: the norm as e4m3 with a scale per row; not
    differentiable."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, residual, weight)):
        raise RuntimeError("avgen_amd.add_rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    return _direct(None, _add_rms_norm_fp8_op, _add_rms_norm_fp8_impl, (x, residual, weight, eps),
                   (x, residual, weight))


def _norm_setup(ctx, inputs, output):
    _x, _residual, weight, ctx.eps = inputs
    ctx.save_for_backward(output[1], weight)


def _norm_backward(ctx, dnorm, dsum):
    total, weight = ctx.saved_tensors
    if dnorm is None:
        # The sum alone was used: its gradient passes through.
        return dsum, dsum, None, None
    dx, dw = add_rms_norm_bwd(dnorm, dsum, total, weight, ctx.eps)
    return dx, dx, dw, None


torch.library.register_autograd("avgen_amd::add_rms_norm", _norm_backward, setup_context=_norm_setup)


class _AddRmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        result = _add_rms_norm_impl(*args)
        ctx.set_materialize_grads(False)
        _norm_setup(ctx, args, result)
        return result

    @staticmethod
    def backward(ctx, dnorm, dsum):
        if dnorm is None or not _grad_direct(dnorm, dsum):
            return _norm_backward(ctx, dnorm, dsum)
        total, weight = ctx.saved_tensors
        dx, dw = _add_rms_norm_bwd_run("avgen_amd.add_rms_norm_bwd", dnorm, dsum, total, weight.contiguous(), ctx.eps)
        return dx, dx, dw, None
