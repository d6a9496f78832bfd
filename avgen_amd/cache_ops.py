"""Ops on a cache of keys and values in pages, and attention over it.

Registered like those of :mod:`avgen_amd.scored_ops` (same checks, streams,
workspaces and errors).  Ops (namespace ``avgen_amd``):

* ``append_paged(...) -> rotated query``, which writes the pages;
* ``page_values(...) -> (key, value)``, what the pages of an e4m3 cache hold;
* ``paged_attention(...) -> (out, lse)``.

None of them is differentiable.  bf16 tensors, head_dim 64 or 128; the layout of
a pool is that of :class:`avgen_amd.cache.PagedCache`, the tables and lengths are
int32 on the GPU and never read by the host.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .block_ops import _on, _one_device, _packed_last
from .ops import SUPPORTED_HEAD_DIMS, _ptr, _stream, _Strides3, _workspace
from .scored_ops import MAX_SLOPE_GROUP, MAX_SOFTCAP_BF16, _deliver, _laid_out, _new_like

__all__ = ["MAX_WINDOW", "PAGE_SIZES", "append_paged", "page_values", "paged_attention"]

#: Slots of a page.
PAGE_SIZES = (16, 32, 64, 128, 256)
#: Largest window of ``paged_attention``.
MAX_WINDOW = 1 << 30

_BF16, _E4M3 = torch.bfloat16, torch.float8_e4m3fn


@lru_cache(maxsize=256)
def _pool_plan(key, value, key_exponent, value_exponent):
    """Of a pool's (shape, strides, type) each, exponents' None without: what
    :func:`check_pool` refuses, else the strides for the C call."""
    shape, _, dtype = key
    if len(shape) != 4 or shape != value[0]:
        raise ValueError(f"pools must be (pages, heads, page_size, head_dim) and agree; got {tuple(shape)} and "
                         f"{tuple(value[0])}")
    pages, heads, page, dim = shape
    if page not in PAGE_SIZES:
        raise ValueError(f"page size {page} not supported (supported: {PAGE_SIZES})")
    if dim not in SUPPORTED_HEAD_DIMS:
        raise ValueError(f"head_dim {dim} not supported (supported: {SUPPORTED_HEAD_DIMS})")
    if heads < 1:
        raise ValueError("a pool needs a head")
    if dtype not in (_BF16, _E4M3) or value[2] is not dtype:
        raise TypeError(f"pools must both be bfloat16 or both float8_e4m3fn; got {dtype} and {value[2]}")
    unit = 16 // dtype.itemsize
    plan = []
    for label, pool, e in (("key", key, key_exponent), ("value", value, value_exponent)):
        sp, sh, ss, sd = pool[1]
        # (Strides of sizes of one may be anything: nothing steps by them.)
        sp, sh = sp if pages > 1 else 0, sh if heads > 1 else 0
        if pages:
            if sd != 1 or ss != dim or sp % unit or sh % unit:
                raise ValueError(f"the slots of a {label} page must be contiguous rows at multiples of 16 bytes "
                                 f"(strides {pool[1]})")
            # Pages and heads in either order, none in another's place.
            least = page * dim
            for s, n in sorted(((sp, pages), (sh, heads))):
                if n > 1:
                    if s < least:
                        raise ValueError(f"{label} pages and heads overlap (strides {pool[1]})")
                    least = s * n
        if (e is not None) is not (dtype is _E4M3):
            raise ValueError("an e4m3 pool has exponents and a bfloat16 one has none")
        es = 0
        if e is not None:
            if e[0] != (pages, heads):
                raise ValueError(f"{label} exponents must be ({pages}, {heads}); got {tuple(e[0])}")
            if e[2] is not torch.int8:
                raise TypeError(f"{label} exponents must be int8; got {e[2]}")
            es = e[1][0] if pages > 1 else 0
            if (heads > 1 and e[1][1] != 1) or (pages > 1 and es < heads):
                raise ValueError(f"the {label} exponents of a page must be contiguous, pages apart")
        plan.append((_Strides3(sp, sh, dim), es))
    return plan


def check_pool(name, key, value, key_exponent, value_exponent):
    """Refuses a pool that the kernels cannot take (but for its device); its
    strides."""
    try:
        plan = _pool_plan(*(None if t is None else (t.shape, t.stride(), t.dtype)
                            for t in (key, value, key_exponent, value_exponent)))
    except (ValueError, TypeError) as e:
        raise type(e)(f"{name}: {e}") from None
    if (key.data_ptr() | value.data_ptr()) % 16:
        raise ValueError(f"{name}: pools must begin at multiples of 16 bytes")
    return plan


def _pool_args(plan, key, value, key_exponent, value_exponent):
    """The C arguments of a pool with these strides: (key, strides, value, strides,
    exponents, stride, exponents, stride)."""
    (ks, kes), (vs, ves) = plan
    if key_exponent is None:
        return key.data_ptr(), ks, value.data_ptr(), vs, None, 0, None, 0
    return key.data_ptr(), ks, value.data_ptr(), vs, key_exponent.data_ptr(), kes, value_exponent.data_ptr(), ves


def _check_tables(name, B, block_table, lengths, counts):
    """(block table, its row stride, lengths, counts), as the kernels read them."""
    if block_table.ndim != 2 or block_table.shape[0] != B:
        raise ValueError(f"{name}: block_table must be ({B}, blocks); got {tuple(block_table.shape)}")
    if block_table.dtype is not torch.int32:
        raise TypeError(f"{name}: block_table must be int32; got {block_table.dtype}")
    for label, t in (("lengths", lengths), ("counts", counts)):
        if t is None:
            continue
        if t.shape != (B,):
            raise ValueError(f"{name}: {label} must be ({B},); got {tuple(t.shape)}")
        if t.dtype is not torch.int32:
            raise TypeError(f"{name}: {label} must be int32; got {t.dtype}")
    stride, step = block_table.stride()
    if (step != 1 and block_table.shape[1] > 1) or 0 < stride < block_table.shape[1]:
        block_table = block_table.contiguous()
        stride = block_table.shape[1]
    return (block_table, stride if B > 1 else block_table.shape[1], lengths.contiguous(),
            None if counts is None else counts.contiguous())


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------


def _append_impl(k, v, query, cos, sin, start, half, block_table, lengths, counts, key_pages, value_pages,
                 key_exponent, value_exponent):
    name = "avgen_amd.append_paged"
    pool = (key_pages, value_pages, key_exponent, value_exponent)
    plan = check_pool(name, *pool)
    pages, heads, page, D = key_pages.shape
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError(f"{name}: key and value must be (batch, heads, length, head_dim) and agree; got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, H, L, _ = k.shape
    if H != heads or k.shape[3] != D:
        raise ValueError(f"{name}: key {tuple(k.shape)} does not fit pages of {heads} heads of {D}")
    for label, t in (("key", k), ("value", v), ("query", query)):
        if t is not None and t.dtype is not _BF16:
            raise TypeError(f"{name}: {label} must be bfloat16; got {t.dtype}")
    if query is not None and (query.ndim != 4 or query.shape[0] != B or query.shape[2] != L or query.shape[3] != D):
        raise ValueError(f"{name}: query {tuple(query.shape)} and key {tuple(k.shape)} differ in more than their heads")
    tsb = pairs = 0
    if (cos is None) is not (sin is None):
        raise ValueError(f"{name}: pass both rotary tables or neither")
    if cos is not None:
        table = cos.shape
        if len(table) != 4 or table != sin.shape:
            raise ValueError(f"{name}: rotary tables must be (batch, 1, length, pairs) and agree")
        if cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
            raise TypeError(f"{name}: rotary tables must be float32")
        TB, TH, TL, pairs = table
        if pairs < 1 or start < 0 or start + 2 * pairs > D:
            raise ValueError(f"{name}: channels [{start}, {start + 2 * pairs}) do not lie in a head of {D}")
        if TL != L:
            raise ValueError(f"{name}: sequence length {L} does not match rotary tables built for length {TL}")
        if TB not in (1, B) or TH != 1:
            raise ValueError(f"{name}: rotary tables batch {TB} does not broadcast to {B}")
        cos, sin = cos.contiguous(), sin.contiguous()
        tsb = 0 if TB == 1 else L * pairs
    block_table, bts, lengths, counts = _check_tables(name, B, block_table, lengths, counts)
    device = _one_device(name, k, v, query, cos, sin, block_table, lengths, counts, *pool)
    k, v = _packed_last(k), _packed_last(v)
    out = written = torch.empty_like(query) if query is not None else None
    q_args = (None, None, 0, None, None)
    if query is not None:
        query = _packed_last(query)
        if out.stride(3) != 1:
            written = torch.empty(out.shape, dtype=_BF16, device=device)
        q_args = (query.data_ptr(), _Strides3(*query.stride()[:3]), query.shape[1], written.data_ptr(),
                  _Strides3(*written.stride()[:3]))
    with _on(device):
        st = _lib.load().avattn_append_paged(
            k.data_ptr(), _Strides3(*k.stride()[:3]), v.data_ptr(), _Strides3(*v.stride()[:3]), *q_args,
            B, H, L, D, _ptr(cos), _ptr(sin), tsb, pairs, start, half,
            block_table.data_ptr(), bts, block_table.shape[1], lengths.data_ptr(), _ptr(counts),
            *_pool_args(plan, *pool), pages, page, _stream(device))
    _lib.check(st, name)
    if written is not out:
        out.copy_(written)
    return out


@torch.library.custom_op("avgen_amd::append_paged",
                         mutates_args=("key_pages", "value_pages", "key_exponent", "value_exponent"))
def _append_op(k: torch.Tensor, v: torch.Tensor, query: Optional[torch.Tensor], cos: Optional[torch.Tensor],
               sin: Optional[torch.Tensor], start: int, half: bool, block_table: torch.Tensor, lengths: torch.Tensor,
               counts: Optional[torch.Tensor], key_pages: torch.Tensor, value_pages: torch.Tensor,
               key_exponent: Optional[torch.Tensor], value_exponent: Optional[torch.Tensor]) -> torch.Tensor:
    """Writes keys and values to their pages; the rotated query (without elements
    for none)."""
    out = _append_impl(k, v, query, cos, sin, start, half, block_table, lengths, counts, key_pages, value_pages,
                       key_exponent, value_exponent)
    return k.new_empty(0) if out is None else out


@_append_op.register_fake
def _(k, v, query, cos, sin, start, half, block_table, lengths, counts, key_pages, value_pages, key_exponent,
      value_exponent):
    return k.new_empty(0) if query is None else torch.empty_like(query)


def _no_gradient(name, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad()")


def append_paged(k, v, query, cos, sin, start: int, half: bool, block_table, lengths, counts, key_pages, value_pages,
                 key_exponent, value_exponent):
    """Writes keys and values to their pages; the rotated query, None for none."""
    calls = _lib.direct_calls(k)
    if calls is not None:
        out = calls.append_paged(k, v, query, cos, sin, block_table, lengths, counts, key_pages, value_pages,
                                 key_exponent, value_exponent, start, half)
        if out is not NotImplemented:
            return out
    _no_gradient("avgen_amd.append_paged", k, v, query, cos, sin, key_pages, value_pages)
    out = _append_op(k, v, query, cos, sin, start, half, block_table, lengths, counts, key_pages, value_pages,
                     key_exponent, value_exponent)
    return None if query is None else out


# ---------------------------------------------------------------------------
# What pages hold
# ---------------------------------------------------------------------------


def _values_impl(key_pages, value_pages, key_exponent, value_exponent):
    name = "avgen_amd.page_values"
    pool = (key_pages, value_pages, key_exponent, value_exponent)
    plan = check_pool(name, *pool)
    if key_exponent is None:
        raise ValueError(f"{name}: the pages hold bfloat16 values as they are")
    pages, heads, page, D = key_pages.shape
    device = _one_device(name, *pool)
    key = torch.empty(key_pages.shape, dtype=_BF16, device=device)
    value = torch.empty(key_pages.shape, dtype=_BF16, device=device)
    kp, kps, vp, vps, ke, kes, ve, ves = _pool_args(plan, *pool)
    with _on(device):
        st = _lib.load().avattn_page_values(kp, kps, ke, kes, key.data_ptr(), vp, vps, ve, ves, value.data_ptr(),
                                            pages, heads, page, D, _stream(device))
    _lib.check(st, name)
    return key, value


@torch.library.custom_op("avgen_amd::page_values", mutates_args=())
def _values_op(key_pages: torch.Tensor, value_pages: torch.Tensor, key_exponent: torch.Tensor,
               value_exponent: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The bf16 values of an e4m3 pool."""
    return _values_impl(key_pages, value_pages, key_exponent, value_exponent)


@_values_op.register_fake
def _(key_pages, value_pages, key_exponent, value_exponent):
    return tuple(t.new_empty(t.shape, dtype=_BF16) for t in (key_pages, value_pages))


def page_values(key_pages, value_pages, key_exponent, value_exponent):
    """The bf16 values of an e4m3 pool: ``(key, value)``."""
    args = (key_pages, value_pages, key_exponent, value_exponent)
    calls = _lib.direct_calls(key_pages)
    if calls is not None:
        out = calls.page_values(*args)
        if out is not NotImplemented:
            return out
    return _values_op(*args)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------


@lru_cache(maxsize=256)
def _attention_workspace_size(*sizes: int) -> int:
    return _lib.load().avattn_paged_attention_workspace_size(*sizes)


def _attention_impl(q, key_pages, value_pages, key_exponent, value_exponent, block_table, lengths, counts, slopes,
                    window, scale, softcap):
    name = "avgen_amd.paged_attention"
    pool = (key_pages, value_pages, key_exponent, value_exponent)
    plan = check_pool(name, *pool)
    pages, Hkv, page, D = key_pages.shape
    if q.ndim != 4 or q.shape[3] != D:
        raise ValueError(f"{name}: query must be (batch, heads, length, {D}); got {tuple(q.shape)}")
    if q.dtype is not _BF16:
        raise TypeError(f"{name}: query must be bfloat16; got {q.dtype}")
    B, Hq, Lq, _ = q.shape
    if Hq == 0 or Hq % Hkv:
        raise ValueError(f"{name}: query heads {Hq} must be a multiple of key heads {Hkv}")
    if not 0 <= window <= MAX_WINDOW:
        raise ValueError(f"{name}: window must be from 1 to {MAX_WINDOW} (0: none); got {window}")
    if not (math.isfinite(scale) and scale > 0.0):
        raise ValueError(f"{name}: scale must be positive and finite; got {scale}")
    if not (math.isfinite(softcap) and 0.0 <= softcap <= MAX_SOFTCAP_BF16):
        raise ValueError(f"{name}: softcap must be from 0 (none) to {MAX_SOFTCAP_BF16}; got {softcap}")
    if slopes is not None:
        if slopes.shape != (Hq,):
            raise ValueError(f"{name}: slopes must have one entry per query head ({Hq},); got {tuple(slopes.shape)}")
        if slopes.dtype is not torch.float32:
            raise TypeError(f"{name}: slopes must be float32; got {slopes.dtype}")
        if Hq // Hkv > MAX_SLOPE_GROUP:
            raise ValueError(f"{name}: slopes take at most {MAX_SLOPE_GROUP} query heads per key head; got {Hq // Hkv}")
        slopes = slopes.contiguous()
    block_table, bts, lengths, counts = _check_tables(name, B, block_table, lengths, counts)
    device = _one_device(name, q, *pool, block_table, lengths, counts, slopes)
    given = q
    q, qs = _laid_out(q, False)
    o = _new_like(given, q, qs, False)
    blocks = block_table.shape[1]
    need = _attention_workspace_size(B, Hq, Hkv, Lq, D, blocks, page, window, key_exponent is not None)
    lse = torch.empty((B, Hq, Lq), device=device, dtype=torch.float32)
    ws = _workspace(need, device)
    with _on(device):
        st = _lib.load().avattn_paged_attention(
            q.data_ptr(), qs, B, Hq, Hkv, Lq, D, block_table.data_ptr(), bts, blocks, lengths.data_ptr(), _ptr(counts),
            *_pool_args(plan, *pool), pages, page, window, scale, softcap, _ptr(slopes),
            o[1].data_ptr(), o[2], lse.data_ptr(), ws.data_ptr(), ws.numel(), _stream(device))
    _lib.check(st, name)
    return _deliver(o)[0], lse


@torch.library.custom_op("avgen_amd::paged_attention", mutates_args=())
def _attention_op(q: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
                  key_exponent: Optional[torch.Tensor], value_exponent: Optional[torch.Tensor],
                  block_table: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor],
                  slopes: Optional[torch.Tensor], window: int, scale: float,
                  softcap: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention over pages: ``(out, lse)``."""
    return _attention_impl(q, key_pages, value_pages, key_exponent, value_exponent, block_table, lengths, counts,
                           slopes, window, scale, softcap)


@_attention_op.register_fake
def _(q, key_pages, value_pages, key_exponent, value_exponent, block_table, lengths, counts, slopes, window, scale,
      softcap):
    return torch.empty_like(q), q.new_empty((q.shape[0], q.shape[1], q.shape[2]), dtype=torch.float32)


def paged_attention(q, key_pages, value_pages, key_exponent, value_exponent, block_table, lengths, counts, slopes,
                    window: int, scale: float, softcap: float):
    """Attention of the newest tokens over pages: the output (the op gives the lse
    too)."""
    args = (q, key_pages, value_pages, key_exponent, value_exponent, block_table, lengths, counts, slopes, window,
            scale, softcap)
    calls = _lib.direct_calls(q)
    if calls is not None:
        out = calls.paged_attention(*args)
        if out is not NotImplemented:
            return out
    _no_gradient("avgen_amd.paged_attention", q, key_pages, value_pages, slopes)
    return _attention_op(*args)[0]
