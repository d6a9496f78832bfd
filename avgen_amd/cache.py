"""A cache of keys and values in pages, for serving (no reference counterpart).

Sequences of any lengths share a pool of pages; a block table names the pages of
each.  :func:`append_paged` writes the newest tokens (rotating the keys, and the
query with them, on the way), :func:`paged_attention` reads them.  Pages hold
bfloat16, or e4m3 codes with an exponent for each page and head, at half the
memory and half the bytes of a decode step.

Everything that changes from step to step (lengths, tables, pages) is device
data that the host never reads, so a step can be captured once and replayed.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import cache_ops, ops
from .block_ops import _one_device
from .rope import RotaryTables, _half_layout

__all__ = ["PagedCache", "append_paged", "paged_attention"]


@dataclass(frozen=True, eq=False)
class PagedCache:
    """A pool of pages: ``key`` and ``value`` ``(pages, heads, page_size,
    head_dim)``, bfloat16 or float8_e4m3fn, on the GPU.

    Token ``t`` of a sequence is in slot ``t % page_size`` of the page that its
    block table names at ``t // page_size``.  With e4m3, ``key_exponent`` and
    ``value_exponent`` (int8 ``(pages, heads)``) scale a page's codes: a value is
    ``code * 2 ** exponent``, which bfloat16 holds exactly for the exponents that
    :func:`append_paged` chooses, -110 to 119.  Pages that a program fills itself may
    have any: past 119 the largest values are infinite in bfloat16, and attention takes
    -127 and -128 as -126.

    page_size is 16, 32, 64, 128 or 256, head_dim 64 or 128; the slots of a page
    and head are contiguous, pages and heads may have any strides of whole 16
    bytes (so ``pool[:, 0]`` and ``pool[:, 1]`` of a joint pool serve).  Pages
    need no clearing: a slot that no token was written to never counts.

    Raises:
        ValueError: shapes, page sizes or layouts other than these.
        TypeError: types other than these.
        RuntimeError: a tensor that is not on the GPU, or not on the same one.
    """

    key: torch.Tensor
    value: torch.Tensor
    key_exponent: torch.Tensor | None = None
    value_exponent: torch.Tensor | None = None

    def __post_init__(self) -> None:
        tensors = (self.key, self.value, self.key_exponent, self.value_exponent)
        cache_ops.check_pool("PagedCache", *tensors)
        _one_device("PagedCache", *tensors)

    @classmethod
    def empty(
        cls,
        pages: int,
        heads: int,
        page_size: int,
        head_dim: int,
        *,
        dtype: torch.dtype = torch.bfloat16,
        device: torch.device | str = "cuda",
    ) -> "PagedCache":
        """A pool of unwritten pages, with exponents if ``dtype`` is
        float8_e4m3fn."""
        key, value = (torch.empty((pages, heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(2))
        if dtype is not torch.float8_e4m3fn:
            return cls(key, value)
        return cls(key, value, *(torch.zeros((pages, heads), dtype=torch.int8, device=device) for _ in range(2)))

    @property
    def page_size(self) -> int:
        return self.key.shape[2]

    def values(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The pages' keys and values in bfloat16, ``(pages, heads, page_size,
        head_dim)``: the pool itself if it is bfloat16, else exact copies of
        what the codes stand for."""
        if self.key_exponent is None:
            return self.key, self.value
        return cache_ops.page_values(self.key, self.value, self.key_exponent, self.value_exponent)


def append_paged(
    cache: PagedCache,
    key: torch.Tensor,
    value: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    counts: torch.Tensor | None = None,
    tables: RotaryTables | None = None,
    layout: str = "interleaved",
    start: int = 0,
    query: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Writes the keys and values of the newest tokens to their pages, in one
    launch, and returns ``query`` rotated (None without one; without ``tables``
    the query itself).

    Args:
        key, value: bf16 ``(batch, heads, length, head_dim)``, any strides.
        block_table: int32 ``(batch, blocks)`` on the GPU.  An entry outside
            the pool (``-1``) names no page; tokens that fall there, or behind
            the table, are left out.
        lengths: int32 ``(batch,)``: the tokens of each sequence, these
            included.
        counts: int32 ``(batch,)``: how many of the ``length`` tokens are real,
            the rest being padding behind them (None: all).  Token ``i`` is at
            position ``lengths - counts + i``.
        tables, layout, start: the rotation of key and query as for
            :func:`avgen_amd.rope.rotate_query_key` (tables of these tokens,
            padding included); None: written as they are.
        query: bf16 ``(batch, query heads, length, head_dim)``.  Every row is
            rotated, padding included.

    e4m3: the exponent of a page and head is the least from -110 to 119 with ``448 *
    2 ** e >=`` the largest finite magnitude of the tokens that this call writes to the
    page (past that they saturate), and not below its present one if the page holds
    earlier tokens of the sequence.  Where that raises it, the page's other codes are
    rounded again, which changes subnormal codes alone; so a page filled token by token
    and one filled at once may differ in those, and in their exponent.  Of a page that
    the tokens begin, slots behind them keep their codes under the new exponent: they
    hold no token.  Codes are rounded to nearest even from the rotation's fp32 result;
    infinities become NaN.

    A page belongs to one sequence while it is written: sequences may share pages
    that are full.  Writing the same tokens again gives the same pages.  Not
    differentiable.

    Raises:
        ValueError, TypeError: shapes, types or layouts other than these.
        RuntimeError: a tensor not on the GPU, or one that requires grad.
    """
    half = _half_layout(layout)
    cos = sin = None
    rotated, start = query, int(start)
    if tables is not None:
        if not 0 <= start < max(ops.SUPPORTED_HEAD_DIMS):
            raise ValueError(f"start must be a channel of the head; got {start}")
        cos, sin = tables.cos, tables.sin
        rotated = None
    out = cache_ops.append_paged(key, value, query if tables is not None else None, cos, sin,
                                 0 if tables is None else start, half,
                                 block_table, lengths, counts, cache.key, cache.value, cache.key_exponent,
                                 cache.value_exponent)
    return out if rotated is None else rotated


def paged_attention(
    query: torch.Tensor,
    cache: PagedCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    counts: torch.Tensor | None = None,
    window: int | None = None,
    softcap: float | None = None,
    distance_slopes: torch.Tensor | None = None,
    scale: float | None = None,
) -> torch.Tensor:
    """Causal attention of the newest tokens of every sequence over its pages,
    these tokens' keys included (:func:`append_paged` comes first).

    Args:
        query: bf16 ``(batch, heads, length, head_dim)``, heads a multiple of
            the cache's.
        block_table, lengths, counts: as for :func:`append_paged`.  Query ``i`` is at
            position ``p = lengths - counts + i`` and sees the keys ``0 .. p``.
        window: see the keys ``p - window + 1 .. p`` only.  Pages in front
            of every query's window are not read: their entries may be ``-1``.
        softcap, distance_slopes, scale: as for
            :func:`avgen_amd.attention.scored_attention` (softcap up to 1,024,
            slopes of up to 64 query heads per kv head), the distance being
            ``p - key``.

    Returns ``(batch, heads, length, head_dim)`` in the query's layout.  Rows of
    padding, and rows whose keys have no page, are zeros.  Slots outside the
    hull of a sequence's windows may hold anything.  Up to some hundred rows (by
    an estimate of both ways' times, from the sizes) read the pages in place, the
    keys split over the chip; more go over a copy in bfloat16 of the pages, with
    memory for all that the table has room for.  Which way, how the keys are split and
    that memory follow the table's room, since the host does not know the lengths: pass
    the part of the table that is in use.  A captured step needs the room of the
    longest sequence that it is to serve, and shorter ones pay for it: with 16 times the
    room in use single tokens take up to a third longer, 64 tokens up to twice as long,
    512 a quarter to nine tenths (and 4 bytes of copies for each channel and slot of that
    room); so capture one for each of a few rooms.  Not differentiable.

    Raises:
        ValueError, TypeError: shapes, types or values other than these.
        RuntimeError: a tensor not on the GPU, or one that requires grad.
    """
    if softcap is not None and not softcap >= torch.finfo(torch.float32).smallest_normal:  # (0 would be none)
        raise ValueError(f"softcap must be positive or None; got {softcap}")
    if window is not None and not 1 <= window <= cache_ops.MAX_WINDOW:
        raise ValueError(f"window must be from 1 to {cache_ops.MAX_WINDOW} or None; got {window}")
    return cache_ops.paged_attention(
        query, cache.key, cache.value, cache.key_exponent, cache.value_exponent, block_table, lengths, counts,
        distance_slopes, 0 if window is None else int(window),
        ops.default_scale(query.shape[-1]) if scale is None else float(scale),
        0.0 if softcap is None else float(softcap))
