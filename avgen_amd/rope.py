"""Axial 3D rotary embeddings from physical coordinates, on gfx950 kernels.

Drop-in for ``avgen.models.rope`` (src/avgen/models/rope.py): same names,
signatures, argument meaning and exceptions.  Table construction
(:func:`build_rotary_tables`) and the rotation (:func:`apply_rotary`) run as
HIP kernels through ``libavattn.so``; the rotation is bit-identical to the
reference's fp32 elementwise chain (each product rounded separately, one
round to bf16), and differentiable.

Token sequences with integer positions (no reference counterpart):
:func:`build_position_tables`, with :class:`PositionScaling` for longer
contexts, and :func:`rotate_heads` / :func:`rotate_query_key`, which rotate
part of each head in either pair layout.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import nn

from . import block_ops, ops

__all__ = [
    "POSITION_SCALING_MODES",
    "PositionScaling",
    "ROPE_SCALING_MODES",
    "RoPEScaling",
    "RotaryEmbedding",
    "RotaryTables",
    "apply_rotary",
    "build_position_tables",
    "build_rotary_tables",
    "inverse_frequencies",
    "position_frequencies",
    "rotate_heads",
    "rotate_query_key",
    "rope_axis_pairs",
]

#: Frequency-scaling modes (src/avgen/models/rope.py:58).
ROPE_SCALING_MODES: tuple[str, ...] = ("none", "linear", "ntk")


@dataclass(frozen=True)
class RoPEScaling:
    """Frequency scaling for extrapolation (src/avgen/models/rope.py:61-125).

    ``"linear"`` divides positions by the factor; ``"ntk"`` raises the base by
    ``factor ** (dim / (dim - 2))``.  Time uses ``time_factor``; height and
    width use ``spatial_factor``.

    Raises:
        ValueError: unknown mode or a non-positive factor.
    """

    mode: str = "none"
    time_factor: float = 1.0
    spatial_factor: float = 1.0

    def __post_init__(self) -> None:
        if self.mode not in ROPE_SCALING_MODES:
            raise ValueError(f"mode must be one of {ROPE_SCALING_MODES}; got {self.mode!r}")
        for name in ("time_factor", "spatial_factor"):
            value = float(getattr(self, name))
            if not value > 0.0:
                raise ValueError(f"{name} must be positive; got {value!r}")

    @property
    def is_identity(self) -> bool:
        """Whether the frequencies are left untouched."""
        return self.mode == "none" or (self.time_factor == 1.0 and self.spatial_factor == 1.0)

    def factors(self) -> tuple[float, float, float]:
        """Per-axis factors ``(time, height, width)``."""
        return (self.time_factor, self.spatial_factor, self.spatial_factor)


def rope_axis_pairs(head_dim: int) -> tuple[int, int, int]:
    """Rotation-pair budgets ``(time, height, width)`` (src/avgen/models/rope.py:128-157).

    ``pairs = head_dim // 2``; height and width get ``pairs // 3`` each and time
    takes the remainder: 64 -> (12, 10, 10), 128 -> (22, 21, 21).

    Raises:
        ValueError: ``head_dim`` odd or below 6.
    """
    if head_dim < 6 or head_dim % 2 != 0:
        raise ValueError(
            f"head_dim must be an even integer of at least 6 so each rotary axis "
            f"gets at least one channel pair; got {head_dim!r}"
        )
    pairs = head_dim // 2
    spatial = pairs // 3
    return (pairs - 2 * spatial, spatial, spatial)


@dataclass(frozen=True)
class RotaryTables:
    """Per-pair cos/sin tables ``(batch, 1, length, pairs)`` float32
    (src/avgen/models/rope.py:160-216)."""

    cos: torch.Tensor
    sin: torch.Tensor

    @property
    def pairs(self) -> int:
        return int(self.cos.shape[-1])

    @property
    def length(self) -> int:
        return int(self.cos.shape[-2])

    @property
    def device(self) -> torch.device:
        return self.cos.device

    def validate(self) -> None:
        """Raise ValueError (rank/shape) or TypeError (dtype) like the reference."""
        if self.cos.ndim != 4 or self.sin.ndim != 4:
            raise ValueError(
                f"rotary tables must have rank 4 (batch, 1, length, pairs); got "
                f"{tuple(self.cos.shape)} and {tuple(self.sin.shape)}"
            )
        if self.cos.shape != self.sin.shape:
            raise ValueError(
                f"cos and sin must have the same shape; got {tuple(self.cos.shape)} and {tuple(self.sin.shape)}"
            )
        for name, tensor in (("cos", self.cos), ("sin", self.sin)):
            if tensor.dtype is not torch.float32:
                raise TypeError(f"{name} must be float32; got {tensor.dtype}")

    def slice(self, start: int, stop: int) -> "RotaryTables":
        """Tables for tokens ``[start, stop)`` (a context-parallel shard or KV chunk)."""
        return RotaryTables(cos=self.cos[:, :, start:stop], sin=self.sin[:, :, start:stop])


def inverse_frequencies(
    head_dim: int, *, theta: float = 10000.0, scaling: RoPEScaling | None = None
) -> tuple[list[float], list[int], tuple, tuple]:
    """Host-side frequency plan for :func:`build_rotary_tables`.

    Returns ``(inv_freq, axis_of_pair, pos_mul, pos_div)`` where inv_freq is
    computed with the reference's fp32 operations
    (src/avgen/models/rope.py:287-290: ``arange(pairs)/pairs`` then
    ``pow(float32(theta_axis), -exponent)``), evaluated on the CPU.  pos_mul
    is filled in by the caller (time_scale); pos_div[a] is the linear factor
    or None.
    """
    plan = scaling if scaling is not None else RoPEScaling()
    budgets = rope_axis_pairs(head_dim)
    inv: list[float] = []
    axes: list[int] = []
    divs: list[float | None] = [None, None, None]
    for axis, (pairs, factor) in enumerate(zip(budgets, plan.factors())):
        axis_theta = theta
        if plan.mode == "linear" and factor != 1.0:
            divs[axis] = float(factor)
        elif plan.mode == "ntk" and factor != 1.0:
            dim = 2 * pairs
            if dim > 2:
                axis_theta = theta * factor ** (dim / (dim - 2))
        exponent = torch.arange(pairs, dtype=torch.float32) / pairs
        freq = torch.pow(torch.tensor(axis_theta, dtype=torch.float32), -exponent)
        inv.extend(float(f) for f in freq.tolist())
        axes.extend([axis] * pairs)
    return inv, axes, (None, None, None), tuple(divs)


def build_rotary_tables(
    coords: torch.Tensor,
    *,
    head_dim: int,
    theta: float = 10000.0,
    time_scale: float = 1.0,
    scaling: RoPEScaling | None = None,
) -> RotaryTables:
    """Tables from ``coords (batch, length, 3)`` float32 (src/avgen/models/rope.py:218-294).

    Raises:
        ValueError: coords not ``(batch, length, 3)``.
        TypeError: coords not float32.
    """
    if coords.ndim != 3 or coords.shape[-1] != 3:
        raise ValueError(
            f"coords must be (batch, length, 3) as (seconds, row, column); got {tuple(coords.shape)}"
        )
    if coords.dtype is not torch.float32:
        raise TypeError(f"coords must be float32; got {coords.dtype}")
    inv, axes, _, divs = inverse_frequencies(head_dim, theta=theta, scaling=scaling)
    muls = (float(time_scale) if time_scale != 1.0 else None, None, None)
    cos, sin = ops.rope_tables(coords, inv, axes, muls, divs)
    return RotaryTables(cos=cos, sin=sin)


def apply_rotary(x: torch.Tensor, tables: RotaryTables) -> torch.Tensor:
    """Interleaved-pair rotation of ``x (batch, heads, length, head_dim)``
    (src/avgen/models/rope.py:297-338); returns a new tensor in x's dtype.

    Raises:
        ValueError: rank != 4, head_dim or length disagreeing with the tables.
    """
    if x.ndim != 4:
        raise ValueError(f"rotary input must be (batch, heads, length, head_dim); got {tuple(x.shape)}")
    if x.shape[-1] != 2 * tables.pairs:
        raise ValueError(
            f"head_dim {x.shape[-1]} does not match rotary tables built for head_dim {2 * tables.pairs}"
        )
    if x.shape[-2] != tables.length:
        raise ValueError(
            f"sequence length {x.shape[-2]} does not match rotary tables built for length {tables.length}; "
            "under context parallelism the tables must be built from the local coordinate shard"
        )
    return ops.rope_apply(x, tables.cos, tables.sin, False)


class RotaryEmbedding(nn.Module):
    """Stateless coords -> tables module (src/avgen/models/rope.py:341-401)."""

    def __init__(
        self,
        head_dim: int,
        *,
        theta: float = 10000.0,
        time_scale: float = 1.0,
        scaling: RoPEScaling | None = None,
    ) -> None:
        super().__init__()
        rope_axis_pairs(head_dim)
        self.head_dim = head_dim
        self.theta = theta
        self.time_scale = time_scale
        self.scaling = scaling if scaling is not None else RoPEScaling()

    def forward(self, coords: torch.Tensor) -> RotaryTables:
        return build_rotary_tables(
            coords, head_dim=self.head_dim, theta=self.theta, time_scale=self.time_scale, scaling=self.scaling
        )

    def extra_repr(self) -> str:
        budgets = rope_axis_pairs(self.head_dim)
        return (
            f"head_dim={self.head_dim}, pairs(t,h,w)={budgets}, theta={self.theta}, "
            f"time_scale={self.time_scale}, scaling={self.scaling.mode}"
        )


# ---------------------------------------------------------------------------
# Token sequences: positions in one dimension, part of the head, either layout
# (no reference counterpart)
# ---------------------------------------------------------------------------

#: Modes of :class:`PositionScaling`.
POSITION_SCALING_MODES: tuple[str, ...] = ("none", "linear", "ntk", "yarn")


@dataclass(frozen=True)
class PositionScaling:
    """Scaling of 1D rotary frequencies for contexts ``factor`` times longer
    than the ``original_length`` they were trained for.

    With ``f_p = theta ** (-2 p / rotary_dim)``:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: ``theta`` raised by ``factor ** (d / (d - 2))``, ``d`` the
      rotary width;
    * ``"yarn"`` (Peng et al., 2023): a pair that turns more than ``beta_fast``
      times over the original length keeps its frequency, one that turns less
      than ``beta_slow`` times has it divided by ``factor``, linearly in the
      turns between; cos and sin are multiplied by ``attention_factor``
      (default ``0.1 ln(factor) + 1``, 1 for factors up to 1).

    Raises:
        ValueError: unknown mode, a non-positive factor, original length or
            attention factor, or ``beta_fast <= beta_slow``.
    """

    mode: str = "none"
    factor: float = 1.0
    original_length: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def __post_init__(self) -> None:
        if self.mode not in POSITION_SCALING_MODES:
            raise ValueError(f"mode must be one of {POSITION_SCALING_MODES}; got {self.mode!r}")
        if not (float(self.factor) > 0.0 and math.isfinite(self.factor)):
            raise ValueError(f"factor must be positive; got {self.factor!r}")
        if self.mode == "yarn":
            if not self.original_length > 0:
                raise ValueError(f"original_length must be positive; got {self.original_length!r}")
            if not self.beta_fast > self.beta_slow:
                raise ValueError(f"beta_fast must exceed beta_slow; got {self.beta_fast!r} and {self.beta_slow!r}")
            a = self.attention_factor
            if a is not None and not (a > 0.0 and math.isfinite(a)):
                raise ValueError(f"attention_factor must be positive; got {a!r}")


def position_frequencies(
    rotary_dim: int, *, theta: float = 10000.0, scaling: PositionScaling | None = None
) -> tuple[list[float], float]:
    """The ``rotary_dim / 2`` frequencies and the amplitude of the tables, in
    double precision.

    Raises:
        ValueError: ``rotary_dim`` odd, below 2 or above twice
            ``block_ops.MAX_TABLE_PAIRS``, or a non-positive ``theta``.
    """
    if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > 2 * block_ops.MAX_TABLE_PAIRS:
        raise ValueError(f"rotary_dim must be even, from 2 to {2 * block_ops.MAX_TABLE_PAIRS}; got {rotary_dim!r}")
    if not (theta > 0.0 and math.isfinite(theta)):
        raise ValueError(f"theta must be positive; got {theta!r}")
    plan = scaling if scaling is not None else PositionScaling()
    if plan.mode == "ntk" and rotary_dim > 2:
        theta = theta * plan.factor ** (rotary_dim / (rotary_dim - 2))
    freq = [theta ** (-2.0 * p / rotary_dim) for p in range(rotary_dim // 2)]
    if plan.mode == "linear":
        return [f / plan.factor for f in freq], 1.0
    if plan.mode != "yarn":
        return freq, 1.0
    scaled = []
    for f in freq:
        turns = plan.original_length * f / (2.0 * math.pi)
        keep = min(1.0, max(0.0, (turns - plan.beta_slow) / (plan.beta_fast - plan.beta_slow)))
        scaled.append(f * (keep + (1.0 - keep) / plan.factor))
    if plan.attention_factor is not None:
        return scaled, float(plan.attention_factor)
    return scaled, 0.1 * math.log(plan.factor) + 1.0 if plan.factor > 1.0 else 1.0


def build_position_tables(
    positions: torch.Tensor,
    *,
    rotary_dim: int,
    theta: float = 10000.0,
    scaling: PositionScaling | None = None,
) -> RotaryTables:
    """Tables of a token sequence: ``positions`` int32 or int64 ``(length,)`` or
    ``(batch, length)`` on the GPU, for :func:`rotate_heads` and
    :func:`rotate_query_key` (and, with ``rotary_dim`` the head's width and the
    interleaved layout, for everything that takes :class:`RotaryTables`).
    Angles are formed and reduced in double precision: far positions lose
    nothing.

    Raises:
        ValueError: wrong rank, or what :func:`position_frequencies` refuses.
        TypeError: positions not int32 or int64.
    """
    if positions.ndim not in (1, 2):
        raise ValueError(f"positions must be (length,) or (batch, length); got {tuple(positions.shape)}")
    freq, amplitude = position_frequencies(rotary_dim, theta=theta, scaling=scaling)
    cos, sin = block_ops.position_tables(positions[None] if positions.ndim == 1 else positions, freq, amplitude)
    return RotaryTables(cos=cos, sin=sin)


def _half_layout(layout: str) -> bool:
    if layout not in ("interleaved", "half"):
        raise ValueError(f"layout must be 'interleaved' or 'half'; got {layout!r}")
    return layout == "half"


def rotate_heads(
    x: torch.Tensor, tables: RotaryTables, *, layout: str = "interleaved", start: int = 0
) -> torch.Tensor:
    """:func:`apply_rotary` on part of each head and in either pair layout:
    channels ``[start, start + 2 * tables.pairs)`` of ``x (batch, heads,
    length, head_dim)`` are rotated, the others copied.

    ``layout``: pair ``p`` is channels ``2p, 2p + 1`` of that range
    (``"interleaved"``) or ``p, pairs + p`` (``"half"``).  bf16 or float32, any
    head_dim; fp32 arithmetic rounded once to x's dtype; differentiable in
    ``x``.  Returns a new tensor.

    Raises:
        ValueError: rank, length, channels or batch that do not fit the tables,
            or an unknown layout.
        TypeError: dtype other than bf16 or float32.
    """
    return block_ops.rotate(x, tables.cos, tables.sin, int(start), _half_layout(layout), False)


def rotate_query_key(
    query: torch.Tensor, key: torch.Tensor, tables: RotaryTables, *, layout: str = "interleaved", start: int = 0
) -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`rotate_heads` of a query and a key of the same tokens (any head
    counts) in one launch, forward and backward."""
    return block_ops.rotate_pair(query, key, tables.cos, tables.sin, int(start), _half_layout(layout), False)
