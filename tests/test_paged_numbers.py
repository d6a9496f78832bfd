"""Numbers no 64-bit integer holds, refused like those out of range (without a GPU:
the checks are before any launch)."""

from __future__ import annotations

import pytest

from avgen_amd.cache import append_paged, paged_attention
from tests.test_paged import K, LEN, POOL, Q, T, TABLE


@pytest.mark.parametrize("window", [0, -1, (1 << 30) + 1, 1 << 40, 1 << 70, -(1 << 70)])
def test_windows_out_of_range(window):
    with pytest.raises(ValueError, match="window"):
        paged_attention(Q, POOL, TABLE, LEN, window=window)


@pytest.mark.parametrize("start", [-1, 128, 1 << 40, 1 << 70, -(1 << 70)])
def test_starts_out_of_range(start):
    with pytest.raises(ValueError, match="start"):
        append_paged(POOL, K, K, TABLE, LEN, tables=T, start=start)
    with pytest.raises(RuntimeError, match="no CPU path"):  # no rotation: no channel to start at
        append_paged(POOL, K, K, TABLE, LEN, start=start)


@pytest.mark.parametrize("softcap", [0.0, -1.0, 1e-60, 1e-40, float("nan"), float("inf"), 1025.0])
def test_caps_out_of_range(softcap):
    """Also those that are 0 in float32, which stands for none."""
    with pytest.raises(ValueError, match="softcap"):
        paged_attention(Q, POOL, TABLE, LEN, softcap=softcap)
