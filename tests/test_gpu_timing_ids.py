"""Launches of the scored forward under their own timer ids."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import _lib
from avgen_amd import attention as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, prepared", [(torch.bfloat16, 1), (torch.float32, 0)])
@pytest.mark.parametrize("monotone", [False, True])
def test_range_of_unsorted_windows_is_not_an_operand_copy(monotone, dtype, prepared):
    q = torch.randn((1, 160, 300, 64), device="cuda").to(dtype)
    lo = torch.zeros(300, device="cuda", dtype=torch.int32)
    hi = torch.arange(1, 301, device="cuda", dtype=torch.int32)
    A.scored_attention(q, q, q, softcap=5.0, window_lo=lo, window_hi=hi, monotone=monotone)
    with _lib.LaunchTiming(64) as timing:
        A.scored_attention(q, q, q, softcap=5.0, window_lo=lo, window_hi=hi, monotone=monotone)
        torch.cuda.synchronize()
        assert timing.read("window_hull")[1] == (0 if monotone else 1)
        assert timing.read("transpose")[1] == prepared
    timing.close()
