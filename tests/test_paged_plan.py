"""Which of its two ways attention over pages takes, by the workspace it asks for: a
few rows in place, many over a copy of the pages."""

from __future__ import annotations

import pytest

from avgen_amd import _lib


def in_place(B, Hq, Hkv, tokens, keys, D, e4m3, window=0, page=64):
    """The in-place way asks for whole slots of its row blocks' parts (or nothing),
    the other for copies of keys and values and more."""
    size = _lib.load().avattn_paged_attention_workspace_size(B, Hq, Hkv, tokens, D, -(-keys // page), page, window,
                                                             e4m3)
    rows = tokens * (Hq // Hkv)
    block = min(rows, 32)
    slot = 4 * (block * (D + 3) + -(block * (D + 3)) % 4)
    return size % (slot * B * Hkv * -(-rows // 32)) == 0


@pytest.mark.parametrize("B, Hq, Hkv, D, keys, e4m3, few, many", [
    # The most tokens that are at least 15 % faster in place, and the least that are over a
    # copy (us in place, over a copy at either).
    (1, 32, 8, 128, 12000, 1, 128, 192),  # 54, 68; 86, 70
    (2, 32, 8, 128, 12000, 1, 96, 192),  # 89, 102; 140, 109
    (4, 32, 8, 128, 12000, 1, 96, 256),  # 140, 200; 326, 224
    (8, 32, 8, 128, 4000, 1, 96, 192),  # 101, 119; 171, 130
    (1, 64, 8, 128, 1000, 1, 256, 512),  # 23, 33; 39, 34
    (1, 16, 2, 64, 12000, 1, 128, 384),  # 33, 41; 72, 53
    (4, 16, 2, 64, 12000, 1, 33, 96),  # 36, 47; 72, 50
    (1, 32, 8, 128, 12000, 0, 64, 128),  # 47, 68; 81, 71
    (2, 32, 8, 128, 12000, 0, 64, 96),  # 88, 110; 128, 113
    (4, 32, 8, 128, 12000, 0, 48, 128),  # 128, 212; 302, 221
    (4, 32, 8, 128, 4000, 0, 33, 96),  # 61, 80; 105, 83
    (8, 32, 8, 128, 1000, 0, 17, 64),  # 23, 38; 49, 39
    (8, 32, 8, 128, 4000, 0, 17, 128),  # 75, 131; 209, 145
    (1, 64, 8, 128, 4000, 0, 64, 192),  # 36, 49; 94, 54
    (4, 16, 2, 64, 12000, 0, 17, 96),  # 24, 47; 74, 51
])
def test_the_faster_way(B, Hq, Hkv, D, keys, e4m3, few, many):
    assert in_place(B, Hq, Hkv, few, keys, D, e4m3)
    assert not in_place(B, Hq, Hkv, many, keys, D, e4m3)


def test_single_tokens_are_always_in_place():
    for B in (1, 3, 64):
        for keys in (64, 5000, 130000):
            for window in (0, 100):
                assert in_place(B, 32, 8, 1, keys, 128, 1, window) and in_place(B, 64, 1, 1, keys, 64, 0, window)
