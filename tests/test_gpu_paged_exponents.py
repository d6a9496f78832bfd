"""Pages whose exponents a program set itself, past those that an append chooses."""

from __future__ import annotations

import pytest
import torch

from avgen_amd.cache import paged_attention
from tests.test_gpu_paged import F8, check_append, filled, heads, i32, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [119, 120, 126, 127])
def test_append_behind_tokens_of_a_large_exponent(exponent):
    """An append never lowers the exponent of a page with earlier tokens: the new ones
    are rounded to codes of it."""
    rows, pages = table_of([20], 32)
    cache = filled(pages, 2, 32, 64, F8, 3)
    cache.key_exponent.fill_(exponent)
    cache.value_exponent.fill_(exponent)
    k, v = heads(1, 2, 3, 64, 4, 2.0**125), heads(1, 2, 3, 64, 5, 2.0**126)
    check_append(cache, k, v, rows, [20])
    assert bool((cache.key_exponent[rows[0][0]] == exponent).all())
    assert bool(cache.value[rows[0][0], :, 17:20].float().any())


@pytest.mark.parametrize("Lq", [1, 6])
def test_attention_over_the_least_exponents(Lq):
    """-126 is exact (a power of two on every value of the page), -127 and -128 are
    taken as -126."""
    rows, pages = table_of([70], 16)
    cache = filled(pages, 2, 16, 64, F8, 6)
    q = heads(1, 4, Lq, 64, 7)
    out = {}
    for e in (0, -126, -127, -128):
        cache.value_exponent.fill_(e)
        out[e] = paged_attention(q, cache, i32(rows), i32([70])).float()
    normal = out[0].abs() >= 1.0  # 2^-126 times it is a normal bf16 number
    assert bool(normal.any()) and torch.equal(out[-126][normal], torch.ldexp(out[0], torch.tensor(-126))[normal])
    assert torch.equal(out[-127], out[-126]) and torch.equal(out[-128], out[-126])
