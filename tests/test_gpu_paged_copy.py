"""Attention over pages by way of a copy (many rows), with several kv heads whose
exponents differ, and its row sums: each case is checked to take that way."""

from __future__ import annotations

import pytest
import torch

import tests.paged_reference as ref
from avgen_amd.cache import PagedCache, paged_attention
from tests.test_gpu_paged import B16, F8, UNIT, check_attention, filled, heads, i32, launched, table_of

pytestmark = pytest.mark.gpu

HQ, H, L = 64, 4, 448  # rows enough for the copy also where a window leaves few keys


def pool(pages, page, D, dtype, seed):
    """Heads of magnitudes 2^-6, 2^-2, 2^2 and 2^6 of one another."""
    cache = filled(pages, H, page, D, dtype, seed)
    for n in range(H):
        for t, e in ((cache.key, cache.key_exponent), (cache.value, cache.value_exponent)):
            step = 4 * n - 6
            if e is None:
                t[:, n] *= 2.0**step
            else:
                e[:, n] += step
    return cache


def queries(B, D, seed):
    """Each kv head's queries scaled against its keys."""
    q = heads(B, HQ, L, D, seed, 2.0)
    scale = torch.exp2(6.0 - 4.0 * (torch.arange(HQ, device="cuda") // (HQ // H)))
    return (q.float() * scale[:, None, None]).to(B16).transpose(1, 2).contiguous().transpose(1, 2)


def check_rows(q, cache, rows, lengths, counts=None, **options):
    """check_attention, and the op's lse, -inf exactly where a row has no key."""
    out = check_attention(q, cache, rows, lengths, counts, **options)
    scale = options.get("scale") or q.shape[3] ** -0.5
    op, lse = torch.ops.avgen_amd.paged_attention(
        q, cache.key, cache.value, cache.key_exponent, cache.value_exponent, i32(rows), i32(lengths),
        None if counts is None else i32(counts), options.get("slopes"), options.get("window") or 0, scale,
        options.get("cap") or 0.0)
    assert torch.equal(op, out)
    key, value = (t.cpu().double() for t in cache.values())
    _, want, _, score = ref.attend(
        q.cpu().double(), key, value, rows, lengths, counts or [q.shape[2]] * q.shape[0],
        window=options.get("window") or 0, cap=options.get("cap") or 0.0, scale=options.get("scale"),
        slopes=None if options.get("slopes") is None else options["slopes"].cpu().double())
    # The largest score's error (as in check_attention), the sum's over the keys, and a
    # few operations on the logarithm.
    D, n = q.shape[3], cache.page_size * len(rows[0])
    tol = ((D + 16) * UNIT * score + (2.0**-20 * options["cap"] if options.get("cap") else 0.0) + (n + 8) * UNIT
           + 4 * UNIT * want.abs().nan_to_num(posinf=0.0))
    lse, none = lse.cpu().double(), want.isinf()
    assert lse.shape == want.shape and torch.equal(lse == -float("inf"), none)
    diff = torch.where(none, 0.0, (lse - want).abs())
    assert bool((diff <= tol).all()), f"lse: {float((diff / tol).max()):.3f} of the tolerance"
    return out


def takes_the_copy(q, cache, rows, lengths, counts=None, kernel="prep_paged", **options):
    return launched(kernel, lambda: paged_attention(
        q, cache, i32(rows), i32(lengths), counts=None if counts is None else i32(counts),
        window=options.get("window"), softcap=options.get("cap"), distance_slopes=options.get("slopes"),
        scale=options.get("scale")))


def slopes(sign=1.0):
    return sign * torch.linspace(0.001, 0.2, HQ, device="cuda")


OPTIONS = {"plain": {}, "window": dict(window=70), "narrow": dict(window=1), "cap": dict(cap=15.0),
           "slopes": dict(slopes=1.0), "negative slopes": dict(slopes=-0.2), "scale": dict(scale=0.2),
           "all": dict(window=130, cap=20.0, slopes=1.0, scale=0.15)}


def given(name):
    options = dict(OPTIONS[name])
    if "slopes" in options:
        options["slopes"] = slopes(options["slopes"])
    return options


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", OPTIONS)
def test_heads_of_different_exponents(name, D, dtype):
    lengths = [L + 333, L]
    rows, pages = table_of(lengths, 32, seed=3)
    cache, q, options = pool(pages, 32, D, dtype, 17), queries(2, D, 3), given(name)
    check_rows(q, cache, rows, lengths, **options)
    assert takes_the_copy(q, cache, rows, lengths, **options)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_counts_out_of_range_and_tokens_without_a_position(page, dtype):
    """Padding, no tokens, more counted than there are, tokens in front of position 0, a
    negative length, and slots behind a sequence that hold anything."""
    lengths, counts = [L + 20, 100, L - 60, 0, 57, -3], [2, 0, L, L, L + 9, 1]
    rows, pages = table_of([max(n, 1) for n in lengths], page)
    cache, q = pool(pages, page, 64, dtype, 9), queries(6, 64, 5)
    for r, n in zip(rows, lengths):
        if n > 0 and n % page:
            for t in (cache.key, cache.value):
                t[r[n // page], :, n % page:].view(torch.uint8).fill_(0xFF)
    for options in ({}, dict(window=33), dict(slopes=slopes())):
        out = check_rows(q, cache, rows, lengths, counts, **options)
        assert not bool(out[0, :, 2:].any() or out[1].any() or out[3].any() or out[5].any())
        assert not bool(out[2, :, :60].any()) and bool(out[2, :, 60:].any())
        assert takes_the_copy(q, cache, rows, lengths, counts, **options)


@pytest.mark.parametrize("dtype", [B16, F8])
def test_entries_that_name_no_page(dtype):
    """Shared by all heads: the keys of such a page are none of any head's."""
    lengths = [L + 200, L + 130]
    rows, pages = table_of(lengths, 16)
    rows[0][3], rows[0][4], rows[1][0], rows[1][-1] = -1, pages, 2**31 - 1, -(2**31)
    cache, q = pool(pages, 16, 128, dtype, 11), queries(2, 128, 6)
    for options in ({}, dict(window=40), dict(cap=9.0)):
        check_rows(q, cache, rows, lengths, **options)
        assert takes_the_copy(q, cache, rows, lengths, **options)
    gone = [[-1] * len(rows[0]), rows[1]]
    assert not bool(check_rows(q, cache, gone, lengths)[0].any())


@pytest.mark.parametrize("dtype", [B16, F8])
def test_lengths_past_the_table(dtype):
    rows, pages = table_of([L + 64, L + 64], 16)
    cache, q = pool(pages, 16, 64, dtype, 15), queries(2, 64, 8)
    for n, options in ((L + 64 + 30, {}), (L + 64 + 30, dict(window=60 + L)), (2**31 - 1, {})):
        check_rows(q, cache, rows, [n, L + 64], **options)
        assert takes_the_copy(q, cache, rows, [n, L + 64], **options)


@pytest.mark.parametrize("dtype", [B16, F8])
def test_layouts(dtype):
    """A joint pool, pages by head, strided tables and queries: the same bits."""
    lengths = [L + 30, L + 150]
    rows, pages = table_of(lengths, 16)
    cache, q = pool(pages, 16, 64, dtype, 17), queries(2, 64, 10)
    want = check_rows(q, cache, rows, lengths)
    assert takes_the_copy(q, cache, rows, lengths)
    joint = torch.stack([cache.key.view(torch.uint8), cache.value.view(torch.uint8)], 1).view(dtype)
    e = (None, None) if dtype is B16 else torch.stack([cache.key_exponent, cache.value_exponent], 1).unbind(1)
    by_head = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (cache.key, cache.value)]
    for other in (PagedCache(joint[:, 0], joint[:, 1], *e),
                  PagedCache(*by_head, cache.key_exponent, cache.value_exponent)):
        assert torch.equal(paged_attention(q, other, i32(rows), i32(lengths)), want)
    table = i32(rows).t().contiguous().t()
    assert torch.equal(paged_attention(q, cache, table, i32([lengths, lengths]).t()[:, 0]), want)
    strided = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(paged_attention(strided, cache, i32(rows), i32(lengths)), want)


# Rows on at most half the CUs, which are split over ranges of keys, and that go over the
# copy also where a window leaves few keys.
WIDE = {64: 320, 128: 512}


@pytest.mark.parametrize("dtype, D, options", [
    (F8, 64, {}), (F8, 128, {}), (B16, 64, {}), (B16, 128, {}), (B16, 64, dict(window=700)),
    (F8, 128, dict(window=700)), (B16, 128, dict(window=30)), (F8, 128, dict(window=30)), (F8, 64, dict(cap=15.0)),
    (B16, 128, dict(cap=15.0)), (B16, 64, dict(slopes=1.0)), (F8, 128, dict(slopes=-0.05)),
    (B16, 128, dict(window=200, cap=15.0, slopes=1.0)),
], ids=str)
def test_split_over_the_keys(dtype, D, options):
    """Parts of the keys, with windows also parts without a key."""
    rows, pages = table_of([6000], 64, seed=4)
    cache = pool(pages, 64, D, dtype, 18)
    q = torch.cat([queries(1, D, 4), queries(1, D, 5)], 2)[:, :, :WIDE[D]]
    options = dict(options)
    if "slopes" in options:
        options["slopes"] = slopes(options["slopes"])
    check_rows(q, cache, rows, [6000], **options)
    assert takes_the_copy(q, cache, rows, [6000], **options)
    assert takes_the_copy(q, cache, rows, [6000], kernel="lse_merge", **options)


# ---------------------------------------------------------------------------
# The row sums of pages read in place
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name", OPTIONS)
@pytest.mark.parametrize("tokens, keys", [(1, 40), (1, 3000), (3, 700), (40, 900)])
def test_row_sums_in_place(tokens, keys, name, D, dtype):
    """Whole and joined from parts, with padded rows and a sequence without keys."""
    lengths, counts = [keys, max(tokens, keys // 3), 0], [tokens, (tokens + 1) // 2, tokens]
    rows, pages = table_of([max(n, 1) for n in lengths], 16, seed=6)
    cache, options = pool(pages, 16, D, dtype, 21), given(name)
    q = queries(3, D, 22)[:, :, :tokens]
    check_rows(q, cache, rows, lengths, counts, **options)
    assert not takes_the_copy(q, cache, rows, lengths, counts, **options)
