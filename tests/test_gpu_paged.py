"""The paged cache on the GPU: append, values and attention against float64."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import _lib, rope
from avgen_amd.cache import PagedCache, append_paged, paged_attention
from avgen_amd.rope import RotaryTables

import tests.paged_reference as ref

pytestmark = pytest.mark.gpu

B16, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32
HALF = 2.0**-8  # a bf16 rounding
UNIT = 2.0**-24  # a float32 one


def normal(shape, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * spread


def heads(B, H, L, D, seed, spread=1.0):
    """(B, H, L, D) as the view of a (B, L, H*D) projection."""
    return normal((B, L, H * D), seed, spread).to(B16).unflatten(-1, (H, D)).transpose(1, 2)


def i32(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def table_of(lengths, page, seed=0, spare=2):
    """A block table with pages in any order, and the number of pages."""
    per = [max(1, -(-n // page)) for n in lengths]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(per) + spare, generator=g).tolist()
    rows, at = [], 0
    for n in per:
        rows.append(order[at:at + n] + [-1] * (max(per) - n))
        at += n
    return rows, sum(per) + spare


def filled(pages, H, page, D, dtype, seed, spread=1.0):
    """A pool with numbers in every slot, pages of different magnitudes."""
    cache = PagedCache.empty(pages, H, page, D, dtype=dtype)
    scale = torch.exp2(torch.arange(pages, device="cuda") % 5 - 2.0)[:, None, None, None]
    for n, (pool, e) in enumerate(((cache.key, cache.key_exponent), (cache.value, cache.value_exponent))):
        x = normal(pool.shape, seed + n, spread) * scale
        if e is None:
            pool.copy_(x)
        else:
            ex = torch.ceil(torch.log2(x.abs().amax((-1, -2)) / 448.0))
            e.copy_(ex)
            pool.copy_((x * torch.exp2(-ex)[..., None, None]).to(F8))
    return cache


def check_attention(q, cache, rows, lengths, counts=None, **options):
    """The op against the reference, row by row."""
    kwargs = dict(window=options.get("window"), softcap=options.get("cap"), distance_slopes=options.get("slopes"),
                  scale=options.get("scale"))
    out = paged_attention(q, cache, i32(rows), i32(lengths), counts=None if counts is None else i32(counts), **kwargs)
    assert out.shape == q.shape and out.dtype is B16
    key, value = (t.cpu().double() for t in cache.values())
    want, lse, spread, score = ref.attend(
        q.cpu().double(), key, value, rows, lengths, counts or [q.shape[2]] * q.shape[0],
        window=options.get("window") or 0, cap=options.get("cap") or 0.0, scale=options.get("scale"),
        slopes=None if options.get("slopes") is None else options["slopes"].cpu().double())
    # The output's rounding; those of the probabilities to bf16, relative to sum p
    # |v|; the scores' sums of D products and their change (a dozen float32
    # operations, the cap's within 2^-22 of it), twice since they enter the sum too; the sums over the
    # keys.
    D, n = q.shape[3], cache.page_size * len(rows[0])
    s = (D + 16) * UNIT * score + (2.0**-20 * options["cap"] if options.get("cap") else 0.0)
    tol = HALF * want.abs() + (HALF + 2 * s + n * UNIT)[..., None] * spread + 1e-30
    diff = (out.cpu().double() - want).abs()
    assert bool((diff <= tol).all()), f"{float((diff / tol).max()):.3f} of the tolerance"
    return out


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_single_tokens_of_ragged_sequences(page, D, dtype):
    lengths = [1, 15, 16, 17, 31, 33, 64, 65, 200, 517]
    rows, pages = table_of(lengths, page)
    cache = filled(pages, 2, page, D, dtype, page + D)
    check_attention(heads(len(lengths), 8, 1, D, 1, 2.0), cache, rows, lengths)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("Lq, Hq, H", [(1, 1, 1), (2, 4, 4), (7, 8, 2), (8, 64, 1), (32, 4, 2), (33, 2, 2), (64, 4, 4),
                                       (40, 8, 1), (300, 4, 2)])
def test_rows_of_every_kind(Lq, Hq, H, dtype):
    """One row block and several, and more rows than the few-row kernel takes."""
    lengths = [Lq, Lq + 100, 2 * Lq + 333]
    rows, pages = table_of(lengths, 16, seed=Lq)
    cache = filled(pages, H, 16, 128, dtype, Lq)
    check_attention(heads(3, Hq, Lq, 128, 2, 2.0), cache, rows, lengths)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("Lq", [1, 5, 70])
@pytest.mark.parametrize("window", [1, 16, 33, 1000])
def test_window(window, Lq, dtype):
    lengths = [Lq, 90, 411]
    rows, pages = table_of(lengths, 32)
    cache = filled(pages, 2, 32, 64, dtype, 5)
    # Pages in front of every window may be gone.
    for r, n in zip(rows, lengths):
        for block in range(max(0, n - Lq - window + 1) // 32):
            r[block] = -1
    check_attention(heads(3, 4, Lq, 64, 3, 2.0), cache, rows, lengths, window=window)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("Lq", [1, 6, 80])
@pytest.mark.parametrize("score", ["cap", "slopes", "negative slopes", "both", "scale"])
def test_scores(score, Lq, dtype):
    lengths = [Lq + 3, 700]
    rows, pages = table_of(lengths, 64)
    cache = filled(pages, 2, 64, 128, dtype, 7)
    slopes = torch.tensor([0.5, 0.1, 0.02, 0.0], device="cuda")
    options = {"cap": dict(cap=3.0), "slopes": dict(slopes=slopes), "negative slopes": dict(slopes=-0.1 * slopes),
               "both": dict(cap=20.0, slopes=slopes), "scale": dict(scale=0.3)}[score]
    check_attention(heads(2, 4, Lq, 128, 4, 2.0), cache, rows, lengths, **options)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("Lq", [4, 90])
def test_counts_and_empty_rows(Lq, dtype):
    """Padding behind the tokens, a sequence without tokens, one whose tokens reach
    in front of position 0, counts out of range."""
    lengths, counts = [Lq + 20, 100, 2, 0, 57, -3], [2, 0, Lq, Lq, Lq + 9, 1]
    rows, pages = table_of([max(n, 1) for n in lengths], 16)
    cache = filled(pages, 2, 16, 64, dtype, 9)
    out = check_attention(heads(6, 4, Lq, 64, 5), cache, rows, lengths, counts)
    assert bool((out[0, :, 2:] == 0).all() and (out[1] == 0).all() and (out[3] == 0).all() and (out[5] == 0).all())


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("Lq", [1, 70])
def test_entries_that_name_no_page(Lq, dtype):
    lengths = [200, 130, 70]
    rows, pages = table_of(lengths, 16)
    rows[0][3], rows[0][4], rows[1][0] = -1, pages, 2**31 - 1
    rows[2][:5] = [-(2**31)] * 5  # every page of that one
    cache = filled(pages, 2, 16, 128, dtype, 11)
    out = check_attention(heads(3, 2, Lq, 128, 6), cache, rows, lengths)
    assert bool((out[2] == 0).all())


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("Lq", [1, 50])
def test_what_unused_slots_hold_never_counts(Lq, dtype):
    lengths = [Lq + 7, 90]
    rows, pages = table_of(lengths, 32)
    cache = filled(pages, 2, 32, 64, dtype, 13)
    q = heads(2, 4, Lq, 64, 7)
    first = paged_attention(q, cache, i32(rows), i32(lengths))
    used = torch.zeros(pages, 32, dtype=torch.bool)
    for r, n in zip(rows, lengths):
        for t in range(n):
            used[r[t // 32], t % 32] = True
    nan = float("nan")
    for pool in (cache.key, cache.value):
        pool.copy_(torch.where(used.cuda()[:, None, :, None], pool.float(), nan).to(pool.dtype))
    assert torch.equal(paged_attention(q, cache, i32(rows), i32(lengths)), first)


@pytest.mark.parametrize("Lq", [1, 70])
def test_lengths_past_the_table(Lq):
    """Keys behind the table do not exist; the queries' positions stay."""
    rows, pages = table_of([64], 16)
    cache = filled(pages, 2, 16, 64, B16, 15)
    check_attention(heads(1, 2, Lq, 64, 8), cache, rows, [64 + Lq + 30], window=60 + Lq)
    check_attention(heads(1, 2, Lq, 64, 8), cache, rows, [2**31 - 1])


@pytest.mark.parametrize("Lq", [1, 70])
def test_no_pages_and_no_blocks(Lq):
    q = heads(2, 4, Lq, 64, 9)
    full, none = PagedCache.empty(3, 2, 16, 64), PagedCache.empty(0, 2, 16, 64)
    for cache, table in ((full, torch.zeros(2, 0, dtype=I32, device="cuda")), (none, i32([[0, 1], [2, 3]]))):
        assert bool((paged_attention(q, cache, table, i32([5, 9])) == 0).all())
    coded = PagedCache.empty(0, 2, 16, 64, dtype=F8)
    assert coded.values()[0].shape == (0, 2, 16, 64)
    k = q[:, :2]
    append_paged(none, k, k, i32([[0, 1], [2, 3]]), i32([5, 9]))
    append_paged(coded, k, k, i32([[0, 1], [2, 3]]), i32([5, 9]))
    assert paged_attention(q[:0], full, i32([[0]])[:0], i32([5])[:0]).shape == (0, 4, Lq, 64)
    assert paged_attention(q[:, :, :0], full, i32([[0], [1]]), i32([5, 4])).shape == (2, 4, 0, 64)
    append_paged(full, k[:, :, :0], k[:, :, :0], i32([[0], [1]]), i32([5, 4]))


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("Lq", [3, 70])
def test_strides(Lq, dtype):
    """A joint pool, head-major pools, a transposed and an expanded table, strided
    lengths and a query with strided channels."""
    lengths = [Lq + 30, 150]
    rows, pages = table_of(lengths, 16)
    cache = filled(pages, 2, 16, 64, dtype, 17)
    q = heads(2, 4, Lq, 64, 10)
    want = paged_attention(q, cache, i32(rows), i32(lengths))
    joint = torch.stack([cache.key.view(torch.uint8), cache.value.view(torch.uint8)], 1).view(dtype)
    e = (None, None) if dtype is B16 else torch.stack([cache.key_exponent, cache.value_exponent], 1).unbind(1)
    by_head = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (cache.key, cache.value)]
    for other in (PagedCache(joint[:, 0], joint[:, 1], *e),
                  PagedCache(*by_head, cache.key_exponent, cache.value_exponent)):
        assert torch.equal(paged_attention(q, other, i32(rows), i32(lengths)), want)
        if dtype is F8:
            assert all(torch.equal(a, b) for a, b in zip(other.values(), cache.values()))
    table = i32(rows).t().contiguous().t()
    assert torch.equal(paged_attention(q, cache, table, i32([lengths, lengths]).t()[:, 0]), want)
    strided = q.transpose(2, 3).contiguous().transpose(2, 3)
    got = paged_attention(strided, cache, i32(rows), i32(lengths))
    assert torch.equal(got, want) and got.stride() == torch.empty_like(strided).stride()
    shared = i32(rows[1]).expand(2, -1)
    assert torch.equal(paged_attention(q, cache, shared, i32([lengths[1]] * 2))[1], want[1])


def test_far_positions_of_a_long_cache():
    """A pool of more than 2^32 bytes a tensor: page offsets past 32 bits."""
    pages, H, page, D = 2**16 + 9, 8, 64, 128
    key, value = (torch.empty((pages, H, page, D), dtype=F8, device="cuda") for _ in range(2))
    e = torch.zeros((2, pages, H), dtype=torch.int8, device="cuda")
    cache = PagedCache(key, value, e[0], e[1])
    rows = [[pages - 1, 0, pages - 3], [pages - 2, 5, 2**15 + 1]]
    for p in set(sum(rows, [])):
        for pool in (key, value):
            pool[p] = normal((H, page, D), p % 1000).to(F8)
    q = heads(2, 16, 1, D, 12)
    got = paged_attention(q, cache, i32(rows), i32([150, 192]))
    names = sorted(set(sum(rows, [])))
    few = PagedCache(*(torch.stack([t[p].view(torch.uint8) for p in names]).view(F8) for t in (key, value)),
                     *(torch.zeros((len(names), H), dtype=torch.int8, device="cuda") for _ in range(2)))
    moved = [[names.index(p) for p in r] for r in rows]
    assert torch.equal(got, check_attention(q, few, moved, [150, 192]))
    k = heads(2, 8, 70, D, 13)
    append_paged(cache, k, k, i32(rows), i32([150, 192]))
    append_paged(few, k, k, i32(moved), i32([150, 192]))
    for a, b in ((cache.key, few.key), (cache.value, few.value)):
        assert all(torch.equal(a[p].view(torch.uint8), b[n].view(torch.uint8)) for n, p in enumerate(names))


def launched(name, call):
    """Whether `call` launches the kernel."""
    with _lib.LaunchTiming(64) as t:
        call()
        torch.cuda.synchronize()
        return t.read(name)[1] > 0


MANY = 300  # tokens that go over a copy of the pages, with 64 heads over one


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("options", [{}, {"window": 70}, {"window": 5}, {"cap": 15.0}, {"slopes": True},
                                     {"window": 130, "cap": 15.0, "slopes": True}], ids=str)
def test_many_rows_over_a_copy(options, D, dtype):
    """Sequences of different lengths, one without the call's tokens, one without
    any, padded rows, entries without a page and slots that hold anything."""
    lengths, counts = [MANY + 700, 1203, 310, 0], [MANY, 211, 0, 0]
    rows, pages = table_of(lengths, 32, seed=3)
    cache = filled(pages, 1, 32, D, dtype, 17)
    rows[1][3], rows[0][20] = -1, pages + 7
    for page, n in ((rows[0][1000 // 32], 1000), (rows[1][1203 // 32], 1203)):
        for pool in (cache.key, cache.value):
            pool[page, :, n % 32:].view(torch.uint8).fill_(0xFF)
    given = dict(options)
    if given.pop("slopes", False):
        given["slopes"] = torch.linspace(0.001, 0.2, 64, device="cuda")
    q = heads(4, 64, MANY, D, 3, 2.0)
    out = check_attention(q, cache, rows, lengths, counts, **given)
    assert not bool(out[1, :, 211:].any()) and not bool(out[2:].any())
    call = lambda: paged_attention(q, cache, i32(rows), i32(lengths), counts=i32(counts))  # noqa: E731
    assert launched("prep_paged", call)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("options", [{}, {"window": 700}, {"window": 30}, {"cap": 15.0}], ids=str)
def test_many_rows_split_over_their_keys(options, D):
    """A grid on half the CUs: parts of the keys, also parts without a key."""
    rows, pages = table_of([6000], 64, seed=4)
    cache = filled(pages, 1, 64, D, F8, 18)
    q = heads(1, 64, MANY, D, 4, 2.0)
    check_attention(q, cache, rows, [6000], **options)
    call = lambda: paged_attention(q, cache, i32(rows), i32([6000]), window=options.get("window"))  # noqa: E731
    if not options:
        assert launched("prep_paged", call) and launched("lse_merge", call)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("D", [64, 128])
def test_many_tiles_of_one_wave(D, dtype):
    """Enough sequences that each is one workgroup's: a wave passes several batches
    of 32 tiles.  They share their pages."""
    B, H = 64, 8
    lengths = [9000 - 131 * b for b in range(B)]
    rows, pages = table_of(lengths[:1], 16, seed=5)
    cache = filled(pages, H, 16, D, dtype, 19)
    check_attention(heads(B, H, 1, D, 5, 2.0), cache, rows * B, lengths)


def test_few_rows_are_read_in_place():
    rows, pages = table_of([900], 16)
    cache = filled(pages, 2, 16, 128, F8, 4)
    for Lq in (1, 40, 70):
        q = heads(1, 8, Lq, 128, 5)
        assert not launched("prep_paged", lambda: paged_attention(q, cache, i32(rows), i32([900])))


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------


def tables_of(lengths, counts, L, dims):
    positions = torch.tensor([[n - c + i for i in range(L)] for n, c in zip(lengths, counts)], device="cuda")
    return rope.build_position_tables(positions, rotary_dim=dims)


def check_append(cache, k, v, rows, lengths, counts=None, tables=None, layout="interleaved", start=0, query=None):
    keys, values = ref.Pool(cache.key, cache.key_exponent), ref.Pool(cache.value, cache.value_exponent)
    old = keys.values().clone()
    given = counts or [k.shape[2]] * k.shape[0]
    out = append_paged(cache, k, v, i32(rows), i32(lengths), counts=None if counts is None else i32(counts),
                       tables=tables, layout=layout, start=start, query=query)
    ref.append(values, v.cpu().double(), rows, lengths, given)
    got = ref.Pool(cache.value, cache.value_exponent)
    assert torch.equal(got.data.nan_to_num(1e30), values.data.nan_to_num(1e30))
    if got.exponent is not None:
        assert torch.equal(got.exponent, values.exponent)
    # Keys: what the kernel rotates in float32, product by product, is what is
    # rounded; next to a border of two codes, or of two exponents, the float64
    # rotation may lie on the other side.
    exact = k.cpu().double()
    rounded, turn = exact, torch.zeros_like(exact)
    if tables is not None:
        c, s = tables.cos.cpu(), tables.sin.cpu()
        exact = ref.rotate(k.cpu(), c, s, start, layout == "half")
        turn = 3 * UNIT * ref.rotate(k.cpu().abs(), c.abs(), -s.abs(), start, layout == "half").abs()
        turn = torch.maximum(turn, 3 * UNIT * exact.abs())
        turn = turn + 3 * UNIT * k.cpu().double().abs().amax()
        rounded = rope.rotate_heads(k.float(), tables, layout=layout, start=start).cpu().double()
        assert bool(((rounded - exact).abs() <= turn).all())
    if cache.key_exponent is None:
        rounded = rounded.to(B16).double()
    ref.append(keys, rounded, rows, lengths, given)
    got = ref.Pool(cache.key, cache.key_exponent)
    assert torch.equal(got.data.nan_to_num(1e30), keys.data.nan_to_num(1e30))
    if got.exponent is not None:
        assert torch.equal(got.exponent, keys.exponent)
    if tables is not None and query is not None:
        assert torch.equal(out, rope.rotate_heads(query, tables, layout=layout, start=start))
    return old


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("page", [16, 32, 256])
@pytest.mark.parametrize("Hkv, Hq", [(1, 1), (5, 9), (8, 30)])
def test_append_any_number_of_heads(Hkv, Hq, page, dtype):
    """Heads that a thread takes together, and what is left of them."""
    L, counts = 45, [45, 31]
    lengths = [45, 31 + 70]
    rows, pages = table_of(lengths, page)
    cache = filled(pages, Hkv, page, 64, dtype, page)
    k, v, q = heads(2, Hkv, L, 64, 50, 3.0), heads(2, Hkv, L, 64, 51), heads(2, Hq, L, 64, 52)
    check_append(cache, k, v, rows, lengths, counts, tables_of(lengths, counts, L, 64), "interleaved", 0, q)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_append_prompts(page, D, dtype):
    """Ragged prompts from any slot on, every page size."""
    L, counts = 150, [150, 149, 1, 0, 77]
    lengths = [150, 149 + 300, 1 + 15, 40, 77 + 100]
    rows, pages = table_of(lengths, page)
    cache = filled(pages, 3, page, D, dtype, page)
    k, v, q = heads(5, 3, L, D, 20, 3.0), heads(5, 3, L, D, 21), heads(5, 6, L, D, 22)
    check_append(cache, k, v, rows, lengths, counts, tables_of(lengths, counts, L, D), "half", 0, q)


@pytest.mark.parametrize("dtype", [B16, F8])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dims, start", [(64, 0), (32, 0), (32, 32), (16, 8), (8, 40), (6, 3), (2, 62), (10, 54)])
def test_append_rotations(dims, start, layout, dtype):
    """Part of a head; chunks and, for widths and starts that are no multiple of
    them, single channels."""
    lengths = [37, 20]
    rows, pages = table_of(lengths, 16)
    cache = filled(pages, 2, 16, 64, dtype, 3)
    k, v, q = heads(2, 2, 19, 64, 23), heads(2, 2, 19, 64, 24), heads(2, 4, 19, 64, 25)
    check_append(cache, k, v, rows, lengths, None, tables_of(lengths, [19, 19], 19, dims), layout, start, q)


@pytest.mark.parametrize("dtype", [B16, F8])
def test_append_without_rotation_and_shared_tables(dtype):
    lengths = [37, 20]
    rows, pages = table_of(lengths, 32)
    cache = filled(pages, 2, 32, 128, dtype, 4)
    k, v, q = heads(2, 2, 20, 128, 26), heads(2, 2, 20, 128, 27), heads(2, 4, 20, 128, 28)
    check_append(cache, k, v, rows, lengths)
    assert append_paged(cache, k, v, i32(rows), i32(lengths)) is None
    assert append_paged(cache, k, v, i32(rows), i32(lengths), query=q) is q
    t = rope.build_position_tables(torch.arange(20, device="cuda"), rotary_dim=128)
    check_append(cache, k, v, rows, lengths, None, RotaryTables(t.cos, t.sin), "half", 0, q)


@pytest.mark.parametrize("dtype", [B16, F8])
def test_token_by_token_raises_exponents(dtype):
    """Tokens of growing and falling magnitude in one page: the exponent never
    falls within it, and the earlier codes are moved."""
    page = 32
    rows, pages = table_of([70, 70], page)
    cache = filled(pages, 2, page, 64, dtype, 6)
    for n in range(1, 71):
        spread = 2.0 ** ((n * 7) % 23 - 12)
        k, v = heads(2, 2, 1, 64, 100 + n, spread), heads(2, 2, 1, 64, 200 + n, 1 / spread)
        check_append(cache, k, v, rows, [n, n], None, tables_of([n, n], [1, 1], 1, 64), "half")


def test_writing_again_changes_nothing():
    rows, pages = table_of([50], 16)
    cache = filled(pages, 2, 16, 64, F8, 8)
    k = heads(1, 2, 23, 64, 30)
    append_paged(cache, k, k, i32(rows), i32([50]))
    before = [t.clone() for t in (cache.key.view(torch.uint8), cache.key_exponent)]
    append_paged(cache, k, k, i32(rows), i32([50]))
    assert torch.equal(cache.key.view(torch.uint8), before[0]) and torch.equal(cache.key_exponent, before[1])


@pytest.mark.parametrize("dtype", [B16, F8])
def test_append_extremes(dtype):
    """Zeros, the smallest and largest numbers, infinities and NaN; a top value on
    the border of two exponents."""
    top = float(torch.finfo(B16).max)
    k = torch.zeros(1, 1, 48, 64, device="cuda")
    k[0, 0, 0, 0], k[0, 0, 1, 3], k[0, 0, 2, 5] = float("inf"), float("nan"), 5.0
    k[0, 0, 16, :3] = torch.tensor([448.0, -17.0, 2.0**-12])
    k[0, 0, 17] = 2.0**-133  # a subnormal
    k[0, 0, 32, 0], k[0, 0, 33, 1] = top, -top
    v = k.clone()
    v[0, 0, 16, 0] = 450.0
    v[0, 0, 32:] = 0.0
    v[0, 0, 40] = 2.0**-126
    rows, pages = table_of([48], 16)
    cache = filled(pages, 1, 16, 64, dtype, 10)
    check_append(cache, k.to(B16), v.to(B16), rows, [48])
    if dtype is F8:
        assert cache.key_exponent[rows[0][1], 0] == 0 and cache.value_exponent[rows[0][1], 0] == 1


@pytest.mark.parametrize("dtype", [B16, F8])
def test_tokens_without_a_page_are_left_out(dtype):
    lengths, counts = [60, 5, 100, 9], [40, 9, 30, -2]  # tokens before position 0, behind the table
    rows, pages = table_of([64, 64, 64, 64], 16)
    rows[0][2], rows[0][1] = -1, pages
    cache = filled(pages, 2, 16, 64, dtype, 12)
    k, v = heads(4, 2, 40, 64, 31), heads(4, 2, 40, 64, 32)
    check_append(cache, k, v, rows, lengths, counts)


@pytest.mark.parametrize("dtype", [B16, F8])
def test_append_strides(dtype):
    """Unaligned, gapped and shared rows; joint pools."""
    lengths = [37, 20]
    rows, pages = table_of(lengths, 16)
    t = tables_of(lengths, [19, 19], 19, 64)
    base = heads(2, 2, 19, 64, 33)
    odd = torch.zeros(2, 2, 19, 65, dtype=B16, device="cuda")
    odd[..., 1:] = base
    wide = torch.zeros(2, 2, 19, 128, dtype=B16, device="cuda")
    wide[..., ::2] = base
    for k in (base.contiguous(), odd[..., 1:], wide[..., ::2], base[:, :1].expand(2, 2, 19, 64)):
        cache = filled(pages, 2, 16, 64, dtype, 14)
        q = k.repeat(1, 2, 1, 1) if k is not odd else odd[..., 1:]
        check_append(cache, k, k, rows, lengths, None, t, "half", 0, q)
    joint = torch.zeros(pages, 2, 2, 16, 64, device="cuda").to(dtype)
    e = (None, None) if dtype is B16 else torch.zeros(pages, 2, 2, dtype=torch.int8, device="cuda").unbind(1)
    check_append(PagedCache(joint[:, 0], joint[:, 1], *e), base, base, rows, lengths, None, t, "half")


def test_no_gradient():
    cache = PagedCache.empty(4, 2, 16, 64)
    q = heads(1, 2, 3, 64, 34).requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        paged_attention(q, cache, i32([[0]]), i32([3]))
    with torch.no_grad():
        append_paged(cache, q, q, i32([[0]]), i32([3]))
        paged_attention(q, cache, i32([[0]]), i32([3]))
    seen = cache.key._version
    append_paged(cache, q.detach(), q.detach(), i32([[0]]), i32([3]))
    assert cache.key._version > seen


@pytest.mark.parametrize("page, D", [(16, 64), (32, 128), (256, 128)])
def test_values_of_every_code_and_exponent(page, D):
    """All 256 codes with all 256 exponents: bf16(code * 2**exponent), exact but for
    results below bf16's smallest normal number or past its largest."""
    pages, H = 129, 2
    cache = PagedCache.empty(pages, H, page, D, dtype=F8)
    codes = torch.arange(page * D, device="cuda", dtype=torch.int32).remainder(256).to(torch.uint8)
    for pool, shift in ((cache.key, 0), (cache.value, 7)):
        pool.view(torch.uint8).copy_(codes.roll(shift).view(page, D).expand(pages, H, page, D))
    e = (torch.arange(pages * H, device="cuda") % 256 - 128).to(torch.int8).view(pages, H)
    cache.key_exponent.copy_(e)
    cache.value_exponent.copy_(e.flip(0))
    for pool, ex, got in zip((cache.key, cache.value), (cache.key_exponent, cache.value_exponent), cache.values()):
        want = torch.ldexp(pool.double(), ex.double()[:, :, None, None]).to(torch.float32).to(B16)
        same = (got == want) | (got.isnan() & want.isnan())
        assert bool(same.all())
