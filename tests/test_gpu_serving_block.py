"""The paged cache and the gated norm together, as a model uses them: a block
with a gated, doubly normed residual served from pages, its training step, both
captured; and the direct calls beside the registered ops.

Tolerance of the bf16 serving block against the same block over whole sequences:
both pass the same roundings at other places; for each of the ~8 on the way
(residual sum, norm, projections, rotation, P, output) two half steps of the
largest value, 16 * 2^-8 = 6.25e-2.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from avgen_amd import _lib, attention, cache_ops, gated_ops, layers, rope
from avgen_amd.cache import PagedCache, append_paged, paged_attention

pytestmark = pytest.mark.gpu

B16, F8 = torch.bfloat16, torch.float8_e4m3fn
WIDTH, HQ, HKV, D, ROT, PAGE = 256, 4, 2, 64, 32, 16
VECTORS = ("weight", "post_weight", "gate", "scale", "shift")


def weights(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def w(o, i):
        return (torch.randn(o, i, generator=g, device="cuda") / math.sqrt(i)).to(B16)

    def gain():
        return (torch.rand(WIDTH, generator=g, device="cuda") + 0.5).to(B16)

    return dict(n1=gain(), n2=gain(), post=gain(), gate=gain(), wq=w(HQ * D, WIDTH), wk=w(HKV * D, WIDTH),
                wv=w(HKV * D, WIDTH), wo=w(WIDTH, HQ * D))


def project(w, n):
    return tuple(F.linear(n, w[name]).unflatten(-1, (-1, D)).transpose(1, 2) for name in ("wq", "wk", "wv"))


def block(w, x, r, attend):
    n, h = layers.gated_add_rms_norm(x, r, w["n1"])
    o = attend(*project(w, n))
    return layers.gated_add_rms_norm(F.linear(o.transpose(1, 2).flatten(2), w["wo"]), h, w["n2"], gate=w["gate"],
                                     post_weight=w["post"], residual_scale=0.5)


def whole(w, x, r):
    """The block over one whole sequence."""
    L = x.shape[1]
    tables = rope.build_position_tables(torch.arange(L, device="cuda"), rotary_dim=ROT)

    def attend(q, k, v):
        q, k = rope.rotate_query_key(q, k, tables, layout="half", start=D - ROT)
        lo, hi = attention.document_windows(torch.tensor([0, L], device="cuda"), L, causal=True)
        return attention.scored_attention(q, k, v, softcap=20.0, window_lo=lo, window_hi=hi, enable_gqa=True,
                                          monotone=True)

    return block(w, x, r, attend)


def serve(w, cache, table, lengths, x, r, counts=None):
    """The block for the newest tokens; ``lengths`` counts them."""
    L = x.shape[1]
    first = lengths - (L if counts is None else counts)
    tables = rope.build_position_tables((first[:, None] + torch.arange(L, device="cuda", dtype=torch.int32)),
                                        rotary_dim=ROT)

    def attend(q, k, v):
        q = append_paged(cache, k, v, table, lengths, counts=counts, tables=tables, layout="half", start=D - ROT,
                         query=q)
        return paged_attention(q, cache, table, lengths, counts=counts, softcap=20.0)

    return block(w, x, r, attend)


def pages(B, tokens, dtype):
    per = -(-tokens // PAGE)
    cache = PagedCache.empty(B * per + 1, HKV, PAGE, D, dtype=dtype)
    for pool in (cache.key, cache.value):
        pool.view(torch.uint8).fill_(0xFF)  # NaN in either type
    order = torch.randperm(B * per, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    return cache, order.view(B, per).cuda()


def test_serving_from_pages():
    """Prompts of different lengths in one padded call, a longer piece, then single
    and drafted tokens: the rows of the forward over each whole sequence."""
    w, total = weights(), 150
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn(3, total, WIDTH, generator=g, device="cuda").to(B16) for _ in range(2))
    cache, table = pages(3, total, B16)
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        want = [whole(w, x[b:b + 1], r[b:b + 1]) for b in range(3)]
        for counts in ([17, 1, 40], [70, 70, 70], [1, 1, 1], [5, 5, 5], [1, 0, 1]):
            L = max(counts)
            at = [int(n) for n in lengths]
            xs, rs = (torch.zeros(3, L, WIDTH, dtype=B16, device="cuda") for _ in range(2))
            for b, c in enumerate(counts):
                xs[b, :c], rs[b, :c] = x[b, at[b]:at[b] + c], r[b, at[b]:at[b] + c]
            new = torch.tensor(counts, dtype=torch.int32, device="cuda")
            lengths = lengths + new
            got = serve(w, cache, table, lengths, xs, rs, new)
            for b, c in enumerate(counts):
                for a, t in zip(got, want[b]):
                    ref = t[0, at[b]:at[b] + c]
                    if c:
                        err = (a[b, :c].double() - ref.double()).abs().max()
                        assert float(err) <= 6.25e-2 * float(t.abs().max()), (counts, b)


@pytest.mark.parametrize("dtype", [B16, F8])
def test_captured_decode_step(dtype):
    """A captured step serves every length: tables, lengths and pages are read when
    it runs."""
    w = weights(3)
    g = torch.Generator(device="cuda").manual_seed(4)
    cache, table = pages(4, 100, dtype)
    for pool in (cache.key, cache.value):  # numbers everywhere: lengths may skip slots
        pool.copy_(torch.randn(pool.shape, generator=g, device="cuda"))
    x, r = (torch.randn(4, 1, WIDTH, generator=g, device="cuda").to(B16) for _ in range(2))
    lengths = torch.tensor([1, 1, 1, 1], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            serve(w, cache, table, lengths, x, r)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = serve(w, cache, table, lengths, x, r)
        other = PagedCache(*(None if t is None else t.clone() for t in
                             (cache.key, cache.value, cache.key_exponent, cache.value_exponent)))
        for step in range(1, 50):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            lengths.copy_(torch.tensor([step, 2 * step, step, max(1, step - 3)], dtype=torch.int32))
            graph.replay()
            eager = serve(w, other, table, lengths, x, r)
            for a, b in zip(outs, eager):
                assert torch.equal(a, b), step
        for a, b in zip(cache.values(), other.values()):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def norm_inputs(dtype, seed=5, lead=(2, 37)):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    mod = rand(lead[0], 1, 3 * WIDTH).chunk(3, -1)
    return dict(x=rand(*lead, WIDTH), residual=rand(*lead, WIDTH), weight=rand(WIDTH), post_weight=rand(WIDTH),
                gate=mod[0], scale=mod[1], shift=mod[2]), rand(*lead, WIDTH), rand(*lead, WIDTH)


@pytest.mark.parametrize("dtype", [B16, torch.float32])
def test_captured_training_step(dtype):
    given, dn, dh = norm_inputs(dtype)
    leaves = {n: t.clone().requires_grad_(True) for n, t in given.items()}

    def step():
        n, h = layers.gated_add_rms_norm(**leaves)
        return (n.detach(), h.detach()) + torch.autograd.grad((n, h), list(leaves.values()), (dn, dh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        with torch.no_grad():
            for t in leaves.values():
                t.copy_(torch.randn_like(t))
        graph.replay()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b), k
        torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# Direct calls and ops
# ---------------------------------------------------------------------------


def attention_args(dtype, Lq=1):
    g = torch.Generator(device="cuda").manual_seed(6)
    cache, table = pages(2, 64, dtype)
    k, v = (torch.randn(2, HKV, 50, D, generator=g, device="cuda").to(B16) for _ in range(2))
    lengths = torch.tensor([50, 50], dtype=torch.int32, device="cuda")
    append_paged(cache, k, v, table, lengths)
    q = torch.randn(2, HQ, Lq, D, generator=g, device="cuda").to(B16)
    pool = (cache.key, cache.value, cache.key_exponent, cache.value_exponent)
    return cache, (q, *pool, table, lengths, None, None, 0, D**-0.5, 0.0)


@pytest.mark.parametrize("dtype", [B16, F8])
def test_paged_ops_and_direct_calls(dtype):
    """Ordinary calls are taken directly and give what the ops do; others go
    through the ops."""
    cache, args = attention_args(dtype)
    calls = _lib.direct_calls(args[0])
    assert calls is not None
    out, lse = torch.ops.avgen_amd.paged_attention(*args)
    assert torch.equal(calls.paged_attention(*args), out) and bool(lse.isfinite().all())
    assert calls.paged_attention(*args[:9], -1, *args[10:]) is NotImplemented
    assert calls.paged_attention(args[0][..., :32], *args[1:]) is NotImplemented
    assert calls.paged_attention(args[0].cpu(), *args[1:]) is NotImplemented
    assert calls.paged_attention(args[0], None, *args[2:]) is NotImplemented
    odd = torch.empty(2, HQ, 1, 2 * D, dtype=B16, device="cuda")[..., ::2].copy_(args[0])
    assert calls.paged_attention(odd, *args[1:]) is NotImplemented
    assert torch.equal(paged_attention(odd, cache, *args[5:7]), out)

    g = torch.Generator(device="cuda").manual_seed(7)
    k = torch.randn(2, HKV, 3, D, generator=g, device="cuda").to(B16)
    q = torch.randn(2, HQ, 3, D, generator=g, device="cuda").to(B16)
    tables = rope.build_position_tables(torch.arange(3, device="cuda"), rotary_dim=ROT)
    results = []
    for call in ("direct", "op"):
        cache, a = attention_args(dtype)
        pool, version = a[1:5], cache.key._version
        lengths = a[6] + 3
        if call == "direct":
            out = calls.append_paged(k, k, q, tables.cos, tables.sin, a[5], lengths, None, *pool, 0, True)
            assert calls.append_paged(k, k, None, None, None, a[5], lengths, None, *pool, 0, True) is None
        else:
            out = torch.ops.avgen_amd.append_paged(k, k, q, tables.cos, tables.sin, 0, True, a[5], lengths, None, *pool)
            torch.ops.avgen_amd.append_paged(k, k, None, None, None, 0, True, a[5], lengths, None, *pool)
        assert cache.key._version > version
        results.append((out, *cache.values()))
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    if dtype is F8:
        for a, b in zip(torch.ops.avgen_amd.page_values(*pool), calls.page_values(*pool)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    with torch.inference_mode():
        assert torch.equal(calls.paged_attention(*args), torch.ops.avgen_amd.paged_attention(*args)[0])
    side = torch.cuda.Stream()
    want = torch.ops.avgen_amd.paged_attention(*args)[0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls.paged_attention(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("drop", [(), ("gate",), ("scale", "shift"), ("post_weight", "gate"), ("weight",)])
def test_norm_op_and_direct_call(drop):
    given, dn, dh = norm_inputs(torch.float32)
    given.update(dict.fromkeys(drop))
    leaves = {n: t if t is None else t.clone().requires_grad_(True) for n, t in given.items()}
    kept = [t for t in leaves.values() if t is not None]
    args = tuple(leaves[n] for n in ("x", "residual", *VECTORS)) + (0.5, 1e-6)
    calls = _lib.direct_calls(args[0])
    results = []
    for fn in (calls.gated_add_rms_norm, lambda *a: torch.ops.avgen_amd.gated_add_rms_norm(*a)[:2]):
        n, h = fn(*args)
        results.append((n, h, *torch.autograd.grad((n, h), kept, (dn, dh))))
        with torch.no_grad():
            for a, b in zip(fn(*args), (n, h)):
                assert torch.equal(a, b) and not a.requires_grad
    for a, b in zip(*results):
        assert torch.equal(a, b) and a.shape == b.shape
    # A second derivative is refused whichever way.
    n, h = calls.gated_add_rms_norm(*args)
    dx, = torch.autograd.grad((n, h), args[:1], (dn, dh), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.sum(), args[:1])
    # A saved tensor that changed is noticed.
    n, h = calls.gated_add_rms_norm(*args)
    with torch.no_grad():
        args[0].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad((n, h), kept, (dn, dh))


def test_norm_calls_that_are_not_direct():
    given, dn, dh = norm_inputs(torch.float32)
    args = tuple(given[n] for n in ("x", "residual", *VECTORS)) + (1.0, 1e-6)
    calls = _lib.direct_calls(args[0])
    want = calls.gated_add_rms_norm(*args)
    for bad in ((args[0].double(), *args[1:]), (args[0], args[1][:1], *args[2:]), (*args[:8], -1.0),
                (*args[:8], float("nan")), (*args[:4], args[4][:1], *args[5:]), (None, *args[1:]),
                (*args[:2], args[2][1:], *args[3:])):
        assert calls.gated_add_rms_norm(*bad) is NotImplemented
    turned = args[0].transpose(0, 1).contiguous().transpose(0, 1)
    assert calls.gated_add_rms_norm(turned, *args[1:]) is NotImplemented
    for a, b in zip(gated_ops.gated_add_rms_norm(turned, *args[1:]), want):
        assert torch.equal(a, b)
    # The gradients' layouts do not matter, nor that one is missing.
    x = args[0].clone().requires_grad_(True)
    n, h = calls.gated_add_rms_norm(x, *args[1:])
    a = torch.autograd.grad((n, h), x, (dn, dh), retain_graph=True)[0]
    b = torch.autograd.grad((n, h), x, tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (dn, dh)),
                            retain_graph=True)[0]
    assert torch.equal(a, b)
    a = torch.autograd.grad(h, x, dh, retain_graph=True)[0]
    b = torch.autograd.grad((n, h), x, (torch.zeros_like(dn), dh))[0]
    assert torch.equal(a, b)


def test_ops_pass_opcheck_and_compile():
    given, _, _ = norm_inputs(torch.float32, lead=(2, 5))
    leaves = [given[n].detach().requires_grad_(True) for n in ("x", "residual", *VECTORS)]
    torch.library.opcheck(gated_ops._op, (*leaves, 0.5, 1e-6))
    fn = torch.compile(lambda a, b, c: layers.gated_add_rms_norm(a, b, c, gate=leaves[4]), fullgraph=True)
    for a, b in zip(fn(*leaves[:3]), layers.gated_add_rms_norm(*leaves[:3], gate=leaves[4])):
        assert torch.equal(a, b)
    for dtype in (B16, F8):
        cache, args = attention_args(dtype)
        # (The schema's test computes with the inputs, which torch cannot in e4m3.)
        which = "ALL" if dtype is B16 else ("test_faketensor", "test_autograd_registration")
        torch.library.opcheck(cache_ops._attention_op, args, test_utils=which)
        k = torch.randn(2, HKV, 3, D, device="cuda").to(B16)
        # (It compares whole pools: no NaN there.)
        for pool in (cache.key, cache.value):
            pool.view(torch.uint8).zero_()
        torch.library.opcheck(cache_ops._append_op,
                              (k, k, k, None, None, 0, True, args[5], args[6] + 3, None, *args[1:5]), test_utils=which)
        if dtype is F8:
            torch.library.opcheck(cache_ops._values_op, args[1:5], test_utils=which)
