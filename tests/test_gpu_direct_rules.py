"""The direct calls take no call that the registered ops refuse, give the ops' bits
for every call they take, and take those that are meant for them.  And what function
transforms make of the same operators."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import _lib, layers
from avgen_amd.cache import PagedCache, append_paged, paged_attention

pytestmark = pytest.mark.gpu

B16, F8, F32, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.int32
B, HQ, H, D, L, PAGE, PAGES = 2, 8, 2, 64, 3, 16, 9
NAN, INF = float("nan"), float("inf")


def normal(shape, seed, dtype=B16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def pool(dtype):
    p = dict(key_pages=normal((PAGES, H, PAGE, D), 1).to(dtype), value_pages=normal((PAGES, H, PAGE, D), 2).to(dtype))
    for n in ("key_exponent", "value_exponent"):
        p[n] = torch.zeros(PAGES, H, dtype=torch.int8, device="cuda") if dtype is F8 else None
    return p


def attend_args(dtype):
    p = pool(dtype)
    return dict(q=normal((B, HQ, L, D), 3), **p, block_table=ints([[0, 1, 2], [3, 4, 5]]), lengths=ints([40, 21]),
                counts=ints([3, 2]), slopes=normal((HQ,), 4, F32), window=0, scale=0.125, softcap=0.0)


def append_args(dtype):
    a = dict(k=normal((B, H, L, D), 5), v=normal((B, H, L, D), 6), query=normal((B, HQ, L, D), 7),
             cos=normal((1, 1, L, 16), 8, F32), sin=normal((1, 1, L, 16), 9, F32), start=8, half=True,
             block_table=ints([[0, 1, 2], [3, 4, 5]]), lengths=ints([40, 21]), counts=ints([3, 2]))
    return {**a, **pool(dtype)}


def norm_args(dtype):
    one = lambda n: normal((1, 1, 40), n, dtype)  # noqa: E731
    return dict(x=normal((B, L, 40), 10, dtype), residual=normal((B, L, 40), 11, dtype),
                weight=normal((40,), 12, dtype), post_weight=normal((40,), 13, dtype), gate=one(14), scale=one(15),
                shift=one(16), residual_scale=0.5, eps=1e-6)


def copied(args):
    """With tensors of its own, laid out the same."""
    out = {}
    for n, t in args.items():
        if torch.is_tensor(t) and t.numel() and t.untyped_storage().nbytes() < 1 << 20:
            whole = t.detach().as_strided((t.untyped_storage().nbytes() // t.element_size(),), (1,), 0).clone()
            t = whole.as_strided(t.shape, t.stride(), t.storage_offset()).requires_grad_(t.requires_grad)
        out[n] = t
    return out


def run(kind, args, direct):
    """The outputs and what was written (tensors), NotImplemented, or None if refused."""
    a = copied(args)
    calls, ops = _lib.direct_calls(normal((1,), 0)), torch.ops.avgen_amd
    order = list(a)
    if kind == "append" and direct:
        order = [n for n in order if n not in ("start", "half")] + ["start", "half"]
    given = [a[n] for n in order]
    fn = {"attend": (ops.paged_attention, calls.paged_attention), "append": (ops.append_paged, calls.append_paged),
          "norm": (ops.gated_add_rms_norm, calls.gated_add_rms_norm)}[kind][direct]
    try:
        out = fn(*given)
    except (ValueError, TypeError, RuntimeError):
        assert not direct, "a direct call refuses nothing"
        return None
    if out is NotImplemented:
        return out
    if kind == "attend":
        return [out if direct else out[0]]
    if kind == "norm":
        return list(out[:2])
    written = [a[n] for n in ("key_pages", "value_pages", "key_exponent", "value_exponent") if a[n] is not None]
    return ([out] if a["query"] is not None else []) + written


def bits(t):
    return t.detach().contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def other(t, at=1):
    """The same values `at` elements behind an aligned address."""
    flat = torch.empty(t.numel() + at, dtype=t.dtype, device="cuda")
    flat[at:].view(t.shape).copy_(t)
    return flat[at:].view(t.shape)


def gapped(t):
    wide = torch.zeros((*t.shape[:-1], 2 * t.shape[-1]), dtype=t.dtype, device="cuda")
    wide[..., ::2] = t
    return wide[..., ::2]


def joint(a):
    both = torch.stack([a["key_pages"].view(torch.uint8), a["value_pages"].view(torch.uint8)], 1)
    both = both.view(a["key_pages"].dtype)
    return dict(key_pages=both[:, 0], value_pages=both[:, 1])


def by_head(a):
    return {n: a[n].transpose(0, 1).contiguous().transpose(0, 1) for n in ("key_pages", "value_pages")}


# Name -> what changes; "take": the direct call is to take it, "leave": it leaves it to the
# op, which computes it, "refuse": the op refuses it.
POOLS = [
    ("take", "as it is", lambda a: {}),
    ("take", "joint", joint),
    ("take", "by head", by_head),
    ("take", "no counts", lambda a: dict(counts=None)),
    ("take", "one table for all", lambda a: dict(block_table=a["block_table"][:1].expand(B, -1))
     if "k" not in a else {}),
    ("take", "part of a table", lambda a: dict(block_table=torch.cat([a["block_table"]] * 2, 1)[:, :3])),
    ("leave", "a table by columns", lambda a: dict(block_table=a["block_table"].t().contiguous().t())),
    ("leave", "strided lengths", lambda a: dict(lengths=torch.stack([a["lengths"]] * 2, 1)[:, 0])),
    ("leave", "no blocks", lambda a: dict(block_table=a["block_table"][:, :0])),
    ("refuse", "pools of different sizes", lambda a: dict(value_pages=a["value_pages"][:5])),
    ("refuse", "pools of different types", lambda a: dict(value_pages=a["value_pages"].float())),
    ("refuse", "a page of 8", lambda a: {n: a[n][:, :, :8].contiguous() for n in ("key_pages", "value_pages")}),
    ("refuse", "half a head", lambda a: {n: a[n][..., :32].contiguous() for n in ("key_pages", "value_pages")}),
    ("refuse", "pages in one place", lambda a: {n: a[n][:1].expand(PAGES, H, PAGE, D) for n in ("key_pages",)}),
    ("refuse", "slots apart", lambda a: dict(key_pages=a["key_pages"].transpose(1, 2).contiguous().transpose(1, 2))),
    ("refuse", "channels apart", lambda a: dict(key_pages=gapped(a["key_pages"]))),
    ("refuse", "an unaligned pool", lambda a: dict(key_pages=other(a["key_pages"]))),
    ("refuse", "one exponent tensor", lambda a: dict(value_exponent=None)
     if a["key_exponent"] is not None else dict(value_exponent=torch.zeros(PAGES, H, dtype=torch.int8, device="cuda"))),
    ("refuse", "exponents of another type", lambda a: {n: torch.zeros(PAGES, H, dtype=I32, device="cuda")
                                                       for n in ("key_exponent", "value_exponent")}),
    ("refuse", "exponents of other sizes", lambda a: {n: torch.zeros(PAGES, H + 1, dtype=torch.int8, device="cuda")
                                                      for n in ("key_exponent", "value_exponent")}),
    ("refuse", "a table of another type", lambda a: dict(block_table=a["block_table"].long())),
    ("refuse", "a table of another batch", lambda a: dict(block_table=a["block_table"][:1])),
    ("refuse", "a flat table", lambda a: dict(block_table=a["block_table"][0])),
    ("refuse", "lengths of another type", lambda a: dict(lengths=a["lengths"].long())),
    ("refuse", "lengths of another batch", lambda a: dict(lengths=a["lengths"][:1])),
    ("refuse", "counts of another type", lambda a: dict(counts=a["counts"].long())),
    ("refuse", "counts of another batch", lambda a: dict(counts=a["counts"][:1])),
    ("refuse", "lengths on the CPU", lambda a: dict(lengths=a["lengths"].cpu())),
    ("refuse", "pages on the CPU", lambda a: dict(key_pages=a["key_pages"].cpu())),
]
ATTEND = [
    ("take", "a window", lambda a: dict(window=1 << 30)),
    ("take", "a cap", lambda a: dict(softcap=1024.0)),
    ("take", "no slopes", lambda a: dict(slopes=None)),
    ("take", "a projection's view", lambda a: dict(q=a["q"].transpose(1, 2).contiguous().transpose(1, 2))),
    ("leave", "a query of strided channels", lambda a: dict(q=gapped(a["q"]))),
    ("leave", "an unaligned query", lambda a: dict(q=other(a["q"]))),
    ("leave", "strided slopes", lambda a: dict(slopes=gapped(a["slopes"]))),
    ("leave", "no tokens", lambda a: dict(q=a["q"][:, :, :0])),
    ("refuse", "a window too large", lambda a: dict(window=(1 << 30) + 1)),
    ("refuse", "a negative window", lambda a: dict(window=-1)),
    *(("refuse", f"a scale of {s}", lambda a, s=s: dict(scale=s)) for s in (0.0, -1.0, NAN, INF, 1e-60, 1e60)),
    *(("refuse", f"a cap of {s}", lambda a, s=s: dict(softcap=s)) for s in (-1.0, 1025.0, NAN, INF, 1e-39)),
    ("refuse", "slopes of other sizes", lambda a: dict(slopes=a["slopes"][1:])),
    ("refuse", "slopes of another type", lambda a: dict(slopes=a["slopes"].double())),
    ("refuse", "a float32 query", lambda a: dict(q=a["q"].float())),
    ("refuse", "a query without a batch", lambda a: dict(q=a["q"][0])),
    ("refuse", "another head size", lambda a: dict(q=torch.cat([a["q"]] * 2, 3))),
    ("refuse", "heads that do not divide", lambda a: dict(q=a["q"][:, :7], slopes=None)),
    ("refuse", "too many heads with slopes", lambda a: dict(q=normal((B, 130, L, D), 3),
                                                               slopes=normal((130,), 4, F32))),
]
APPEND = [
    ("take", "no query", lambda a: dict(query=None)),
    ("take", "no rotation", lambda a: dict(cos=None, sin=None)),
    ("take", "tables of a batch", lambda a: {n: a[n].expand(B, -1, -1, -1).contiguous() for n in ("cos", "sin")}),
    ("take", "odd pairs", lambda a: {n: a[n][..., :3].contiguous() for n in ("cos", "sin")}),
    ("leave", "expanded tables", lambda a: {n: a[n].expand(B, -1, -1, -1) for n in ("cos", "sin")}),
    ("leave", "keys of strided channels", lambda a: dict(k=gapped(a["k"]))),
    ("leave", "unaligned values", lambda a: dict(v=other(a["v"]))),
    ("leave", "no tokens", lambda a: {**{n: a[n][:, :, :0] for n in ("k", "v", "query", "cos", "sin")}}),
    ("refuse", "one table", lambda a: dict(sin=None)),
    ("refuse", "tables of another length", lambda a: {n: a[n][:, :, :2].contiguous() for n in ("cos", "sin")}),
    ("refuse", "tables of heads", lambda a: {n: a[n].expand(-1, 2, -1, -1).contiguous() for n in ("cos", "sin")}),
    ("refuse", "tables of another batch", lambda a: {n: a[n].expand(3, -1, -1, -1).contiguous()
                                                     for n in ("cos", "sin")}),
    ("refuse", "tables of different sizes", lambda a: dict(sin=a["sin"][..., :8].contiguous())),
    ("refuse", "float64 tables", lambda a: {n: a[n].double() for n in ("cos", "sin")}),
    ("refuse", "no pairs", lambda a: {n: a[n][..., :0] for n in ("cos", "sin")}),
    ("refuse", "channels behind the head", lambda a: dict(start=33)),
    ("refuse", "channels in front of it", lambda a: dict(start=-1)),
    ("refuse", "float32 keys", lambda a: dict(k=a["k"].float())),
    ("refuse", "values of another length", lambda a: dict(v=a["v"][:, :, :2])),
    ("refuse", "other heads", lambda a: dict(k=a["query"], v=a["query"])),
    ("refuse", "a query of another length", lambda a: dict(query=a["query"][:, :, :2])),
    ("refuse", "a query of another type", lambda a: dict(query=a["query"].float())),
]
NORM = [
    ("take", "as it is", lambda a: {}),
    ("take", "nothing", lambda a: dict.fromkeys(("weight", "post_weight", "gate", "scale", "shift"))),
    ("take", "a row per sample", lambda a: {n: a[n].expand(B, 1, 40).contiguous() for n in ("gate", "scale", "shift")}),
    ("take", "one row for all samples", lambda a: {n: a[n].expand(B, 1, 40) for n in ("gate", "scale", "shift")}),
    ("take", "a row per token", lambda a: {n: a[n].expand(B, L, 40).contiguous() for n in ("gate", "scale", "shift")}),
    ("take", "float32 vectors", lambda a: {n: a[n].float()
                                           for n in ("weight", "post_weight", "gate", "scale", "shift")}),
    ("take", "unaligned rows", lambda a: dict(x=other(a["x"]))),
    ("take", "rows apart", lambda a: dict(x=torch.cat([a["x"]] * 2, 2)[..., :40])),
    ("take", "the same twice", lambda a: dict(residual=a["x"])),
    ("leave", "strided columns", lambda a: dict(x=gapped(a["x"]))),
    ("leave", "tokens first", lambda a: dict(residual=a["residual"].transpose(0, 1).contiguous().transpose(0, 1))),
    ("leave", "a strided gain", lambda a: dict(weight=gapped(a["weight"]))),
    ("leave", "no rows", lambda a: dict(x=a["x"][:, :0], residual=a["residual"][:, :0])),
    ("leave", "groups of other sizes", lambda a: {n: a[n].expand(3, 1, 40).reshape(3, 40).contiguous()
                                                  for n in ("gate", "scale", "shift")}),
    ("refuse", "a residual of another shape", lambda a: dict(residual=a["residual"][:1])),
    ("refuse", "float64 rows", lambda a: dict(x=a["x"].double(), residual=a["residual"].double())),
    ("refuse", "a residual of another type", lambda a: dict(residual=a["residual"].double())),
    ("refuse", "a gain of another width", lambda a: dict(weight=a["weight"][:39])),
    ("refuse", "a gain of another type", lambda a: dict(weight=a["weight"].half())),
    ("refuse", "a gain of more sizes", lambda a: dict(post_weight=a["gate"])),
    ("refuse", "a gate of another type", lambda a: dict(gate=a["gate"].half())),
    ("refuse", "a gate and a scale of two types", lambda a: dict(gate=a["gate"].double())),
    ("refuse", "a gate and a scale of two shapes", lambda a: dict(gate=a["gate"].expand(B, 1, 40).contiguous())),
    ("refuse", "rows that no groups divide", lambda a: {n: a[n].expand(4, 1, 40).contiguous()
                                                        for n in ("gate", "scale", "shift")}),
    ("refuse", "a gate of another width", lambda a: {n: a[n][..., :39].contiguous()
                                                     for n in ("gate", "scale", "shift")}),
    *(("refuse", f"eps {e}", lambda a, e=e: dict(eps=e)) for e in (-1.0, NAN, INF, 1e39)),
    *(("refuse", f"factor {e}", lambda a, e=e: dict(residual_scale=e)) for e in (NAN, INF, -1e39)),
    ("refuse", "a residual on the CPU", lambda a: dict(residual=a["residual"].cpu())),
]
CASES = ([("attend", d, *c) for d in (B16, F8) for c in POOLS + ATTEND]
         + [("append", d, *c) for d in (B16, F8) for c in POOLS + APPEND]
         + [("norm", d, *c) for d in (B16, F32) for c in NORM])


@pytest.mark.parametrize("kind, dtype, way, name, change", CASES,
                         ids=[f"{c[0]}-{str(c[1])[6:]}-{c[3].replace(' ', '_')}" for c in CASES])
def test_direct_calls_and_ops_agree(kind, dtype, way, name, change):
    args = {"attend": attend_args, "append": append_args, "norm": norm_args}[kind](dtype)
    args.update(change(args))
    with torch.no_grad():
        want, got = run(kind, args, False), run(kind, args, True)
    if way == "refuse":
        assert want is None and got is NotImplemented
        return
    assert want is not None
    if way == "leave":
        assert got is NotImplemented
        return
    assert got is not NotImplemented and len(got) == len(want)
    for a, b in zip(got, want):
        assert a.shape == b.shape and a.dtype is b.dtype and torch.equal(bits(a), bits(b))


# ---------------------------------------------------------------------------
# Function transforms
# ---------------------------------------------------------------------------


def test_vmap_of_the_norm_is_one_call_each():
    def step(x, r, w, g):
        return torch.cat(layers.gated_add_rms_norm(x, r, w, gate=g, post_weight=w), -1)

    many = [normal((3, *s), n, F32) for n, s in enumerate(((7, 40), (7, 40), (40,), (40,)))]
    got = torch.vmap(step)(*many)
    assert torch.equal(got, torch.stack([step(*(t[n] for t in many)) for n in range(3)]))


@pytest.mark.parametrize("dtype", [B16, F8])
def test_vmap_over_a_pool(dtype):
    """Attention is one call each; an append, which writes its pool, says that it is not."""
    a = attend_args(dtype)
    cache = PagedCache(a["key_pages"], a["value_pages"], a["key_exponent"], a["value_exponent"])
    q = normal((B, 1, HQ, L, D), 20)
    got = torch.vmap(lambda q, t, n: paged_attention(q, cache, t[None], n[None]))(q, a["block_table"], a["lengths"])
    for n in range(B):
        assert torch.equal(got[n], paged_attention(q[n], cache, a["block_table"][n:n + 1], a["lengths"][n:n + 1]))
    before = bits(cache.key).clone()
    k = normal((B, 1, H, L, D), 21)
    with pytest.raises(RuntimeError, match="[Bb]atching rule"):
        torch.vmap(lambda k, t, n: append_paged(cache, k, k, t[None], n[None], query=k))(k, a["block_table"],
                                                                                        a["lengths"])
    assert torch.equal(bits(cache.key), before)


def test_functional_and_forward_mode_gradients_say_that_they_are_not_there():
    x, r = normal((4, 40), 30, F32), normal((4, 40), 31, F32)
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.grad(lambda t: layers.gated_add_rms_norm(t, r)[0].sum())(x)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.clone().requires_grad_(True), r)
        with pytest.raises(NotImplementedError, match="jvp"):
            layers.gated_add_rms_norm(dual, r)
