"""Performance cases of the paged key/value cache and of the gated residual norm.

Each case is one pass through an operator as a serving or training program
calls it.  ``listed()`` names a fixed set, ``draw(rng)`` gives further cases of
the same ranges; ``prepare`` makes a case's inputs, ``run`` computes it (with
``own`` through the package, otherwise with elementary torch operations in
float32), ``exact`` computes the same outputs in float64 and ``work`` counts
the bytes and operations the case cannot do without.

Kinds (``case["kind"]``):

* ``attend`` paged_attention: the last ``Lq`` tokens of every sequence against
  the pages that hold its tokens, these included;
* ``append`` append_paged: the keys and values of ``L`` new tokens of every
  sequence are rotated and written to their pages, the query rotated with them;
* ``norm``   gated_add_rms_norm, forward only or forward and backward.

A cache is a pool of pages; a page holds ``page`` consecutive tokens of one
sequence, in bfloat16 or as e4m3 codes with one exponent per page and head (a
value is ``code * 2**exponent``).  ``lengths`` counts a sequence's tokens, the
new ones included; of a batch padded to ``L`` tokens, ``counts`` are new.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
E4M3 = torch.float8_e4m3fn


def listed():
    """The fixed cases."""
    return [
        # The first tokens of one chat on a small model: latency alone.
        dict(name="attend_token_small", kind="attend", pages="e4m3", B=1, H=8, Hkv=2, D=64, Lq=1, page=16, room=64,
             length=33, spread=0, window=0, cap=0.0, slopes=False),
        # A decode step of 8 sequences, the cache three quarters full.
        dict(name="attend_token", kind="attend", pages="e4m3", B=8, H=32, Hkv=8, D=128, Lq=1, page=64, room=8192,
             length=6200, spread=37, window=0, cap=0.0, slopes=False),
        # Four drafted tokens of one long sequence.
        dict(name="attend_draft_long", kind="attend", pages="e4m3", B=1, H=16, Hkv=4, D=128, Lq=4, page=32,
             room=100000, length=99991, spread=0, window=0, cap=50.0, slopes=False),
        # A decode step of 16 sequences of very different lengths, small
        # bfloat16 pages.
        dict(name="attend_ragged_bf16", kind="attend", pages="bfloat16", B=16, H=32, Hkv=8, D=128, Lq=1, page=16,
             room=16384, length=16001, spread=999, window=0, cap=0.0, slopes=False),
        # A layer with a sliding window, 32 long sequences.
        dict(name="attend_window", kind="attend", pages="e4m3", B=32, H=16, Hkv=8, D=128, Lq=1, page=64, room=16384,
             length=16000, spread=101, window=4096, cap=0.0, slopes=False),
        # A piece of two prompts read behind what is cached.
        dict(name="attend_chunk", kind="attend", pages="e4m3", B=2, H=32, Hkv=8, D=128, Lq=512, page=64, room=12288,
             length=12001, spread=700, window=0, cap=0.0, slopes=False),
        # One decoded token of each of 16 sequences.
        dict(name="append_token", kind="append", pages="e4m3", B=16, H=32, Hkv=8, D=128, L=1, page=64, before=100,
             spread=3, ragged=0, dims=128, start=0, layout="half"),
        # Two whole prompts of different lengths, padded, into bfloat16 pages.
        dict(name="append_prompt_bf16", kind="append", pages="bfloat16", B=2, H=32, Hkv=32, D=128, L=8192, page=16,
             before=0, spread=0, ragged=1100, dims=128, start=0, layout="interleaved"),
        # The next piece of four prompts, ending and beginning inside pages.
        dict(name="append_prompt_e4m3", kind="append", pages="e4m3", B=4, H=32, Hkv=8, D=128, L=4133, page=32,
             before=1001, spread=13, ragged=7, dims=64, start=0, layout="half"),
        # The step between two sections of a block, one token of 8 samples.
        dict(name="norm_token", kind="norm", dtype="bfloat16", B=8, L=1, W=5120, modulation="batch", post=False,
             gain=True, alpha=1.0, grad=False),
        # The same in training, modulated by each sample's time embedding.
        dict(name="norm_train", kind="norm", dtype="bfloat16", B=2, L=9450, W=5120, modulation="batch", post=False,
             gain=True, alpha=1.0, grad=True),
        # Norms on both sides and a learned gate, float32 in training.
        dict(name="norm_post_f32", kind="norm", dtype="float32", B=1, L=4133, W=2560, modulation="gate", post=True,
             gain=True, alpha=0.5, grad=True),
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges ``listed()`` stands for."""
    kind = rng.choice(["attend", "attend", "attend", "append", "append", "norm", "norm"])
    if kind == "norm":
        W = rng.choice([_log(rng, 1, 16384), 8 * _log(rng, 1, 2048)])
        B = rng.choice([1, 2, 3, 8])
        modulation = rng.choice(["none", "gate", "batch", "batch", "token"])
        L = _log(rng, 1, max(1, min(20000, (20_000_000 if modulation == "token" else 45_000_000) // (W * B))))
        return dict(kind=kind, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), B=B, L=L, W=W,
                    modulation=modulation, post=rng.choice([False, True]),
                    gain=rng.choice([True, True, False]), alpha=rng.choice([1.0, 0.5]),
                    grad=rng.choice([False, True]))
    pages = rng.choice(["e4m3", "e4m3", "bfloat16"])
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        B = rng.choice([1, 2, 4, 16])
        L = rng.choice([1, _log(rng, 1, max(1, 4096 * 64 // (B * (H + Hkv))))])
        dims = rng.choice([D, D // 2])
        return dict(kind=kind, pages=pages, B=B, H=H, Hkv=Hkv, D=D, L=L, page=page, before=_log(rng, 1, 3000) - 1,
                    spread=rng.randint(0, 50), ragged=rng.randint(0, max(0, (L - 1) // B)), dims=dims,
                    start=rng.choice([0, D - dims]), layout=rng.choice(["half", "interleaved"]))
    score = rng.choice(["", "", "cap", "slopes", "both"])
    if rng.random() < 0.7:
        B = rng.choice([1, 2, 5, 8, 16, 40])
        Lq = rng.choice([1, 1, 1, 2, 4, 7])
        length = _log(rng, max(Lq, 16), 120000 // B)
    else:
        B = rng.choice([1, 2])
        Lq = _log(rng, 8, 512)
        length = _log(rng, Lq, 384000 // max(32, H * B))
    room = -(-rng.randint(length, length + length // 2) // page) * page
    return dict(kind=kind, pages=pages, B=B, H=H, Hkv=Hkv, D=D, Lq=Lq, page=page, room=room, length=length,
                spread=rng.randint(0, max(0, (length - Lq) // B)),
                window=rng.choice([0, 0, _log(rng, 1, length)]),
                cap=rng.choice([20.0, 50.0]) if score in ("cap", "both") else 0.0, slopes=score in ("slopes", "both"))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _heads(gen, B, L, H, D, dtype, spread=1.0):
    """(B, H, L, D) as the view of a (B, L, H*D) projection."""
    x = torch.randn((B, L, H * D), generator=gen, device="cuda") * spread
    return x.to(dtype).unflatten(-1, (H, D)).transpose(1, 2)


def _lengths(case):
    """A sequence's tokens and how many of them are new, as lists."""
    B = case["B"]
    if case["kind"] == "attend":
        return [case["length"] - b * case["spread"] for b in range(B)], [case["Lq"]] * B
    new = [case["L"] - b * case["ragged"] for b in range(B)]
    return [case["before"] + b * case["spread"] + n for b, n in enumerate(new)], new


def _pool(gen, case):
    """The block table (B, pages of a sequence), its pages in any order, and
    how many pages there are (one more than the table names)."""
    lengths, _ = _lengths(case)
    room = case.get("room") or max(lengths)
    per = -(-room // case["page"])
    order = torch.randperm(case["B"] * per, generator=gen, device="cuda").to(torch.int32)
    return order.view(case["B"], per).contiguous(), case["B"] * per + 1


def prepare(case, seed):
    """The inputs a program holds before the call, from ``seed``."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 23)
    st = dict(case=case)
    if case["kind"] == "norm":
        _prepare_norm(st, gen)
        return st
    B, H, Hkv, D, page = (case[n] for n in ("B", "H", "Hkv", "D", "page"))
    st["table"], pages = _pool(gen, case)
    lengths, new = _lengths(case)
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    st["counts"] = torch.tensor(new, dtype=torch.int32, device="cuda")
    # What the cache holds: keys with a few large channels, as after a norm
    # with a gain.
    gain = torch.ones(D, device="cuda")
    gain[::16] = 4.0
    for name in ("key", "value"):
        x = torch.randn((pages, Hkv, page, D), generator=gen, device="cuda")
        if name == "key":
            x *= gain
        if case["pages"] == "e4m3":
            e = torch.ceil(torch.log2(x.abs().amax((-1, -2)) / 448.0))
            st[name] = (x * torch.exp2(-e)[..., None, None]).to(E4M3)
            st[name + "_exponent"] = e.to(torch.int8)
        else:
            st[name] = x.to(torch.bfloat16)
            st[name + "_exponent"] = None
        del x
    if own:
        from avgen_amd.cache import PagedCache

        st["cache"] = PagedCache(st["key"], st["value"], st["key_exponent"], st["value_exponent"])
    if case["kind"] == "attend":
        st["q"] = _heads(gen, B, case["Lq"], H, D, torch.bfloat16, 2.0)
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32,
                                    device="cuda") if case["slopes"] else None
        return st
    L = case["L"]
    st["q"] = _heads(gen, B, L, H, D, torch.bfloat16)
    st["k"] = _heads(gen, B, L, Hkv, D, torch.bfloat16, 1.5)
    st["v"] = _heads(gen, B, L, Hkv, D, torch.bfloat16)
    f = torch.tensor([10000.0 ** (-2.0 * i / case["dims"]) for i in range(case["dims"] // 2)], device="cuda",
                     dtype=torch.float64)
    positions = (st["lengths"] - st["counts"]).long()[:, None] + torch.arange(L, device="cuda")
    angle = positions[:, None, :, None].double() * f
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    if own:
        from avgen_amd.rope import RotaryTables

        st["tables"] = RotaryTables(cos=st["cos"], sin=st["sin"])
    return st


def _prepare_norm(st, gen):
    case = st["case"]
    B, L, W = case["B"], case["L"], case["W"]
    dtype = DTYPES[case["dtype"]]

    def rand(shape, spread, middle=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * spread + middle).to(dtype)

    st["x"], st["r"] = rand((B, L, W), 1.0), rand((B, L, W), 3.0)
    st["w"] = rand((W,), 0.2, 1.0) if case["gain"] else None
    st["p"] = rand((W,), 0.2, 1.0) if case["post"] else None
    st["gate"] = st["scale"] = st["shift"] = None
    if case["modulation"] == "gate":
        st["gate"] = rand((W,), 0.3, 0.5)
    elif case["modulation"] != "none":
        # Three pieces of one projection of the time embedding.
        rows = 1 if case["modulation"] == "batch" else L
        st["gate"], st["scale"], st["shift"] = rand((B, rows, 3 * W), 0.3).chunk(3, -1)
    if case["grad"]:
        st["dn"], st["dh"] = rand((B, L, W), 1.0), rand((B, L, W), 1.0)
        for name in NORM_INPUTS:
            if st[name] is not None:
                st[name] = st[name].detach().requires_grad_(True)


NORM_INPUTS = ("x", "r", "w", "gate", "scale", "shift", "p")


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _held(codes, exponent):
    """What pages of the cache hold, in float32."""
    x = codes.float()
    return x if exponent is None else x * torch.exp2(exponent.float())[..., None, None]


def _attend(st):
    case = st["case"]
    q = st["q"].float()
    B, H, Lq, D = q.shape
    Hkv, page = case["Hkv"], case["page"]
    used = -(-case["length"] // page)  # no sequence is longer
    table = st["table"][:, :used].long()
    k, v = (_held(st[n][table], None if st[n + "_exponent"] is None else st[n + "_exponent"][table])
            .transpose(1, 2).flatten(2, 3) for n in ("key", "value"))
    s = (q.reshape(B, Hkv, H // Hkv * Lq, D) @ k.transpose(-1, -2).contiguous()).view(B, H, Lq, -1) / math.sqrt(D)
    if case["cap"] > 0:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    j = torch.arange(used * page, device="cuda")
    at = ((st["lengths"] - st["counts"])[:, None] + torch.arange(Lq, device="cuda"))[:, None, :, None]
    if st["slopes"] is not None:
        s = s - st["slopes"][:, None, None] * (at - j).abs().float()
    allowed = (j <= at) & (j > at - case["window"]) if case["window"] else j <= at
    s = s.masked_fill(~allowed, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    # A masked slot may hold anything; here every page holds numbers.
    out = (p.view(B, Hkv, H // Hkv * Lq, -1) @ v).view(B, H, Lq, D)
    return (out / p.sum(-1, keepdim=True)).to(torch.bfloat16)


def _rotate(x, cos, sin, case):
    d, start = case["dims"], case["start"]
    y = x[..., start:start + d]
    if case["layout"] == "half":
        a, b = y[..., :d // 2], y[..., d // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = y[..., 0::2], y[..., 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([x[..., :start], r, x[..., start + d:]], -1)


def _e4m3(y):
    """The nearest e4m3 values of ``|y| <= 448``, ties to even."""
    a = y.abs().clamp(min=2.0 ** -6)
    e = torch.floor(torch.log2(a))
    # floor(log2) may land one off next to a power of two.
    e = torch.where(torch.exp2(e) > a, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= a, e + 1, e)
    step = torch.exp2(e - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exponent(top):
    """The least exponent with ``448 * 2**e >= top``, from -110 on."""
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -120) / 448.0))
    e = torch.where(448.0 * torch.exp2(e) < top, e + 1, e)
    e = torch.where(448.0 * torch.exp2(e - 1) >= top, e - 1, e)
    return e.clamp(-110, 119)


def _append(st):
    case = st["case"]
    B, Hkv, D, L, page = (case[n] for n in ("B", "Hkv", "D", "L", "page"))
    q = _rotate(st["q"].float(), st["cos"], st["sin"], case).to(torch.bfloat16)
    blocks = (L - 1) // page + 2  # that L tokens may touch
    first = (st["lengths"] - st["counts"]).long()
    i = torch.arange(L, device="cuda")
    # Slots of the touched blocks; tokens behind a sequence's count go to one
    # behind the last.
    slot = torch.where(i < st["counts"][:, None], first[:, None] % page + i, blocks * page)
    b = torch.arange(blocks, device="cuda")
    touched = b <= (first[:, None] % page + st["counts"][:, None] - 1) // page
    at = (first[:, None] // page + b).clamp(max=st["table"].shape[1] - 1)
    spare = st["key"].shape[0] - 1
    pages = torch.where(touched, st["table"].long().gather(1, at), spare)
    index = slot[:, None, :, None].expand(B, Hkv, L, D)
    fresh = torch.zeros((B, blocks * page + 1), dtype=torch.bool, device="cuda").scatter(1, slot, True)
    fresh = fresh[:, :-1].view(B, blocks, 1, page, 1)
    before = (b * page < first[:, None] % page)[:, :, None]
    for name, x in (("key", _rotate(st["k"].float(), st["cos"], st["sin"], case)), ("value", st["v"].float())):
        frame = torch.zeros((B, Hkv, blocks * page + 1, D), device="cuda").scatter(2, index, x)
        frame = frame[:, :, :-1].view(B, Hkv, blocks, page, D).transpose(1, 2)
        old, exponent = st[name][pages].float(), st[name + "_exponent"]
        if exponent is not None:
            e0 = exponent[pages].float()
            e = _exponent(frame.abs().amax((-1, -2)))
            e = torch.where(before, torch.maximum(e, e0), e)
            frame = _e4m3(frame * torch.exp2(-e)[..., None, None])
            # Codes of the block's earlier tokens; where the exponent stays,
            # and behind the new tokens, as they are.
            kept = _e4m3(old * torch.exp2((e0 - e).clamp(max=0.0))[..., None, None])
            old = torch.where(before[..., None, None], kept, old)
            exponent[pages] = torch.where(touched[..., None], e, e0).to(torch.int8)
        st[name][pages] = torch.where(fresh, frame, old).to(st[name].dtype)
    return q, *_pages(st)


def _pages(st):
    """The pages that sequences own, as the values they stand for."""
    if st["key_exponent"] is None:
        return st["key"][:-1], st["value"][:-1]
    return tuple(_held(st[n][:-1], st[n + "_exponent"][:-1]).to(torch.bfloat16) for n in ("key", "value"))


def _norm(x, r, w, gate, scale, shift, p, alpha):
    if p is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * p
    if gate is not None:
        x = x * gate
    h = alpha * r + x
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-6)
    if w is not None:
        n = n * w
    if scale is not None:
        n = n * (1 + scale) + shift
    return n, h


def _gradients(st, n, h):
    inputs = [st[name] for name in NORM_INPUTS if st[name] is not None]
    return (n, h) + torch.autograd.grad((n, h), inputs, (st["dn"], st["dh"]))


def _run_own(st):
    case = st["case"]
    if case["kind"] == "norm":
        from avgen_amd.layers import gated_add_rms_norm

        n, h = gated_add_rms_norm(st["x"], st["r"], st["w"], gate=st["gate"], scale=st["scale"], shift=st["shift"],
                                  post_weight=st["p"], residual_scale=case["alpha"])
        return _gradients(st, n, h) if case["grad"] else (n, h)
    from avgen_amd.cache import append_paged, paged_attention

    if case["kind"] == "attend":
        return paged_attention(st["q"], st["cache"], st["table"], st["lengths"], window=case["window"] or None,
                               softcap=case["cap"] or None, distance_slopes=st["slopes"])
    q = append_paged(st["cache"], st["k"], st["v"], st["table"], st["lengths"], counts=st["counts"],
                     tables=st["tables"], layout=case["layout"], start=case["start"], query=st["q"])
    if st["key_exponent"] is None:
        return q, st["key"][:-1], st["value"][:-1]
    key, value = st["cache"].values()
    return q, key[:-1], value[:-1]


def run(st):
    """One pass, as a program calls it."""
    if own:
        return _run_own(st)
    case = st["case"]
    if case["kind"] == "attend":
        return _attend(st)
    if case["kind"] == "append":
        return _append(st)
    dtype = DTYPES[case["dtype"]]
    n, h = _norm(*(None if st[name] is None else st[name].float() for name in NORM_INPUTS), case["alpha"])
    n, h = n.to(dtype), h.to(dtype)
    return _gradients(st, n, h) if case["grad"] else (n, h)


# ---------------------------------------------------------------------------
# Float64
# ---------------------------------------------------------------------------


def _sequence(st, name, b, h, n):
    """The first n tokens of one head of one sequence, in float64."""
    pages = st["table"][b, :-(-n // st["case"]["page"])].long()
    x = st[name][pages, h].double()
    if st[name + "_exponent"] is not None:
        x = torch.ldexp(x, st[name + "_exponent"][pages, h].double()[:, None, None])
    return x.flatten(0, 1)[:n]


def _exact_attend(st):
    case = st["case"]
    B, H, Lq, D = st["q"].shape
    lengths, _ = _lengths(case)
    out = torch.empty((B, H, Lq, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        j = torch.arange(n, device="cuda")
        i = torch.arange(n - Lq, n, device="cuda")
        for h in range(H):
            hk = h * case["Hkv"] // H
            z = st["q"][b, h].double() @ _sequence(st, "key", b, hk, n).T.contiguous() * D ** -0.5
            if case["cap"] > 0:
                z = case["cap"] * torch.tanh(z / case["cap"])
            distance = i[:, None] - j
            if st["slopes"] is not None:
                z = z - st["slopes"][h].double() * distance.abs()
            z[distance < 0] = float("-inf")
            if case["window"]:
                z[distance >= case["window"]] = float("-inf")
            out[b, h] = torch.softmax(z, -1) @ _sequence(st, "value", b, hk, n)
    return out


def _turned(x, cos, sin, case):
    """The rotation as complex numbers."""
    d, start = case["dims"], case["start"]
    y = x[..., start:start + d].double()
    pairs = y.unflatten(-1, (2, d // 2)).transpose(-1, -2) if case["layout"] == "half" else y.unflatten(-1, (d // 2, 2))
    z = torch.view_as_complex(pairs.contiguous()) * torch.complex(cos, sin)
    pairs = torch.view_as_real(z)
    out = x.double().clone()
    out[..., start:start + d] = (pairs.transpose(-1, -2) if case["layout"] == "half" else pairs).flatten(-2)
    return out


def _nearest_e4m3(y):
    """By the list of all e4m3 magnitudes: the nearest, the even code on ties."""
    grid = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    grid = torch.tensor(grid[:127], dtype=torch.float64, device=y.device)
    up = torch.searchsorted(grid, y.abs().contiguous()).clamp(max=126)
    down = (up - 1).clamp(min=0)
    above, below = grid[up] - y.abs(), y.abs() - grid[down]
    pick = torch.where((below < above) | ((below == above) & (down % 2 == 0)), down, up)
    return torch.sign(y) * grid[pick]


def _exact_append(st):
    case = st["case"]
    cos, sin = st["cos"].double(), st["sin"].double()
    q, k = (_turned(st[n], cos, sin, case) for n in ("q", "k"))
    lengths, new = _lengths(case)
    page, coded = case["page"], case["pages"] == "e4m3"
    pools = []
    for name, x in (("key", k), ("value", st["v"].double())):
        pool = st[name].double()
        e = None
        if coded:
            e = st[name + "_exponent"].double()
            pool = torch.ldexp(pool, e[:, :, None, None])
        for b, (n, m) in enumerate(zip(lengths, new)):
            table = st["table"][b].tolist()
            for block in range((n - m) // page, -(-n // page)):
                lo, hi = max(n - m, block * page), min(n, (block + 1) * page)
                y = x[b, :, lo - n + m:hi - n + m]
                at = table[block]
                if coded:
                    _, need = torch.frexp(y.abs().amax((-1, -2)) / 448.0)
                    need = need.double()
                    # frexp gives 2^e > top / 448; equality wants one less.
                    need = torch.where(y.abs().amax((-1, -2)) <= 448.0 * torch.exp2(need - 1), need - 1, need)
                    need = need.clamp(-110, 119)
                    if lo > block * page:
                        need = torch.maximum(need, e[at])
                    unit = torch.exp2(need)[:, None, None]
                    y = _nearest_e4m3(y / unit) * unit
                    head = pool[at, :, :lo - block * page]
                    pool[at, :, :lo - block * page] = _nearest_e4m3(head / unit) * unit
                    # Slots behind the new tokens keep their codes.
                    pool[at, :, hi - block * page:] *= torch.exp2(need - e[at])[:, None, None]
                pool[at, :, lo - block * page:hi - block * page] = y
        pools.append(pool[:-1])
    # A rotated key lies next to a border of its code now and then.
    return q, None if coded else pools[0], pools[1]


def _exact_norm(st):
    case = st["case"]
    x, r, w, gate, scale, shift, p = (None if st[n] is None else st[n].detach().double() for n in NORM_INPUTS)
    W, alpha = case["W"], case["alpha"]
    one = torch.ones((), dtype=torch.float64, device="cuda")
    g, s = (one if gate is None else gate), (one if scale is None else 1 + scale)
    gain, post = (one if w is None else w), (one if p is None else p)
    rx = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / W + 1e-6) if p is not None else one
    nx = x * rx
    h = alpha * r + g * (nx * post)
    rh = 1.0 / torch.sqrt((h * h).sum(-1, keepdim=True) / W + 1e-6)
    nh = h * rh
    n = nh * gain * s + (0.0 if shift is None else shift)
    if not case["grad"]:
        return n, h
    dn = st["dn"].double()
    t = dn * gain * s
    dh = st["dh"].double() + rh * (t - nh * (t * nh).sum(-1, keepdim=True) / W)
    dnx = dh * g * post
    dx = dnx if p is None else rx * (dnx - nx * (dnx * nx).sum(-1, keepdim=True) / W)

    def shaped(d, like):
        return d.sum_to_size(like.shape)

    grads = [dx, alpha * dh]
    if w is not None:
        grads.append(shaped(dn * s * nh, w))
    if gate is not None:
        grads.append(shaped(dh * nx * post, gate))
    if scale is not None:
        grads += [shaped(dn * nh * gain, scale), shaped(dn, shift)]
    if p is not None:
        grads.append(shaped(dh * g * nx, p))
    return (n, h, *grads)


def exact(case, seed):
    """What ``run`` returns, in float64 from the definition."""
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "attend":
            return _exact_attend(st)
        if case["kind"] == "append":
            return _exact_append(st)
        return _exact_norm(st)


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    if case["kind"] == "norm":
        size = 2 if case["dtype"] == "bfloat16" else 4
        B, W, n = case["B"], case["W"], case["B"] * case["L"] * case["W"]
        rows = {"none": 0, "gate": 1, "batch": 3 * B, "token": 3 * B * case["L"]}[case["modulation"]]
        small = (rows + int(case["gain"]) + int(case["post"])) * W * size
        if case["grad"]:
            # x, the residual and both gradients in; norm, sum and two
            # gradients out (the same one where neither gate, norm nor factor
            # tells them apart).
            alike = rows == 0 and not case["post"] and case["alpha"] == 1.0
            return {"bytes": (7 if alike else 8) * n * size + 2 * small, "flops": 30 * n}
        return {"bytes": 4 * n * size + small, "flops": 10 * n}
    B, H, Hkv, D, page = (case[n] for n in ("B", "H", "Hkv", "D", "page"))
    size = 1 if case["pages"] == "e4m3" else 2
    lengths, new = _lengths(case)
    if case["kind"] == "attend":
        reach = case["window"] or case["length"]
        seen = sum(min(n, m + reach - 1) for n, m in zip(lengths, new))
        pairs = sum(min(n - m + i + 1, reach) for n, m in zip(lengths, new) for i in range(m))
        blocks = -(-seen // page)
        return {"bytes": 2 * Hkv * seen * D * size + 2 * 2 * B * H * case["Lq"] * D + 4 * blocks,
                "flops": 4 * H * D * pairs}
    tokens = sum(new)
    table = 2 * 4 * tokens * case["dims"] // 2
    owned = B * (-(-max(lengths) // page)) * page * Hkv * D * 2
    # The values that the pages hold, read and written out, where they are
    # codes.
    held = owned * (1 + 2) if size == 1 else 0
    return {"bytes": 2 * (2 * B * case["L"] * H * D) + 2 * tokens * Hkv * D * (2 + size) + table + held,
            "flops": 3 * tokens * (H + Hkv) * case["dims"]}
