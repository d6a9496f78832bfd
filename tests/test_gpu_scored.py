"""Attention with changed scores on the GPU against dense float64.

Tolerances.  bf16 (u = 2^-8, half a step): P enters the second product rounded
(u of sum P|v|), the output is rounded (u of it).  Backward: the exchanged
P (1 - tanh^2) and dS are rounded (2 u of |dS|), delta comes from the rounded
output (its error times |dO|), each gradient is rounded.  float32: u = 2^-24,
no rounding of P or dS.  On top of these every probability is off by at most
``DP`` relatively: fp32 scores of head_dim products, of size up to ~30, summed
in any order (D/2 * 2^-24 * 30 in the worst case), the score's own operations,
and exp2.
"""

from __future__ import annotations

import math

import pytest
import torch

from avgen_amd import attention as A
from avgen_amd import scored_ops

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
DP = 64 * 2.0**-24 * 30 * 2


def heads(B, L, H, D, dtype, gen, spread=1.0):
    x = torch.randn((B, L, H * D), generator=gen, device="cuda") * spread
    return x.to(dtype).unflatten(-1, (H, D)).transpose(1, 2)


def make(B, Hq, Hkv, Lq, Lk, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (heads(B, Lq, Hq, D, dtype, g, 3.0), heads(B, Lk, Hkv, D, dtype, g), heads(B, Lk, Hkv, D, dtype, g),
            heads(B, Lq, Hq, D, dtype, g))


def slopes_of(Hq):
    return torch.tensor([2.0 ** (-8 * (h + 1) / Hq) for h in range(Hq)], device="cuda")


def dense_mask(B, Lq, Lk, lo=None, hi=None, mask=None):
    m = torch.ones((B, 1, Lq, Lk), dtype=torch.bool, device="cuda")
    if lo is not None:
        j = torch.arange(Lk, device="cuda")
        w = (j >= lo[..., None]) & (j < hi[..., None])
        m = m & (w[:, None] if w.ndim == 3 else w)
    if mask is not None:
        m = m & mask.bool().expand(B, Lk)[:, None, None]
    return m


class Oracle:
    """Dense float64 attention and its gradients, with the error bounds above.
    Keys that no row attends are taken as zeros."""

    def __init__(self, q, k, v, dout=None, cap=None, slopes=None, offset=0, lo=None, hi=None, mask=None, scale=None):
        B, Hq, Lq, D = q.shape
        Hkv, Lk = k.shape[1], k.shape[2]
        u = U[q.dtype]
        g = Hq // Hkv
        allow = dense_mask(B, Lq, Lk, lo, hi, mask)
        used = allow.any(2)[:, 0, :, None]  # (B, Lk, 1)
        kk, vv = (torch.where(used[:, None], t, torch.zeros_like(t)).double().repeat_interleave(g, 1) for t in (k, v))
        q = q.double()
        scale = 1 / math.sqrt(D) if scale is None else scale
        z = scale * q @ kk.transpose(-1, -2).contiguous()
        fac = torch.ones_like(z)
        if cap is not None:
            t = torch.tanh(z / cap)
            fac, z = 1 - t * t, cap * t
        if slopes is not None:
            off = torch.as_tensor(offset, device="cuda").reshape(-1, 1, 1)
            d = (torch.arange(Lq, device="cuda")[:, None] + off - torch.arange(Lk, device="cuda")).abs()
            z = z - slopes.double()[:, None, None] * d[:, None]
        z = torch.where(allow, z, torch.full_like(z, -math.inf))
        self.lse = torch.logsumexp(z, -1)
        p = torch.exp(z - torch.where(self.lse.isfinite(), self.lse, torch.zeros_like(self.lse))[..., None])
        self.out = p @ vv
        size = p @ vv.abs()
        self.out_tol = u * self.out.abs() + ((u if u > 1e-5 else 0) + DP) * size
        if dout is None:
            return
        do = dout.double()
        dp = do @ vv.transpose(-1, -2).contiguous()
        delta = (p * dp).sum(-1, keepdim=True)
        ds = p * (dp - delta) * fac
        ddelta = (do.abs() * self.out_tol).sum(-1, keepdim=True)
        dpsize = do.abs() @ vv.abs().transpose(-1, -2).contiguous()
        r = 2 * u if u > 1e-5 else 0.0
        e = (r * 1.02 + 2 * DP) * ds.abs() + p * fac.abs() * (ddelta * 1.02 + 2 * DP * (dpsize + delta.abs()))

        def kv(t):
            return t.unflatten(1, (Hkv, g)).sum(2)

        T = lambda t: t.transpose(-1, -2).contiguous()
        self.dq, self.dq_tol = scale * ds @ kk, scale * e @ kk.abs()
        self.dk, self.dk_tol = scale * kv(T(ds) @ q), scale * kv(T(e) @ q.abs())
        self.dv = kv(T(p) @ do)
        self.dv_tol = ((u if u > 1e-5 else 0) + 2 * DP) * kv(T(p) @ do.abs())
        for n in ("dq", "dk", "dv"):
            setattr(self, n + "_tol", getattr(self, n + "_tol") + u * getattr(self, n).abs())

    def check(self, **got):
        for name, x in got.items():
            want, tol = getattr(self, name), getattr(self, name + "_tol")
            assert x.isfinite().all(), name
            err = (x.double() - want).abs()
            assert bool((err <= tol * 1.01 + 1e-7).all()), (name, float((err - tol).max()), float(err.max()))

    def check_lse(self, lse):
        dead = self.lse == -math.inf
        assert torch.equal(lse == -math.inf, dead)
        ok = ~dead
        assert bool(((lse.double() - self.lse).abs()[ok] <= DP + 2.0**-22 * self.lse.abs()[ok]).all())


def windows(kind, B, Lq, Lk, seed=0):
    """(lo, hi, key mask) of a kind of mask."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    i = torch.arange(Lq, device="cuda")
    shift = Lk - Lq
    if kind == "none":
        return None, None, None
    if kind == "causal":
        return torch.zeros_like(i).int(), (i + 1 + shift).clamp(0, Lk).int(), None
    if kind == "sliding":
        return (i + shift - 40).clamp(0, Lk).int(), (i + 1 + shift).clamp(0, Lk).int(), None
    if kind == "documents":
        cu = torch.tensor([0, Lk // 3, Lk // 3 + 1, Lk // 2, max(Lk - 5, Lk // 2)], device="cuda")
        lo, hi = A.document_windows(cu, max(Lq, Lk))
        return lo[:Lq], hi[:Lq], None
    mask = torch.rand((B, Lk), generator=g, device="cuda") > 0.3
    if kind == "padding":
        mask[:, (2 * Lk) // 3:] = False
        mask[B - 1] = False  # a batch row without keys
        return None, None, mask
    if kind == "both":
        lo, hi, _ = windows("sliding", B, Lq, Lk)
        lo = torch.stack([(lo - 7 * b).clamp(min=0) for b in range(B)])
        hi = torch.stack([hi] * B)
        if Lq > 2:  # rows without keys: the first, and the last two past the end
            hi[:, :1] = 0
            lo[:, :1] = 0
            lo[:, -2:] = Lk
            hi[:, -2:] = Lk
        return lo.int().contiguous(), hi.int().contiguous(), mask
    raise AssertionError(kind)


SHAPES = [
    (1, 1, 1, 1, 1, 64),
    (1, 2, 1, 3, 5, 128),
    (2, 4, 2, 70, 130, 64),
    (2, 6, 6, 65, 65, 128),
    (1, 8, 2, 257, 300, 128),
    (1, 4, 4, 400, 1100, 128),
    (1, 2, 1, 1000, 1025, 64),
    (1, 12, 3, 513, 513, 128),
    # More row blocks than the few-row kernels take:
    (2, 16, 16, 300, 333, 128),
    (1, 36, 18, 515, 520, 64),
    (1, 8, 8, 400, 2100, 128),
    (1, 4, 4, 1000, 2500, 128),  # 256-row workgroups
    (1, 12, 6, 700, 2300, 64),
]
SCORES = [("cap", 20.0), ("slopes", None), ("both", 5.0), ("none", None)]
MASKS = ["none", "causal", "sliding", "documents", "padding", "both"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("score", SCORES, ids=[s[0] for s in SCORES])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, score, kind, dtype):
    B, Hq, Hkv, Lq, Lk, D = shape
    q, k, v, do = make(*shape, dtype, seed=Lq + Lk)
    lo, hi, mask = windows(kind, B, Lq, Lk)
    cap = score[1]
    slopes = slopes_of(Hq) if score[0] in ("slopes", "both") else None
    offset = Lk - Lq
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(q, k, v, softcap=cap, distance_slopes=slopes, query_offset=offset, window_lo=lo,
                             window_hi=hi, attn_mask=None if mask is None else mask[:, None, None], enable_gqa=True)
    grads = torch.autograd.grad(out, leaves, do)
    o = Oracle(*(t.detach() for t in (q, k, v)), do, cap, slopes, offset, lo, hi, mask)
    o.check(out=out.detach(), dq=grads[0], dk=grads[1], dv=grads[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 1, 128), (8, 8, 2, 1, 1000, 128), (2, 8, 2, 4, 333, 64), (1, 4, 4, 33, 500, 128),
    (1, 64, 1, 1, 4096, 64), (3, 5, 5, 7, 31, 64), (1, 16, 4, 4, 40000, 128), (2, 2, 1, 2, 9001, 128),
    (40, 8, 8, 1, 257, 128), (1, 32, 2, 4, 65, 128),
])
@pytest.mark.parametrize("score", SCORES, ids=[s[0] for s in SCORES])
def test_few_rows_against_a_cache(shape, score, dtype):
    """A cache of Lk slots, each sequence with a length of its own; the unused
    slots hold NaN."""
    B, Hq, Hkv, Lq, Lk, D = shape
    q, k, v, _ = make(*shape, dtype, seed=Lk)
    g = torch.Generator().manual_seed(Lk)
    length = torch.randint(min(Lk, max(Lq, Lk // 2)), Lk + 1, (B,), generator=g).to("cuda", torch.int32)
    for b in range(B):
        k[b, :, length[b]:] = float("nan")
        v[b, :, length[b]:] = float("nan")
    i = torch.arange(Lq, device="cuda", dtype=torch.int32)
    hi = (length[:, None] - Lq + 1 + i).clamp(min=0)
    lo = torch.zeros_like(hi)
    slopes = slopes_of(Hq) if score[0] in ("slopes", "both") else None
    offsets = (length - Lq).to(torch.int32)
    out, lse = scored_ops.flash_fwd_scored(q, k, v, lo, hi, None, slopes, offsets, 1 / math.sqrt(D), score[1] or 0.0, 0)
    o = Oracle(q, k, v, None, score[1], slopes, offsets, lo, hi)
    o.check(out=out)
    o.check_lse(lse)


@pytest.mark.parametrize("kind", ["padding", "both", "documents", "none"])
@pytest.mark.parametrize("shape", [(3, 8, 2, 2, 700, 128), (2, 4, 4, 5, 100, 64), (2, 16, 1, 3, 2000, 64)])
def test_few_rows_masks(shape, kind):
    B, Hq, Hkv, Lq, Lk, D = shape
    q, k, v, do = make(*shape, torch.bfloat16, seed=7)
    lo, hi, mask = windows(kind, B, Lq, Lk)
    slopes = slopes_of(Hq)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(q, k, v, softcap=10.0, distance_slopes=slopes, query_offset=Lk - Lq, window_lo=lo,
                             window_hi=hi, attn_mask=None if mask is None else mask[:, None, None], enable_gqa=True)
    o = Oracle(*(t.detach() for t in (q, k, v)), do, 10.0, slopes, Lk - Lq, lo, hi, mask)
    grads = torch.autograd.grad(out, leaves, do)
    o.check(out=out.detach(), dq=grads[0], dk=grads[1], dv=grads[2])


@pytest.mark.parametrize("kind", ["padding", "both", "documents", "none"])
@pytest.mark.parametrize("shape", [(3, 8, 2, 2, 700, 128), (2, 4, 4, 5, 100, 64), (2, 16, 1, 1, 2000, 64),
                                   (2, 3, 3, 3, 95, 128)])
@pytest.mark.parametrize("score", SCORES, ids=[s[0] for s in SCORES])
def test_few_rows_masks_float32(shape, kind, score):
    B, Hq, Hkv, Lq, Lk, D = shape
    q, k, v, _ = make(*shape, torch.float32, seed=9)
    lo, hi, mask = windows(kind, B, Lq, Lk)
    slopes = slopes_of(Hq) if score[0] in ("slopes", "both") else None
    with torch.no_grad():
        out = A.scored_attention(q, k, v, softcap=score[1], distance_slopes=slopes, query_offset=Lk - Lq,
                                 window_lo=lo, window_hi=hi,
                                 attn_mask=None if mask is None else mask[:, None, None], enable_gqa=True)
    Oracle(q, k, v, None, score[1], slopes, Lk - Lq, lo, hi, mask).check(out=out)


@pytest.mark.parametrize("dtype,shape", [
    (torch.bfloat16, (1, 8, 2, 32, 300, 64)), (torch.bfloat16, (1, 8, 2, 33, 300, 64)),
    (torch.bfloat16, (2, 2, 2, 64, 200, 128)), (torch.bfloat16, (2, 2, 2, 65, 200, 128)),
    (torch.bfloat16, (1, 80, 2, 1, 300, 128)), (torch.float32, (1, 8, 2, 16, 300, 64)),
    (torch.float32, (1, 8, 2, 17, 300, 64)), (torch.float32, (2, 3, 3, 16, 200, 128)),
    (torch.float32, (2, 40, 2, 1, 200, 128)),
    (torch.bfloat16, (1, 64, 64, 256, 256, 64)), (torch.bfloat16, (1, 64, 64, 257, 256, 64)),
    (torch.bfloat16, (1, 32, 32, 256, 200, 128)), (torch.bfloat16, (1, 32, 32, 257, 200, 128)),
    (torch.bfloat16, (1, 8, 8, 256, 2049, 128)), (torch.bfloat16, (1, 8, 8, 257, 2049, 128)),
    (torch.float32, (1, 8, 8, 256, 512, 64)), (torch.float32, (1, 8, 8, 260, 512, 64)),
    (torch.float32, (1, 8, 8, 128, 513, 64)), (torch.float32, (1, 8, 8, 132, 513, 64)),
], ids=str)
def test_either_side_of_the_few_rows(dtype, shape):
    """The largest sizes of the few-row kernels and the next ones."""
    q, k, v, _ = make(*shape, dtype, seed=11)
    B, Hq, Hkv, Lq, Lk, D = shape
    lo, hi, mask = windows("both", B, Lq, Lk)
    slopes = slopes_of(Hq)
    with torch.no_grad():
        out = A.scored_attention(q, k, v, softcap=20.0, distance_slopes=slopes, query_offset=Lk - Lq, window_lo=lo,
                                 window_hi=hi, attn_mask=mask[:, None, None], enable_gqa=True)
    Oracle(q, k, v, None, 20.0, slopes, Lk - Lq, lo, hi, mask).check(out=out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(2, 4, 2, 3, 300, 64), (2, 4, 2, 200, 300, 128), (1, 2, 2, 300, 1200, 128),
                                   (2, 72, 36, 200, 300, 64), (1, 16, 16, 1000, 1200, 128)])
def test_windows_in_any_order(shape, dtype):
    """Forward only: windows that are not sorted, wider and narrower, empty,
    reversed or out of range (clamped)."""
    B, Hq, Hkv, Lq, Lk, D = shape
    q, k, v, _ = make(*shape, dtype, seed=3)
    g = torch.Generator(device="cuda").manual_seed(1)
    lo = torch.randint(-20, Lk + 20, (B, Lq), generator=g, device="cuda", dtype=torch.int32)
    hi = torch.randint(-20, Lk + 20, (B, Lq), generator=g, device="cuda", dtype=torch.int32)
    out = A.scored_attention(q, k, v, softcap=15.0, window_lo=lo, window_hi=hi, enable_gqa=True)
    Oracle(q, k, v, None, 15.0, None, 0, lo.clamp(0, Lk), hi.clamp(0, Lk)).check(out=out)
    with pytest.raises(ValueError, match="non-decreasing"):
        qq = q.clone().requires_grad_(True)
        A.scored_attention(qq, k, v, softcap=15.0, window_lo=lo, window_hi=hi, enable_gqa=True).sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq, Hq, Hkv", [(2, 4, 2), (300, 4, 2), (300, 40, 20)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_unattended_keys_hold_never_counts(Lq, Hq, Hkv, bad, dtype):
    B, Lk, D = 2, 310, 128
    q, k, v, do = make(B, Hq, Hkv, Lq, Lk, D, dtype)
    mask = torch.rand((B, Lk), device="cuda") > 0.4
    mask[1, 200:] = False
    lo = torch.full((Lq,), 5, device="cuda", dtype=torch.int32)
    hi = torch.full((Lq,), 290, device="cuda", dtype=torch.int32)
    dead = ~mask.clone()
    dead[:, :5] = True
    dead[:, 290:] = True
    clean = [t.clone() for t in (k, v)]
    for t in (k, v):
        t[dead[:, None].expand(B, Hkv, Lk)] = bad
    for kw in (dict(softcap=20.0), dict(distance_slopes=slopes_of(Hq))):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        args = dict(window_lo=lo, window_hi=hi, attn_mask=mask[:, None, None], enable_gqa=True, **kw)
        out = A.scored_attention(*leaves, **args)
        got = (out,) + torch.autograd.grad(out, leaves, do)
        leaves = [t.detach().requires_grad_(True) for t in (q, *clean)]
        out = A.scored_attention(*leaves, **args)
        want = (out,) + torch.autograd.grad(out, leaves, do)
        for a, b in zip(got, want):
            assert a.isfinite().all() and torch.equal(a, b)
        for t in got[2:]:
            assert not t[dead[:, None].expand(B, Hkv, Lk)].any()


@pytest.mark.parametrize("Lq, heads", [(1, 4), (200, 4), (200, 160)])
def test_garbage_in_queries_without_keys(Lq, heads):
    q, k, v, _ = make(1, heads, heads // 2, Lq, 200, 64, torch.bfloat16)
    lo = torch.zeros(Lq, device="cuda", dtype=torch.int32)
    hi = torch.full_like(lo, 150)
    hi[Lq // 2:] = 0
    q[:, :, Lq // 2:] = float("nan")
    for kw in (dict(softcap=9.0), dict(distance_slopes=slopes_of(heads))):
        out = A.scored_attention(q, k, v, window_lo=lo, window_hi=hi, enable_gqa=True, **kw)
        assert not out[:, :, Lq // 2:].any() and out.isfinite().all()


@pytest.mark.parametrize("heads", [2, 264])
def test_nan_key_reaches_the_rows_that_attend_it(heads):
    q, k, v, _ = make(1, heads, heads, 64, 64, 64, torch.bfloat16)
    k[0, 0, 10] = float("nan")
    lo, hi, _ = windows("causal", 1, 64, 64)
    out = A.scored_attention(q, k, v, softcap=9.0, window_lo=lo, window_hi=hi)
    assert out[0, 0, 10:].isnan().all() and out[0, 1:].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq, Hq, Hkv", [(3, 4, 2), (130, 4, 2), (130, 128, 64)])
@pytest.mark.parametrize("kw", [dict(cap=0.5), dict(cap=50.0, spread=40.0), dict(slope=30.0), dict(slope=-0.5),
                                dict(slope=-3.0, cap=4.0), dict(cap=1e4), dict(slope=0.0)], ids=str)
def test_extreme_scores(Lq, Hq, Hkv, kw, dtype):
    """Caps far below and above the scores, scores far beyond the cap, slopes
    that leave one key and slopes that favour the farthest."""
    B, Lk, D = 1, 200, 64
    q, k, v, do = make(B, Hq, Hkv, Lq, Lk, D, dtype, 11)
    q = (q.float() * kw.get("spread", 1.0)).to(dtype)
    slopes = None if "slope" not in kw else torch.full((Hq,), kw["slope"], device="cuda")
    cap = kw.get("cap")
    if dtype is torch.bfloat16 and cap == 1e4:
        cap = 1024.0  # the largest there
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(*leaves, softcap=cap, distance_slopes=slopes, query_offset=10, enable_gqa=True)
    grads = torch.autograd.grad(out, leaves, do)
    o = Oracle(q, k, v, do, cap, slopes, 10)
    if kw.get("spread", 1.0) > 1:  # the raw scores' error grows with them: 40 times the size DP stands for
        for n in ("out", "dq", "dk", "dv"):
            setattr(o, n + "_tol", getattr(o, n + "_tol") * 40)
    o.check(out=out.detach(), dq=grads[0], dk=grads[1], dv=grads[2])


@pytest.mark.parametrize("heads", [1, 180])
def test_infinite_scores_with_a_cap_are_the_cap(heads):
    q = torch.full((1, 1, 70, 64), 3e38, device="cuda")
    k = torch.randn((1, 1, 70, 64), device="cuda").sign() * torch.ones((1, 1, 70, 1), device="cuda")
    k[:, :, ::2] = 1.0
    k[:, :, 1::2] = -1.0
    v = torch.randn((1, 1, 70, 64), device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        out = A.scored_attention(*(t.to(dtype).expand(1, heads, 70, 64) for t in (q, k, v)), softcap=2.0)
        assert bool((out == out[:, :1]).all())
        w = torch.where(torch.arange(70, device="cuda") % 2 == 0, 2.0, -2.0).double().softmax(0)
        want = (w[:, None] * v.to(dtype)[0, 0].double()).sum(0)
        size = (w[:, None] * v[0, 0].double().abs()).sum(0)
        assert bool(((out[0, 0].double() - want).abs() <= (2 * U[dtype] + 1e-5) * size).all())


def test_gradient_against_differences():
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v, w = (torch.randn((1, 2, 9, 64), generator=g, device="cuda").double() for _ in range(4))
    slopes = torch.tensor([0.1, 0.3], device="cuda")
    lo, hi, _ = windows("causal", 1, 9, 9)

    def loss(q, k, v):
        return (Oracle(q.float(), k.float(), v.float(), None, 2.0, slopes, 0, lo, hi).out * w).sum().item()

    leaves = [t.float().requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(*leaves, softcap=2.0, distance_slopes=slopes, window_lo=lo, window_hi=hi)
    grads = torch.autograd.grad(out, leaves, w.float())
    step = 2.0**-7  # inputs reach the oracle as float32: steps it holds; error ~ step^2 / 6 of a third derivative
    for n in range(3):
        for idx in range(0, 2 * 9 * 64, 97):
            t = [x.float().double() for x in (q, k, v)]
            flat = t[n].reshape(-1)
            keep = flat[idx].item()
            flat[idx] = keep + step
            up = loss(*t)
            flat[idx] = keep - step
            down = loss(*t)
            assert abs((up - down) / (2 * step) - grads[n].reshape(-1)[idx].item()) < 2e-3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq, Hq, Hkv", [(2, 4, 2), (150, 4, 2), (150, 56, 28)])
def test_layouts(Lq, Hq, Hkv, dtype):
    """Contiguous, (B, L, H, D) views, keys shared by expansion, slices of a
    cache, unaligned rows: the same values."""
    B, Lk, D = 2, 150, 64
    q, k, v, _ = make(B, Hq, Hkv, Lq, Lk, D, dtype)
    base = A.scored_attention(q.contiguous(), k.contiguous(), v.contiguous(), softcap=7.0, enable_gqa=True)
    assert torch.equal(A.scored_attention(q, k, v, softcap=7.0, enable_gqa=True), base)
    cache = torch.full((B, 400, Hkv, 2 * D), float("nan"), device="cuda", dtype=dtype)
    cache[:, 30:30 + Lk, :, :D] = k.transpose(1, 2)
    cache[:, 30:30 + Lk, :, D:] = v.transpose(1, 2)
    kc, vc = (t[:, 30:30 + Lk].transpose(1, 2) for t in (cache[..., :D], cache[..., D:]))
    assert torch.equal(A.scored_attention(q, kc, vc, softcap=7.0, enable_gqa=True), base)
    pad = torch.zeros((B, Hkv, Lk, D + 1), device="cuda", dtype=dtype)
    pad[..., 1:] = k
    assert torch.equal(A.scored_attention(q, pad[..., 1:], v, softcap=7.0, enable_gqa=True), base)
    one = A.scored_attention(q[:1], k[:1], v[:1], softcap=7.0, enable_gqa=True)
    both = A.scored_attention(q[:1].expand(3, -1, -1, -1), k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1),
                              softcap=7.0, enable_gqa=True)
    for b in range(3):
        assert bool(((both[b] - one[0]).abs() <= 4 * U[dtype] * one[0].abs().amax()).all())
    same = A.scored_attention(q, k[:, :, :1].expand(-1, -1, 90, -1), v[:, :, :1].expand(-1, -1, 90, -1), softcap=7.0,
                              enable_gqa=True)
    want = v[:, :, :1].repeat_interleave(2, 1).expand(-1, -1, Lq, -1)
    assert bool(((same - want).abs() <= 2 * U[dtype] * want.abs() + DP).all())


def test_one_row_at_a_time_is_the_whole_prefill():
    """Decoding token by token against a filling cache gives the rows of the
    causal forward."""
    B, Hq, Hkv, L, D = 2, 8, 2, 97, 128
    q, k, v, _ = make(B, Hq, Hkv, L, L, D, torch.bfloat16)
    slopes = slopes_of(Hq)
    lo, hi = A.document_windows(torch.tensor([0, L]), L, causal=True, device="cuda")
    whole = A.scored_attention(q, k, v, softcap=12.0, distance_slopes=slopes, window_lo=lo, window_hi=hi,
                               enable_gqa=True, monotone=True)
    o = Oracle(q, k, v, None, 12.0, slopes, 0, lo, hi)
    o.check(out=whole)
    cache_k, cache_v = (torch.full_like(t, float("nan")) for t in (k, v))
    rows = []
    for i in range(L):
        cache_k[:, :, i], cache_v[:, :, i] = k[:, :, i], v[:, :, i]
        end = torch.full((B, 1), i + 1, device="cuda", dtype=torch.int32)
        rows.append(A.scored_attention(q[:, :, i:i + 1], cache_k, cache_v, softcap=12.0, distance_slopes=slopes,
                                       query_offset=end[:, 0] - 1, window_lo=torch.zeros_like(end), window_hi=end,
                                       enable_gqa=True, monotone=True))
    o.check(out=torch.cat(rows, 2))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_staging_in_passes_and_compactly(dtype, monkeypatch):
    from avgen_amd import ops

    shape = (2, 4, 2, 300, 400, 64)
    q, k, v, do = make(*shape, dtype)
    lo, hi, _ = windows("sliding", 2, 300, 400)

    def grads(**kw):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = A.scored_attention(*leaves, softcap=6.0, enable_gqa=True, **kw)
        return torch.autograd.grad(out, leaves, do)

    for kw in (dict(), dict(window_lo=lo, window_hi=hi)):
        want = grads(**kw)
        try:
            for budget in (0, 3 * 2 * 2 * 320 * 512 * 4):
                ops.set_ds_budget(budget)
                for a, b in zip(grads(**kw), want):
                    tol = 2 * U[dtype] * b.abs() + 1e-5 * b.abs().amax()
                    assert bool(((a - b).abs() <= tol).all())
        finally:
            ops.set_ds_budget(None)


@pytest.mark.parametrize("heads", [8, 16])
def test_repeatable_on_any_stream(heads):
    q, k, v, do = make(1, heads, heads // 4, 700, 700, 128, torch.bfloat16)
    lo, hi, _ = windows("causal", 1, 700, 700)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        out = A.scored_attention(*leaves, softcap=30.0, window_lo=lo, window_hi=hi, enable_gqa=True, monotone=True)
        few = A.scored_attention(q[:, :, :2], k, v, softcap=30.0, enable_gqa=True)
        return (out, few) + torch.autograd.grad(out, leaves, do)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
        third = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("heads", [4, 64])
def test_captured_and_replayed(heads):
    """Two graphs, replayed in turn with eager calls between them."""
    L = 300
    q, k, v, do = make(1, heads, heads // 2, L, L, 64, torch.bfloat16)
    lo, hi, _ = windows("causal", 1, L, L)
    slopes = slopes_of(heads)
    scale = 0.125
    end = torch.full((1, 1), 200, device="cuda", dtype=torch.int32)

    def train():
        out, lse = scored_ops.flash_fwd_scored(q, k, v, lo, hi, None, slopes, None, scale, 8.0, 0, True)
        return (out, lse) + tuple(scored_ops.flash_bwd_scored(do, q, k, v, out, lse, lo, hi, None, slopes, None, scale,
                                                              8.0, 0, True))

    def serve():
        return scored_ops.flash_fwd_scored(q[:, :, :1], k, v, torch.zeros_like(end), end, None, slopes, end[:, 0], scale,
                                           8.0, 0, True)

    with torch.no_grad():
        graphs = []
        for fn in (train, serve):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                fn()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = fn()
            graphs.append((graph, outs, fn))
        for step in range(4):
            q.copy_(torch.randn_like(q))
            end.fill_(100 + 7 * step)
            for graph, _, _ in graphs:
                graph.replay()
            for _, outs, fn in graphs:
                torch.cuda.synchronize()
                for a, b in zip(outs, fn()):
                    assert torch.equal(a, b)


def test_empty_sizes():
    q, k, v, _ = make(2, 4, 2, 5, 7, 64, torch.bfloat16)
    assert not A.scored_attention(q, k[:, :, :0], v[:, :, :0], softcap=3.0, enable_gqa=True).any()
    assert A.scored_attention(q[:, :, :0], k, v, softcap=3.0, enable_gqa=True).shape == (2, 4, 0, 64)
    assert A.scored_attention(q[:0], k[:0], v[:0], softcap=3.0, enable_gqa=True).shape == (0, 4, 5, 64)
    out, lse = scored_ops.flash_fwd_scored(q, k[:, :, :0], v[:, :, :0], None, None, None, None, None, 0.1, 3.0, 0)
    assert not out.any() and bool((lse == -math.inf).all())


def test_ops_pass_opcheck_and_compile():
    q, k, v, _ = make(1, 2, 1, 9, 12, 64, torch.float32)
    q.requires_grad_(True)
    lo, hi, _ = windows("causal", 1, 9, 12)
    args = (q, k, v, lo, hi, None, slopes_of(2), None, 0.125, 5.0, 3, True)
    torch.library.opcheck(scored_ops._fwd_op, args)
    fn = torch.compile(lambda a: A.scored_attention(a, k, v, softcap=5.0, window_lo=lo, window_hi=hi, enable_gqa=True,
                                                    monotone=True), fullgraph=True)
    want = A.scored_attention(q, k, v, softcap=5.0, window_lo=lo, window_hi=hi, enable_gqa=True, monotone=True)
    assert torch.equal(fn(q), want)


def test_document_windows():
    cu = torch.tensor([0, 4, 5, 9])
    lo, hi = A.document_windows(cu, 11)
    assert lo.tolist() == [0] * 4 + [4] + [5] * 4 + [9, 9] and hi.tolist() == [4] * 4 + [5] + [9] * 4 + [9, 9]
    lo, hi = A.document_windows(cu, 11, causal=True)
    assert hi.tolist() == [1, 2, 3, 4, 5, 6, 7, 8, 9, 9, 9]
    lo, hi = A.document_windows(cu, 11, causal=True, prefix_lengths=torch.tensor([3, 7, 2]))
    assert hi.tolist() == [3, 3, 3, 4, 5, 7, 7, 8, 9, 9, 9]
    lo, hi = A.document_windows(torch.tensor([0, 6]), 6, causal=True, prefix_lengths=4, device="cuda")
    assert hi.tolist() == [4, 4, 4, 4, 5, 6] and hi.is_cuda and hi.dtype is torch.int32
    lo, hi = A.document_windows(torch.tensor([0]), 3, causal=True)
    assert lo.tolist() == hi.tolist() == [0, 0, 0]
    with pytest.raises(ValueError):
        A.document_windows(cu, 11, causal=True, prefix_lengths=torch.tensor([3, 7]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq, Lk", [(3, 0), (200, 0), (0, 7)])
def test_gradients_of_empty_sizes(Lq, Lk, dtype):
    q, k, v, do = make(2, 4, 2, Lq, Lk, 64, dtype)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(*leaves, softcap=3.0, distance_slopes=slopes_of(4), enable_gqa=True)
    assert not out.any()
    for g, t in zip(torch.autograd.grad(out, leaves, do), leaves):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_broadcast_inputs(dtype):
    """Keys shared by the batch rows and an output gradient without strides."""
    B, Hq, Hkv, Lq, Lk, D = 3, 4, 2, 70, 90, 64
    q, k, v, _ = make(B, Hq, Hkv, Lq, Lk, D, dtype)
    one = [t[:1].detach().requires_grad_(True) for t in (k, v)]
    leaves = [q.requires_grad_(True), *one]
    out = A.scored_attention(q, *(t.expand(B, -1, -1, -1) for t in one), softcap=9.0, enable_gqa=True)
    got = torch.autograd.grad(out.sum(), leaves)
    o = Oracle(q.detach(), *(t.detach().expand(B, -1, -1, -1) for t in one), torch.ones_like(q), 9.0)
    o.check(out=out.detach(), dq=got[0])
    # Summed over the batch by three more roundings at most.
    for name, g in (("dk", got[1]), ("dv", got[2])):
        want, tol = getattr(o, name), getattr(o, name + "_tol")
        bound = tol.sum(0, keepdim=True) + 3 * U[dtype] * want.abs().sum(0, keepdim=True)
        assert bool(((g.double() - want.sum(0, keepdim=True)).abs() <= bound * 1.01 + 1e-7).all()), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["none", "causal", "both"])
@pytest.mark.parametrize("shape", [(3, 32, 32, 150, 390, 64), (2, 40, 20, 200, 900, 128)])
def test_grids_past_one_round(shape, kind, dtype):
    """More key blocks than the chip holds at once, a last round that is split,
    and heads that do not divide over its eighths."""
    B, Hq, Hkv, Lq, Lk, D = shape
    q, k, v, do = make(*shape, dtype, seed=21)
    lo, hi, mask = windows(kind, B, Lq, Lk)
    slopes = slopes_of(Hq)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(*leaves, softcap=12.0, distance_slopes=slopes, query_offset=Lk - Lq, window_lo=lo,
                             window_hi=hi, attn_mask=None if mask is None else mask[:, None, None], enable_gqa=True)
    grads = torch.autograd.grad(out, leaves, do)
    o = Oracle(*(t.detach() for t in leaves), do, 12.0, slopes, Lk - Lq, lo, hi, mask)
    o.check(out=out.detach(), dq=grads[0], dk=grads[1], dv=grads[2])


@pytest.mark.parametrize("L, heads, kv", [(128, 4, 2), (384, 4, 1), (1024, 2, 1), (2048, 4, 1)])
@pytest.mark.parametrize("kind", ["none", "causal", "documents"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_split_backward(L, heads, kv, kind, dtype):
    """Few key blocks of many or few query tiles: parts down to a tile, and
    empty ones."""
    D = 64
    q, k, v, do = make(1, heads, kv, L, L, D, dtype, seed=L)
    lo, hi, _ = windows(kind, 1, L, L)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(*leaves, softcap=12.0, window_lo=lo, window_hi=hi, enable_gqa=True, monotone=True)
    grads = torch.autograd.grad(out, leaves, do)
    o = Oracle(*(t.detach() for t in leaves), do, 12.0, None, 0, lo, hi)
    o.check(out=out.detach(), dq=grads[0], dk=grads[1], dv=grads[2])
