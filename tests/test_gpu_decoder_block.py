"""A decoder block from the operators together: residual norm, projections,
rotation, attention with capped and distance-biased scores, residual norm, in
training over packed documents and in serving token by token from a cache.

Tolerances.  Training, float32: every step's result is off by at most 256
roundings (its longest sums) of 2^-24 of its largest value, 1.5e-5; scores of
size up to ~30 turn that into a relative error of 30 times as much in a
probability, 4.6e-4; the few steps in sequence stay below 2e-3 of the largest
value of each result.  A wrong angle, mask, offset, cap or slope is off by the
order of the values themselves.  Serving, bf16: the rows of prefill and of
decoding pass the same roundings at other places: for each of the ~8 roundings
on the way (residual sum, norm, projections, rotation, P, output) two half
steps of the largest value, 16 * 2^-8 = 6.25e-2.
"""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from avgen_amd import attention as A
from avgen_amd import layers, rope

pytestmark = pytest.mark.gpu

WIDTH, HQ, HKV, D, ROT = 256, 4, 2, 64, 32
CAP = 15.0


def weights(dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def w(o, i):
        return (torch.randn(o, i, generator=g, device="cuda") / math.sqrt(i)).to(dtype)

    return dict(n1=torch.rand(WIDTH, generator=g, device="cuda").to(dtype) + 0.5, wq=w(HQ * D, WIDTH),
                wk=w(HKV * D, WIDTH), wv=w(HKV * D, WIDTH), wo=w(WIDTH, HQ * D),
                n2=torch.rand(WIDTH, generator=g, device="cuda").to(dtype) + 0.5)


def slopes():
    return torch.exp2(-2.0 * (torch.arange(HQ, device="cuda", dtype=torch.float32) + 1))


def split(x, heads):
    return x.unflatten(-1, (heads, D)).transpose(1, 2)


def project(w, n):
    return (split(F.linear(n, w["wq"]), HQ), split(F.linear(n, w["wk"]), HKV), split(F.linear(n, w["wv"]), HKV))


def block(w, x, r, tables, lo, hi):
    n, h = layers.add_rms_norm(x, r, w["n1"])
    q, k, v = project(w, n)
    q, k = rope.rotate_query_key(q, k, tables, layout="half", start=D - ROT)
    o = A.scored_attention(q, k, v, softcap=CAP, distance_slopes=slopes(), window_lo=lo, window_hi=hi, enable_gqa=True,
                           monotone=True)
    return layers.add_rms_norm(F.linear(o.transpose(1, 2).flatten(2), w["wo"]), h, w["n2"])


def plain(w, x, r, positions, scaling, allow):
    """The same block in float64 from the formulas."""
    def norm(h, g):
        return h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * g

    def rotate(t):
        freq, amp = rope.position_frequencies(ROT, scaling=scaling)
        a = positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
        c, s = amp * torch.cos(a), amp * torch.sin(a)
        at = D - ROT
        t0, t1 = t[..., at:at + ROT // 2], t[..., at + ROT // 2:]
        return torch.cat([t[..., :at], t0 * c - t1 * s, t0 * s + t1 * c], -1)

    h = x + r
    q, k, v = project(w, norm(h, w["n1"]))
    q, k = rotate(q), rotate(k)
    k, v = (t.repeat_interleave(HQ // HKV, 1) for t in (k, v))
    z = CAP * torch.tanh(q @ k.transpose(-1, -2).contiguous() / math.sqrt(D) / CAP)
    i = torch.arange(x.shape[1], device="cuda", dtype=torch.float64)
    z = z - slopes().double()[:, None, None] * (i[:, None] - i).abs()
    z = torch.where(allow, z, torch.full_like(z, -math.inf))
    p = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-1e30))
    o = p @ v / p.sum(-1, keepdim=True).clamp(min=1e-300)
    h = F.linear(o.transpose(1, 2).flatten(2), w["wo"]) + h
    return norm(h, w["n2"]), h


def dense(lo, hi, L):
    j = torch.arange(L, device="cuda")
    return (j >= lo[:, None]) & (j < hi[:, None])


def test_training_over_packed_documents():
    B, L = 2, 333
    w = weights(torch.float32)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, r, dn, dh = (torch.randn(B, L, WIDTH, generator=g, device="cuda") for _ in range(4))
    cu = torch.tensor([0, 130, 131, 300], device="cuda")  # then 33 rows of padding
    lo, hi = A.document_windows(cu, L, causal=True, prefix_lengths=torch.tensor([17, 5, 64], device="cuda"))
    scaling = rope.PositionScaling("yarn", 4.0, original_length=64)
    positions = torch.arange(L, device="cuda") - lo  # from each document's start
    tables = rope.build_position_tables(positions, rotary_dim=ROT, scaling=scaling)

    leaves = {n: t.clone().requires_grad_(True) for n, t in dict(w, x=x, r=r).items()}
    n, h = block(leaves, leaves["x"], leaves["r"], tables, lo, hi)
    got = dict(zip(leaves, torch.autograd.grad((n, h), list(leaves.values()), (dn, dh))), n=n.detach(), h=h.detach())

    ref = {n: t.double().requires_grad_(True) for n, t in dict(w, x=x, r=r).items()}
    rn, rh = plain(ref, ref["x"], ref["r"], positions, scaling, dense(lo, hi, L))
    want = dict(zip(ref, torch.autograd.grad((rn, rh), list(ref.values()), (dn.double(), dh.double()))),
                n=rn.detach(), h=rh.detach())
    for name, t in want.items():
        # The norms' gains named n1 and n2, the results n and h.
        err = (got[name].double() - t).abs().max()
        assert float(err) <= 2e-3 * float(t.abs().max()), (name, float(err), float(t.abs().max()))


class Cache:
    """A cache with room for `size` tokens per sequence, unused slots NaN."""

    def __init__(self, B, size, dtype):
        self.k = torch.full((B, size, HKV, D), float("nan"), device="cuda", dtype=dtype)
        self.v = torch.full_like(self.k, float("nan"))
        self.batch = torch.arange(B, device="cuda")

    def put(self, at, k, v):  # at (B, L): the slots of k and v (B, HKV, L, D)
        self.k[self.batch[:, None], at] = k.transpose(1, 2)
        self.v[self.batch[:, None], at] = v.transpose(1, 2)


def serve(w, cache, x, r, length):
    """The block for the newest tokens of each sequence: `length` (B,) int32
    tokens are in the cache before them."""
    L = x.shape[1]
    at = length[:, None] + torch.arange(L, device="cuda", dtype=torch.int32)
    tables = rope.build_position_tables(at, rotary_dim=ROT)
    n, h = layers.add_rms_norm(x, r, w["n1"])
    q, k, v = project(w, n)
    q, k = rope.rotate_query_key(q, k, tables, layout="half", start=D - ROT)
    cache.put(at.long(), k, v)
    o = A.scored_attention(q, cache.k.transpose(1, 2), cache.v.transpose(1, 2), softcap=CAP, distance_slopes=slopes(),
                           query_offset=length, window_lo=torch.zeros_like(at), window_hi=at + 1, enable_gqa=True,
                           monotone=True)
    return layers.add_rms_norm(F.linear(o.transpose(1, 2).flatten(2), w["wo"]), h, w["n2"])


@pytest.mark.parametrize("dtype, tol", [(torch.float32, 2e-3), (torch.bfloat16, 6.25e-2)])
def test_serving_from_a_cache(dtype, tol):
    """Prefill of prompts, then single and drafted tokens: the rows of the
    causal forward over each whole sequence."""
    B, size = 3, 300
    w = weights(dtype)
    g = torch.Generator(device="cuda").manual_seed(2)
    total = 110
    x, r = (torch.randn(B, total, WIDTH, generator=g, device="cuda").to(dtype) for _ in range(2))
    start = torch.tensor([0, 40, 7], device="cuda", dtype=torch.int32)  # tokens cached before x
    before = torch.randn(B, 40, WIDTH, generator=g, device="cuda").to(dtype)

    with torch.no_grad():
        whole = []
        for b in range(B):
            s = int(start[b])
            seq = torch.cat([before[b:b + 1, :s], x[b:b + 1]], 1)
            res = torch.cat([torch.zeros_like(before[b:b + 1, :s]), r[b:b + 1]], 1)
            L = seq.shape[1]
            lo, hi = A.document_windows(torch.tensor([0, L], device="cuda"), L, causal=True)
            tables = rope.build_position_tables(torch.arange(L, device="cuda"), rotary_dim=ROT)
            whole.append([t[:, s:] for t in block(w, seq, res, tables, lo, hi)])
        whole_n, whole_h = (torch.cat([t[i] for t in whole]) for i in range(2))

        cache = Cache(B, size, dtype)
        for b in range(1, B):
            s = int(start[b])
            one = Cache(1, size, dtype)
            serve(w, one, before[b:b + 1, :s], torch.zeros_like(before[b:b + 1, :s]), torch.zeros_like(start[:1]))
            cache.k[b], cache.v[b] = one.k[0], one.v[0]
        at, rows = 0, []
        for step in (77, 1, 1, 5, 1, 20, 1, 4):
            rows.append(serve(w, cache, x[:, at:at + step], r[:, at:at + step], start + at))
            at += step
        assert at == total
        for got, want in zip((torch.cat([t[i] for t in rows], 1) for i in range(2)), (whole_n, whole_h)):
            assert got.isfinite().all()
            err = (got.double() - want.double()).abs().max()
            assert float(err) <= tol * float(want.abs().max()), float(err)

        # The next projection's fp8 input: codes of the same norm.
        codes, scale, h = layers.add_rms_norm_fp8(x, r, w["n2"])
        n, h2 = layers.add_rms_norm(x, r, w["n2"])
        assert torch.equal(h, h2)
        back = codes.float() * scale[..., None]
        # e4m3 normal 2^-4 of the value, subnormal 2^-10 of the scale; n's own rounding.
        bound = n.float().abs() * (2.0**-4 + 2.0**-7) + scale[..., None] * 2.0**-10
        assert bool(((back - n.float()).abs() <= bound).all())


def test_a_captured_decoding_step():
    """One token for every sequence as a graph over fixed buffers, replayed
    while the sequences grow, with eager work between the replays."""
    B, size, dtype = 4, 200, torch.bfloat16
    w = weights(dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.zeros(B, 1, WIDTH, device="cuda", dtype=dtype) for _ in range(2))
    length = torch.tensor([3, 0, 120, 64], device="cuda", dtype=torch.int32)
    captured, eager = Cache(B, size, dtype), Cache(B, size, dtype)
    captured.k.normal_(generator=g), captured.v.normal_(generator=g)
    eager.k.copy_(captured.k), eager.v.copy_(captured.v)

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            serve(w, captured, x, r, length)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = serve(w, captured, x, r, length)
        captured.k.copy_(eager.k), captured.v.copy_(eager.v)
        for _ in range(6):
            x.normal_(generator=g), r.normal_(generator=g)
            graph.replay()
            want = serve(w, eager, x, r, length)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            assert torch.equal(captured.k, eager.k) and torch.equal(captured.v, eager.v)
            length += 1


def test_a_captured_training_step():
    """Forward and backward of the block as a graph (no eager graph of the same
    leaves alive), replayed with new inputs and eager steps between."""
    B, L, dtype = 2, 200, torch.bfloat16
    w = weights(dtype)
    g = torch.Generator(device="cuda").manual_seed(4)
    lo, hi = A.document_windows(torch.tensor([0, 90, 180], device="cuda"), L, causal=True, prefix_lengths=8)
    tables = rope.build_position_tables(torch.arange(L, device="cuda") - lo, rotary_dim=ROT)
    x, r, dn, dh = (torch.zeros(B, L, WIDTH, device="cuda", dtype=dtype) for _ in range(4))

    def step():
        leaves = {n: t.detach().requires_grad_(True) for n, t in dict(w, x=x, r=r).items()}
        n, h = block(leaves, leaves["x"], leaves["r"], tables, lo, hi)
        return (n.detach(), h.detach()) + torch.autograd.grad((n, h), list(leaves.values()), (dn, dh))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        for t in (x, r, dn, dh):
            t.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)
