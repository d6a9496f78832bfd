"""Distance biases far from zero on the GPU against dense float64: positions
up to 2^30 from the keys, and slopes that favour the farthest of many keys.

The tolerances are those of ``test_gpu_scored``: there every probability may
be off by ``DP`` relatively, for scores of size up to 30.  The softmax does not
change when a row's scores are all moved, so neither may its error: what
counts is how far a key lies from the row's nearest (slope >= 0) or farthest
(slope < 0) one.  At x = slope times that distance, float32 rounds the score by
up to (30 + x) 2^-24 twice, and P is at most e^(30 - x) of the largest:
x <= 60 wherever P is above 2^-43, 180 * 2^-24 = 1.1e-5 in all, a twentieth of
``DP``.
"""

from __future__ import annotations

import math

import pytest
import torch

from avgen_amd import attention as A
from avgen_amd import scored_ops

from .test_gpu_scored import Oracle, make, windows

pytestmark = pytest.mark.gpu

FAR = [1_000_003, (1 << 24) + 13, 1 << 30, -(1 << 26) - 3]
KINDS = ["none", "sliding", "documents", "both"]


def slopes_of(Hq, sign):
    """Slopes of 1/64 to 3/4, of one sign or both."""
    s = torch.tensor([(1 + 47 * h / max(1, Hq - 1)) / 64 for h in range(Hq)], device="cuda")
    return s * (torch.tensor([1.0, -1.0], device="cuda").repeat(Hq)[:Hq] if sign == 0 else sign)


def check(shape, dtype, slopes, offset, lo, hi, mask, cap=None, backward=True, **kw):
    q, k, v, do = make(*shape, dtype, seed=shape[3] + shape[4])
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = A.scored_attention(*leaves, softcap=cap, distance_slopes=slopes, query_offset=offset, window_lo=lo,
                             window_hi=hi, attn_mask=None if mask is None else mask[:, None, None], enable_gqa=True,
                             **kw)
    o = Oracle(*(t.detach() for t in leaves), do, cap, slopes, offset, lo, hi, mask)
    o.check(out=out.detach())
    if backward:
        grads = torch.autograd.grad(out, leaves, do)
        o.check(dq=grads[0], dk=grads[1], dv=grads[2])
    return o, leaves


SHAPES = {
    torch.bfloat16: [(2, 4, 2, 3, 333, 64), (1, 4, 2, 70, 130, 128), (1, 36, 18, 515, 520, 64),
                     (1, 8, 8, 400, 2100, 128), (1, 4, 4, 1000, 2500, 128)],
    torch.float32: [(2, 4, 2, 3, 333, 64), (1, 8, 2, 1, 1000, 128), (1, 8, 8, 260, 512, 64), (2, 10, 5, 300, 333, 128)],
}
ALL = [(t, s) for t, shapes in SHAPES.items() for s in shapes]


@pytest.mark.parametrize("dtype, shape", ALL, ids=str)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("offset", FAR)
@pytest.mark.parametrize("sign", [1, -1, 0])
def test_far_positions(dtype, shape, kind, offset, sign):
    B, Hq, Hkv, Lq, Lk, D = shape
    lo, hi, mask = windows(kind, B, Lq, Lk)
    check(shape, dtype, slopes_of(Hq, sign), offset, lo, hi, mask,
          20.0 if (FAR.index(offset) + KINDS.index(kind)) % 2 else None)


@pytest.mark.parametrize("dtype, shape", ALL, ids=str)
@pytest.mark.parametrize("sign", [1, -1, 0])
def test_offsets_of_their_own(dtype, shape, sign):
    """Each batch row far off in a way of its own, some rows inside."""
    B, Hq, Hkv, Lq, Lk, D = shape
    offset = torch.tensor([(1 << 27) + 1, -5][:B], device="cuda", dtype=torch.int32)
    lo, hi, mask = windows("both", B, Lq, Lk)
    check(shape, dtype, slopes_of(Hq, sign), offset, lo, hi, mask, 9.0)


@pytest.mark.parametrize("dtype, shape", [
    (torch.bfloat16, (1, 4, 2, 3, 100_000, 64)), (torch.bfloat16, (1, 2, 2, 160, 100_000, 64)),
    (torch.bfloat16, (1, 2, 1, 300, 50_000, 128)), (torch.float32, (1, 4, 2, 3, 100_000, 64)),
    (torch.float32, (1, 2, 2, 160, 100_000, 64)), (torch.float32, (1, 2, 1, 300, 50_000, 128)),
], ids=str)
@pytest.mark.parametrize("where", ["inside", "end"])
@pytest.mark.parametrize("kind", ["none", "sliding", "padded"])
@pytest.mark.parametrize("sign", [-1, 0])
def test_farthest_of_many_keys(dtype, shape, where, kind, sign):
    """Slopes below zero: what counts lies at the far end of the keys."""
    B, Hq, Hkv, Lq, Lk, D = shape
    lo = hi = mask = None
    if kind == "sliding":
        i = torch.arange(Lq, device="cuda")
        lo, hi = (10 + 3 * i).int(), (Lk - 2000 + i).int()
    if kind == "padded":  # far beyond the last key that counts, and before the first
        mask = torch.zeros((B, Lk), dtype=torch.bool, device="cuda")
        mask[:, 77:Lk // 5] = True
    offset = (Lk // 10 if kind == "padded" else Lk // 2) if where == "inside" else Lk - Lq
    check(shape, dtype, slopes_of(Hq, sign), offset, lo, hi, mask)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq", [2, 300])
@pytest.mark.parametrize("sign", [1, -1])
def test_logsumexp_is_that_of_the_scores(Lq, sign, dtype):
    """The lse of the ops holds the bias whole, in float32."""
    B, Hq, Hkv, Lk, D = 2, 40, 20, 400, 64
    q, k, v, _ = make(B, Hq, Hkv, Lq, Lk, D, dtype)
    lo, hi, mask = windows("both", B, Lq, Lk)
    for offset in (0, 1 << 20, 1 << 30, -(1 << 25)):
        out, lse = scored_ops.flash_fwd_scored(q, k, v, lo, hi, mask, slopes_of(Hq, sign), None, 1 / math.sqrt(D), 7.0,
                                               offset)
        o = Oracle(q, k, v, None, 7.0, slopes_of(Hq, sign), offset, lo, hi, mask)
        o.check(out=out)
        o.check_lse(lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_far_offset_is_a_constant(dtype):
    """Without windows, queries behind all keys: any two offsets give the same
    attention (the bias moves by a constant per row)."""
    q, k, v, do = make(1, 20, 20, 300, 700, 64, dtype)
    got = []
    for offset in (700, 1 << 22, (1 << 30) - 1):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = A.scored_attention(*leaves, distance_slopes=slopes_of(20, 1), query_offset=offset)
        got.append((out,) + torch.autograd.grad(out, leaves, do))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_compiled_call_far_away(dtype):
    shape = (1, 4, 2, 70, 130, 64)
    q, k, v, do = make(*shape, dtype)
    slopes = slopes_of(4, 0)
    fn = torch.compile(lambda a, b, c: A.scored_attention(a, b, c, distance_slopes=slopes, query_offset=(1 << 26) + 5,
                                                          enable_gqa=True), fullgraph=True)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = fn(*leaves)
    grads = torch.autograd.grad(out, leaves, do)
    o = Oracle(*(t.detach() for t in leaves), do, None, slopes, (1 << 26) + 5)
    o.check(out=out.detach(), dq=grads[0], dk=grads[1], dv=grads[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Lq, Hq, Hkv", [(3, 4, 2), (300, 40, 20)])
@pytest.mark.parametrize("sign", [1, -1, 0])
def test_ops_with_and_without_the_row_statistic(Lq, Hq, Hkv, sign, dtype):
    """``flash_bwd_scored`` from ``row_lse`` and from ``lse`` alone, which near by
    holds the bias exactly enough: relative errors of up to |lse| 2^-24, |lse| <
    0.75 * 400 + 30, 2e-5 in all, a tenth of ``DP``."""
    B, Lk, D = 2, 400, 64
    q, k, v, do = make(B, Hq, Hkv, Lq, Lk, D, dtype)
    lo, hi, mask = windows("both", B, Lq, Lk)
    slopes = slopes_of(Hq, sign)
    args = (lo, hi, mask, slopes, None, 1 / math.sqrt(D), 7.0, 50, True)
    out, lse, row_lse = scored_ops._fwd_rows_op(q, k, v, *args)
    assert torch.equal(out, scored_ops.flash_fwd_scored(q, k, v, *args)[0])
    o = Oracle(q, k, v, do, 7.0, slopes, 50, lo, hi, mask)
    o.check(out=out)
    o.check_lse(lse)
    for stat in (row_lse, None):
        dq, dk, dv = scored_ops.flash_bwd_scored(do, q, k, v, out, lse, *args, stat)
        o.check(dq=dq, dk=dk, dv=dv)


def test_row_statistic_op_passes_opcheck():
    q, k, v, _ = make(1, 2, 1, 9, 12, 64, torch.float32)
    q.requires_grad_(True)
    lo, hi, _ = windows("causal", 1, 9, 12)
    torch.library.opcheck(scored_ops._fwd_rows_op, (q, k, v, lo, hi, None, slopes_of(2, 0), None, 0.125, 5.0, 3, True))


def test_captured_far_away():
    """A training step of far positions, captured and replayed with new inputs."""
    q, k, v, do = make(1, 20, 20, 150, 300, 64, torch.bfloat16)
    offset = torch.tensor([1 << 26], device="cuda", dtype=torch.int32)
    slopes = slopes_of(20, 0)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        out = A.scored_attention(*leaves, softcap=9.0, distance_slopes=slopes, query_offset=offset)
        return (out.detach(),) + torch.autograd.grad(out, leaves, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for n in range(3):
        with torch.no_grad():
            q.copy_(torch.randn_like(q))
            offset.fill_((1 << 25) + 1000 * n if n else 100)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)
