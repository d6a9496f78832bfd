"""What the fake forms of the ops promise a compiled graph is what the real
ones return, strides included, for inputs in any layout."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import attention as A
from avgen_amd import block_ops, layers, rope, scored_ops

pytestmark = pytest.mark.gpu

B16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def compiled_anew():
    """Each test compiles its calls for itself."""
    torch._dynamo.reset()


def laid(shape, dtype, how, seed=0):
    """Random values of ``shape (batch, heads, length, channels)`` in a layout."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, L, D = shape
    t = torch.randn(shape, generator=g, device="cuda").to(dtype)
    if how == "contiguous":
        return t
    if how == "tokens":  # (B, L, H, D)
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "channels outside":  # the last dimension strided
        return t.transpose(2, 3).contiguous().transpose(2, 3)
    if how == "channels and heads swapped":
        return t.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    if how == "every second":  # gaps
        wide = torch.zeros((B, H, L, 2 * D), device="cuda", dtype=dtype)
        wide[..., ::2] = t
        return wide[..., ::2]
    if how == "unaligned":
        wide = torch.zeros((B, H, L, D + 1), device="cuda", dtype=dtype)
        wide[..., 1:] = t
        return wide[..., 1:]
    if how == "shared heads":
        return t[:, :1].expand(shape)
    raise AssertionError(how)


LAYOUTS = ["contiguous", "tokens", "channels outside", "channels and heads swapped", "every second", "unaligned",
           "shared heads"]


def promised(op, args):
    """The strides of the op's fake outputs."""
    from torch._subclasses import FakeTensorMode

    with FakeTensorMode() as mode:
        fakes = [mode.from_tensor(a) if isinstance(a, torch.Tensor) else a for a in args]
        outs = op(*fakes)
    return [(tuple(o.shape), o.stride(), o.dtype) for o in (outs if isinstance(outs, (tuple, list)) else (outs,))]


def returned(op, args):
    outs = op(*args)
    return [(tuple(o.shape), o.stride(), o.dtype) for o in (outs if isinstance(outs, (tuple, list)) else (outs,))]


def tables(L, pairs):
    return rope.build_position_tables(torch.arange(L, device="cuda"), rotary_dim=2 * pairs)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("how", LAYOUTS)
def test_rotation(how, dtype):
    q, k = laid((2, 3, 5, 64), dtype, how), laid((2, 2, 5, 64), dtype, how, 1)
    t = tables(5, 32)
    args = (q, t.cos, t.sin, 0, True, False)
    assert returned(block_ops._rotate_op, args) == promised(block_ops._rotate_op, args)
    args = (q, k, t.cos, t.sin, 0, True, False)
    assert returned(block_ops._rotate_pair_op, args) == promised(block_ops._rotate_pair_op, args)
    fn = torch.compile(lambda a, b: rope.rotate_query_key(a, b, t, layout="half"), fullgraph=True)
    for got, want in zip(fn(q, k), rope.rotate_query_key(q.contiguous(), k.contiguous(), t, layout="half")):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("how", LAYOUTS)
@pytest.mark.parametrize("Lq", [3, 200])
@pytest.mark.parametrize("slopes", [False, True])
def test_scored_attention(how, dtype, Lq, slopes):
    q, k, v, do = (laid((2, h, n, 64), dtype, how, s) for s, (h, n) in enumerate(((4, Lq), (2, 150), (2, 150), (4, Lq))))
    s = torch.tensor([0.5, 0.25, 0.1, 0.01], device="cuda") if slopes else None
    args = (q, k, v, None, None, None, s, None, 0.125, 5.0, 0, True)
    assert returned(scored_ops._fwd_op, args) == promised(scored_ops._fwd_op, args)
    out, lse = scored_ops._fwd_op(*args)
    back = (do, q, k, v, out, lse, None, None, None, s, None, 0.125, 5.0, 0, True)
    assert returned(scored_ops._bwd_op, back) == promised(scored_ops._bwd_op, back)

    def step(q, k, v):
        return A.scored_attention(q, k, v, softcap=5.0, distance_slopes=s, enable_gqa=True)

    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    plain = [t.detach().contiguous().requires_grad_(True) for t in (q, k, v)]
    got, want = torch.compile(step, fullgraph=True)(*leaves), step(*plain)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, do), torch.autograd.grad(want, plain, do)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("how", LAYOUTS)
def test_residual_norm(how, dtype):
    x, r = laid((2, 3, 5, 64), dtype, how), laid((2, 3, 5, 64), dtype, how, 1)
    w = torch.ones(64, device="cuda", dtype=dtype)
    for op, args in ((block_ops._add_rms_norm_op, (x, r, w, 1e-6)), (block_ops._add_rms_norm_fp8_op, (x, r, w, 1e-6)),
                     (block_ops._add_rms_norm_bwd_op, (x, r, x, w, 1e-6))):
        assert returned(op, args) == promised(op, args)
    n, h = torch.compile(lambda a, b: layers.add_rms_norm(a, b, w), fullgraph=True)(x, r)
    for got, want in zip((n, h), layers.add_rms_norm(x, r, w)):
        assert torch.equal(got, want)
