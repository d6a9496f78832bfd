"""Rotation of more tokens, and residual norm over wider rows, than one launch
of a thread group each can hold."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import layers, rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout, D", [("half", 258), ("interleaved", 258)])
def test_rotation_of_many_tokens(layout, D):
    """2^24 + 77 tokens of one head, a workgroup each (8.7 GB)."""
    B = (1 << 24) + 77
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((B, 1, 1, D), device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    k = x[:, :, :, :].expand(-1, 2, -1, -1) if layout == "half" else None
    tables = rope.build_position_tables(torch.tensor([123_457], device="cuda"), rotary_dim=D)
    half = 1 << 23
    if k is None:
        out = rope.rotate_heads(x, tables, layout=layout)
        for a in range(0, B, half):
            assert torch.equal(out[a:a + half], rope.rotate_heads(x[a:a + half], tables, layout=layout))
    else:
        out, both = rope.rotate_query_key(x, k, tables, layout=layout)
        for a in range(0, B, half):
            one, two = rope.rotate_query_key(x[a:a + half], k[a:a + half], tables, layout=layout)
            assert torch.equal(out[a:a + half], one) and torch.equal(both[a:a + half], two)


def test_tables_of_many_tokens_in_the_rotation():
    """2^24 + 9 positions in two batch rows of their own tables: the tokens on
    both sides of a launch's last one take their own rows."""
    L = (1 << 23) + 9
    D = 516
    x = torch.zeros((2, 1, 1, D), device="cuda", dtype=torch.bfloat16)
    x[..., :2] = 1.0
    x = x.expand(2, 1, L, D)
    positions = torch.stack([torch.arange(L, device="cuda") % 4096, torch.arange(L, device="cuda") % 4096 + 7])
    tables = rope.build_position_tables(positions, rotary_dim=2)
    out = rope.rotate_heads(x, tables)
    c, s = tables.cos[..., 0], tables.sin[..., 0]
    assert torch.equal(out[..., 0], (c - s).bfloat16()) and torch.equal(out[..., 1], (s + c).bfloat16())
    assert not out[..., 2:].any()


def test_residual_norm_backward_of_wide_rows():
    """One row of 2^29 + 8 values: more columns than the threads of a launch."""
    W = (1 << 29) + 8
    x = torch.zeros((1, W), device="cuda", dtype=torch.bfloat16)
    x[0, ::3] = 1.0
    r = torch.zeros((1, 1), device="cuda", dtype=torch.bfloat16).expand(1, W)
    w = torch.ones(W, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    n, h = layers.add_rms_norm(x, r, w)
    dn = torch.zeros((1, W), device="cuda", dtype=torch.bfloat16)
    dn[0, 0] = 1.0
    dn[0, -1] = 4.0  # W - 1 = 3 m: a value of 1
    dn[0, -2] = 2.0  # a value of 0
    (dw,) = torch.autograd.grad(n, (w,), dn)
    # Every third value is 1: rstd = sqrt(W / ceil(W / 3)) = sqrt(3) to 1e-8.
    assert (W - 1) % 3 == 0
    want = torch.tensor([3.0**0.5, 0.0, 0.0, 4 * 3.0**0.5])
    got = torch.stack([dw[0], dw[1], dw[-2], dw[-1]]).float().cpu()
    # A bf16 rounding of the gradient, and sums of 2^29 / 3 ones in float32 partial sums.
    assert bool(((got - want).abs() <= (2.0**-8 + 2.0**-12) * want).all())
    assert int((dw != 0).sum()) == 2
