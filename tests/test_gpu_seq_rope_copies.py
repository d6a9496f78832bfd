"""Rotation of inputs that have to be copied first: every copy lives until the
launch that reads it."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import block_ops, rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("Hq, Hk", [(3, 3), (3, 2), (1, 4), (8, 1)])
@pytest.mark.parametrize("L", [5, 300])
def test_query_and_key_with_strided_channels(L, Hq, Hk, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(L)
    wide = [torch.randn((2, h, L, 128), generator=g, device="cuda").to(dtype) for h in (Hq, Hk, Hq, Hk)]
    q, k, dq, dk = (t[..., ::2] for t in wide)
    tables = rope.build_position_tables(torch.arange(L, device="cuda"), rotary_dim=64)

    def step(q, k, dq, dk):
        q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        out = rope.rotate_query_key(q, k, tables, layout=layout)
        return out + torch.autograd.grad(out, (q, k), (dq, dk))

    want = step(*(t.contiguous() for t in (q, k, dq, dk)))
    for _ in range(3):
        for a, b in zip(step(q, k, dq, dk), want):
            assert torch.equal(a, b)
    one = block_ops._rotate_pair_op(q, k, tables.cos, tables.sin, 0, layout == "half", False)
    assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[1])
