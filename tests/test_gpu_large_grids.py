"""Rotation of more tokens than one launch can hold."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import rope

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
