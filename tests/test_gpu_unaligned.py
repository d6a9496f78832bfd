"""Contiguous tensors that start between two aligned addresses (a slice of a flat
buffer): the same values as aligned ones, from attention, rotation and q/k norm."""

from __future__ import annotations

import math

import pytest
import torch

from avgen_amd import attention as A
from avgen_amd import layers, rope

pytestmark = pytest.mark.gpu


def aligned(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def moved(t):
    n = math.prod(t.shape)
    flat = torch.empty(n + 1, device="cuda", dtype=t.dtype)
    flat[1:] = t.reshape(-1)
    return flat[1:].view(t.shape)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L", [1, 7, 130])
@pytest.mark.parametrize("name", ["scored", "few", "plain", "windowed", "norm and rotation", "rotation"])
def test_unaligned_is_the_same(name, L, dtype):
    shape = (1, 1 if L == 1 else 4, L, 64)
    lo, hi = torch.zeros(L, device="cuda", dtype=torch.int32), torch.arange(1, L + 1, device="cuda", dtype=torch.int32)
    tables = rope.build_position_tables(torch.arange(L, device="cuda"), rotary_dim=64)
    w = aligned((64,), dtype, 9)
    call = {
        "scored": lambda q, k, v: A.scored_attention(q, k, v, softcap=5.0),
        "few": lambda q, k, v: A.scored_attention(q[:, :, :1], k, v, softcap=5.0),
        "plain": lambda q, k, v: A.attention(q, k, v),
        "windowed": lambda q, k, v: A.windowed_attention(q, k, v, lo, hi),
        "norm and rotation": lambda q, k, v: layers.qk_norm_rope(q, w, tables=tables) + layers.qk_norm_rope(k, w) + v,
        "rotation": lambda q, k, v: sum(rope.rotate_query_key(q, k, tables, layout="half")) + rope.apply_rotary(v, tables),
    }[name]
    x = [aligned(shape, dtype, n) for n in range(4)]
    results = []
    for arrange in (lambda t: t, moved):
        q, k, v, do = (arrange(t) for t in x)
        assert (q.data_ptr() % 16 != 0) == (arrange is moved)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = call(*leaves)
        results.append((out,) + torch.autograd.grad(out, leaves, do[:, :, :out.shape[2]]))
    for a, b in zip(*results):
        assert torch.equal(a, b)
