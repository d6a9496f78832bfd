"""Sizes of one, whose strides mean nothing, on the GPU: any of them will do."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import attention as A
from avgen_amd import layers, rope

pytestmark = pytest.mark.gpu

B16, F32 = torch.bfloat16, torch.float32


def normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def odd(t, dim, stride):
    """``t``, of size 1 in ``dim``, with another stride there."""
    strides = list(t.stride())
    strides[dim] = stride
    return t.as_strided(t.shape, strides)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("Lq, heads", [(1, 4), (1, 300), (150, 4), (200, 160)])
def test_strides_of_sizes_of_one(Lq, heads, dtype):
    """A batch of one, one head or one row, with strides that no kernel could
    step by: they are never stepped by."""
    q, k, v, do = (normal((1, h, n, 64), dtype, s)
                   for s, (h, n) in enumerate(((heads, Lq), (1, 170), (1, 170), (heads, Lq))))
    results = []
    for change in (lambda t: t, lambda t: odd(odd(t, 0, 12_345), 1, 777) if t.shape[1] == 1 else odd(t, 0, 12_345)):
        a = [change(t) for t in (q, k, v, do)]
        if Lq == 1 and change(q) is not q:
            a[0], a[3] = odd(a[0], 2, 67), odd(a[3], 2, 67)
        leaves = [t.detach().requires_grad_(True) for t in a[:3]]
        out = A.scored_attention(*leaves, softcap=5.0, enable_gqa=True)
        results.append((out,) + torch.autograd.grad(out, leaves, a[3]))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [B16, F32])
def test_one_key_of_any_row_stride(dtype):
    """The one row of k and v of rows that lie far apart."""
    q, k, v, do = (normal((1, 4, n, 64), dtype, s) for s, n in enumerate((3, 1, 1, 3)))
    results = []
    for far in (False, True):
        a = [odd(t, 2, 1 << 24) if far else t for t in (k, v)]
        leaves = [t.detach().requires_grad_(True) for t in (q, *a)]
        out = A.scored_attention(*leaves, softcap=5.0)
        results.append((out,) + torch.autograd.grad(out, leaves, do))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [B16, F32])
def test_strides_of_sizes_of_one_in_plain_attention(dtype):
    q, k, v, do = (normal((1, 4, 90, 64), dtype, s) for s in range(4))
    results = []
    for a in ([q, k, v, do], [odd(t, 0, 12_345) for t in (q, k, v, do)]):
        leaves = [t.detach().requires_grad_(True) for t in a[:3]]
        out = A.attention(*leaves)
        results.append((out,) + torch.autograd.grad(out, leaves, a[3]))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [B16, F32])
def test_strides_of_sizes_of_one_in_norm_and_rotation(dtype):
    x, dy = normal((1, 4, 90, 64), dtype, 0), normal((1, 4, 90, 64), dtype, 1)
    w = torch.ones(64, device="cuda", dtype=dtype)
    tables = rope.build_position_tables(torch.arange(90, device="cuda"), rotary_dim=64)
    results = []
    for t in (x, odd(x, 0, 12_345)):
        t = t.detach().requires_grad_(True)
        y = layers.qk_norm_rope(t, w, tables=tables)
        z = rope.apply_rotary(t, tables)
        results.append((y, z) + torch.autograd.grad((y, z), (t,), (dy, odd(dy, 0, 12_345))))
    for a, b in zip(*results):
        assert torch.equal(a, b)
