"""Second derivatives and function transforms of scored attention, sequence
rotation and residual norm: what has them is right, what has not says so."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import attention as A
from avgen_amd import layers, rope

pytestmark = pytest.mark.gpu


def normal(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda")


def attend(q, k, v):
    return A.scored_attention(q, k, v, softcap=5.0, distance_slopes=torch.full((2,), 0.1, device="cuda"))


def norm(x, r, w):
    return layers.add_rms_norm(x, r, w)[0]


QKV = [(1, 2, 9, 64)] * 3
NORM = [(7, 40), (7, 40), (40,)]


@pytest.mark.parametrize("fn, shapes", [(attend, QKV), (norm, NORM)], ids=["scored", "norm"])
def test_no_second_derivative(fn, shapes):
    leaves = [normal(s, n).requires_grad_(True) for n, s in enumerate(shapes)]
    out = fn(*leaves)
    first = torch.autograd.grad((out * out.detach()).sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="autograd"):
        torch.autograd.grad(sum(g.square().sum() for g in first), leaves)


def test_second_derivative_of_the_rotation():
    """Linear: the gradient of |R^T g|^2 / 2 by g is R R^T g = g."""
    tables = rope.build_position_tables(torch.arange(9, device="cuda"), rotary_dim=32)
    x, g = normal((1, 2, 9, 64), 0).requires_grad_(True), normal((1, 2, 9, 64), 1).requires_grad_(True)
    (dx,) = torch.autograd.grad(rope.rotate_heads(x, tables), (x,), g, create_graph=True)
    (back,) = torch.autograd.grad(dx.square().sum() / 2, (g,))
    # Two rotations of float32: a few roundings of values of about 4.
    assert bool(((back - g).abs() <= 8 * 2.0**-24 * 8).all())


@pytest.mark.parametrize("fn, shapes", [
    (attend, QKV), (norm, NORM),
    (lambda x: rope.rotate_heads(x, rope.build_position_tables(torch.arange(9, device="cuda"), rotary_dim=32)),
     [(1, 2, 9, 64)]),
], ids=["scored", "norm", "rotation"])
def test_vmap_is_one_call_each(fn, shapes):
    many = [normal((3, *s), n) for n, s in enumerate(shapes)]
    got = torch.vmap(fn)(*many)
    assert torch.equal(got, torch.stack([fn(*(t[n] for t in many)) for n in range(3)]))
