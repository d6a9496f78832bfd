"""The gated residual step where a vector is not finite in one column: the columns
of a row are each other's only through the row's sums."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import layers

pytestmark = pytest.mark.gpu

B16, F32 = torch.bfloat16, torch.float32
INF = float("inf")

# Widths whose last threads have no column (several rows a wave, one, workgroups of
# every size, off the 16-byte grid), that fill their threads, and of any width.
WIDTHS = [5, 40, 129, 520, 777, 1152, 2560, 5120, 6152, 8200, 12296, 20001]


def rows(n, W, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x, r, d, e = (torch.randn(2, n, W, generator=g, device="cuda").to(dtype) for _ in range(4))
    return x, r, d, e


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("which", ["gate", "post_weight", "token gate"])
@pytest.mark.parametrize("W", WIDTHS)
def test_an_infinite_gate_stays_in_its_column(W, which, dtype):
    """h is infinite in column 0, so the row's factor is 0: the other columns of the norm
    are the shift, those of the sum as ever."""
    x, r, _, _ = rows(3, W, dtype, W)
    x[..., 0] = 1.0
    v = torch.ones((2, 3, W) if which == "token gate" else (W,), device="cuda", dtype=dtype)
    more = {which.split()[-1]: v}
    _, plain = layers.gated_add_rms_norm(x, r, **more)
    v[..., 0] = INF
    shift = torch.full_like(v, 0.5)
    n, h = layers.gated_add_rms_norm(x, r, shift=shift, **more)
    assert bool((n[..., 1:] == 0.5).all()) and bool(n[..., 0].isnan().all())
    assert torch.equal(h[..., 1:], plain[..., 1:]) and bool((h[..., 0] == INF).all())


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("W", WIDTHS)
def test_an_infinite_scale_in_the_backward(W, per_row, dtype):
    """With weight (1 + scale) infinite in column 0 and h positive there, A h dn is +-inf in
    that column and m with it; d is -+inf in every other column, of the sign that -h m
    has.  No column is NaN but the first, whose terms cancel."""
    x, r, dn, dh = rows(3, W, dtype, W + 1)
    x, r, dn = x.abs() + 1, r.abs() + 1, dn.abs() + 1
    scale = torch.zeros((2, 3, W) if per_row else (W,), device="cuda", dtype=dtype)
    scale[..., 0] = INF
    leaves = [t.detach().requires_grad_(True) for t in (x, r)]
    n, h = layers.gated_add_rms_norm(*leaves, scale=scale)
    dx, dr = torch.autograd.grad((n, h), leaves, (dn, dh))
    assert bool((n[..., 0] == INF).all()) and bool(n[..., 1:].isfinite().all())
    for d in (dx, dr):
        assert bool(d[..., 0].isnan().all()) and bool((d[..., 1:] == -INF).all())
