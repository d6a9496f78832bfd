"""Calls of the gated residual step that its documentation allows, at the edges."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_gated_norm import NAMES, call, check_backward, check_forward, inputs

pytestmark = pytest.mark.gpu

B16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("modulation", ["none", "shared", "token"])
@pytest.mark.parametrize("W", [1, 40, 2560])
def test_a_single_row_without_leading_sizes(W, modulation, dtype):
    st = inputs((1,), W, dtype, modulation, True, True, seed=W)
    st = {name: t[0] if t is not None and t.ndim > 1 else t for name, t in st.items()}
    assert st["x"].shape == (W,)
    with torch.no_grad():
        check_forward(st, 0.5, *call(st, 0.5))
    leaves = {n: st[n].detach().requires_grad_(True) for n in NAMES if st[n] is not None}
    grads = torch.autograd.grad(call({**st, **leaves}, 0.5), list(leaves.values()), (st["dn"], st["dh"]))
    check_backward(st, 0.5, dict(zip(leaves, grads)))
