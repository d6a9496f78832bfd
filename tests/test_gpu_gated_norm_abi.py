"""The gated residual step through its C entry points, with what the package never
passes."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import _lib
from tests.test_gpu_gated_norm import EPS, check_backward, inputs

pytestmark = pytest.mark.gpu

B16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("at", [0, 1, 4])
@pytest.mark.parametrize("W", [64, 520, 2560])
def test_modulation_gradients_at_any_element(W, at, post, dtype):
    """dgate, dscale and dshift of a row per token as parts of one buffer that begins
    `at` elements behind an aligned address."""
    n = 11
    st = inputs((n,), W, dtype, "token", post, True, seed=W + at)
    lib, f32 = _lib.load(), dtype is F32
    stream = torch.cuda.current_stream().cuda_stream
    gate, scale, shift = st["gate"], st["scale"], st["shift"]  # pieces of a projection: 3 W apart
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    vectors = (ptr(st["w"]), f32, ptr(st["p"]), f32, ptr(gate), 3 * W, ptr(scale), 3 * W, ptr(shift), 3 * W, f32)
    total, norm, dx, dr = (torch.empty(n, W, dtype=dtype, device="cuda") for _ in range(4))
    stats = torch.empty(n, 2, device="cuda")
    _lib.check(lib.avattn_gated_add_rms_norm(
        ptr(st["x"]), W, ptr(st["r"]), W, *vectors, n, W, 1, f32, 0.5, EPS, ptr(total), ptr(norm), ptr(stats), stream),
        "forward")
    flat = torch.full((at + 3 * n * W + 8,), 7.0, dtype=dtype, device="cuda")
    dg, ds, dt = flat[at:at + 3 * n * W].view(3, n, W).unbind(0)
    dw, dp = torch.empty(W, dtype=dtype, device="cuda"), torch.empty(W, dtype=dtype, device="cuda")
    size = lib.avattn_gated_add_rms_norm_bwd_workspace_size(n, W, 1, 1)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    _lib.check(lib.avattn_gated_add_rms_norm_bwd(
        ptr(st["dn"]), W, ptr(st["dh"]), W, ptr(st["x"]), W, ptr(st["r"]), W, ptr(stats), *vectors, n, W, 1, f32, 0.5,
        EPS, ptr(dx), ptr(dr), ptr(dw), ptr(dp) if post else None, ptr(dg), ptr(ds), ptr(dt), ptr(ws), size, stream),
        "backward")
    grads = {"x": dx, "r": dr, "w": dw, "gate": dg, "scale": ds, "shift": dt}
    if post:
        grads["p"] = dp
    check_backward(st, 0.5, grads)
    assert bool((flat[:at] == 7.0).all() and (flat[at + 3 * n * W:] == 7.0).all())
