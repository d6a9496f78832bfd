"""Residual addition + RMS norm on the GPU against float64.

Tolerances.  u = eps / 2 of the outputs' type is the one rounding of each
stored value; the fp32 arithmetic before it adds at most ``slack(W)``: a sum of
W squares in at most W/64 + 16 additions per thread, half of which reaches
1/sqrt, plus a dozen elementwise operations, each 2^-24.
"""

from __future__ import annotations

import pytest
import torch

from avgen_amd import layers

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def slack(W):
    return (W / 64 + 40) * 2.0**-24


def _inputs(shape, dtype, seed=0, wdtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda").to(dtype)
    r = (3 * torch.randn(shape, generator=g, device="cuda")).to(dtype)
    w = (1 + 0.3 * torch.randn(shape[-1:], generator=g, device="cuda")).to(wdtype or dtype)
    return x, r, w


def _norm64(h, w, eps):
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * rstd * w.double(), rstd


def _grads64(h, w, eps, dn, dh):
    n, rstd = _norm64(h, w, eps)
    g, xh = dn.double() * w.double(), h * rstd
    m = (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - xh * m) + (0 if dh is None else dh.double())
    size = rstd * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)) + (0 if dh is None else dh.double().abs())
    flat = (-1, h.shape[-1])
    dw = (dn.double() * xh).reshape(flat).sum(0)
    dwsize = (dn.double() * xh).abs().reshape(flat).sum(0)
    return dx, size, dw, dwsize


def _check(got, want, u, rel, size=None):
    size = want.abs() if size is None else size
    err = (got.double() - want).abs()
    bound = u * want.abs() + rel * size + 1e-37
    assert bool((err <= bound * 1.0001).all()), float((err / bound).max())


WIDTHS = [1, 2, 7, 8, 64, 100, 256, 512, 513, 1000, 1024, 2560, 4096, 5120, 8192, 12288, 16384, 16392, 20000]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("W", WIDTHS)
@pytest.mark.parametrize("rows", [1, 5, 1030])
def test_forward_and_backward(W, rows, dtype):
    if rows > 1000 and W > 8192:
        rows = 600
    eps = 1e-6
    x, r, w = _inputs((rows, W), dtype, W + rows)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    n, h = layers.add_rms_norm(x, r, w, eps=eps)
    h64 = x.detach().double() + r.detach().double()
    _check(h.detach(), h64, U[dtype], 2.0**-24)
    n64, _ = _norm64(h64, w.detach(), eps)
    _check(n.detach(), n64, U[dtype], slack(W))
    g = torch.Generator(device="cuda").manual_seed(9)
    dn, dh = (torch.randn((rows, W), generator=g, device="cuda").to(dtype) for _ in range(2))
    dx, dr, dw = torch.autograd.grad((n, h), leaves, (dn, dh))
    want, size, dw64, dwsize = _grads64(h.detach().double(), w.detach(), eps, dn, dh)
    assert torch.equal(dx, dr)
    _check(dx, want, U[dtype], 4 * slack(W), size)
    _check(dw, dw64, U[dtype], slack(W) + (rows + 64) * 2.0**-24, dwsize)


@pytest.mark.parametrize("W", [8, 100, 513, 5120, 16392])
def test_float32_gain_of_bf16_rows(W):
    x, r, w = _inputs((70, W), torch.bfloat16, 1, torch.float32)
    w.requires_grad_(True)
    n, h = layers.add_rms_norm(x, r, w)
    _check(n.detach(), _norm64(x.double() + r.double(), w.detach(), 1e-6)[0], U[torch.bfloat16], slack(W))
    dn = torch.randn_like(n)
    (dw,) = torch.autograd.grad(n, w, dn)
    assert dw.dtype is torch.float32
    _, _, dw64, dwsize = _grads64(h.double(), w.detach(), 1e-6, dn, None)
    _check(dw, dw64, U[torch.float32], slack(W) + 134 * 2.0**-24, dwsize)


def test_each_output_alone():
    x, r, w = _inputs((33, 640), torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    dn = torch.randn((33, 640), device="cuda", dtype=torch.bfloat16)
    n, h = layers.add_rms_norm(x, r, w)
    dx, dr, dw = torch.autograd.grad(n, leaves, dn)
    want, size, dw64, dwsize = _grads64(h.detach().double(), w.detach(), 1e-6, dn, None)
    _check(dx, want, U[torch.bfloat16], 4 * slack(640), size)
    _check(dw, dw64, U[torch.bfloat16], slack(640) + 97 * 2.0**-24, dwsize)
    n, h = layers.add_rms_norm(x, r, w)
    dx, dr = torch.autograd.grad(h, leaves[:2], dn)
    assert torch.equal(dx, dn) and torch.equal(dr, dn)


def test_gradient_against_differences():
    x, r, w = (t.double() for t in _inputs((3, 24), torch.float32, 5))
    gen = torch.Generator(device="cuda").manual_seed(3)
    dn, dh = (torch.randn((3, 24), generator=gen, device="cuda").double() for _ in range(2))

    def loss(x, r, w):
        h = x + r
        return ((_norm64(h, w, 1e-6)[0] * dn).sum() + (h * dh).sum()).item()

    leaves = [t.float().requires_grad_(True) for t in (x, r, w)]
    n, h = layers.add_rms_norm(*leaves)
    got = torch.autograd.grad((n, h), leaves, (dn.float(), dh.float()))
    step = 1e-4  # central differences of a smooth function: error ~ step^2 = 1e-8 of its third derivative
    for k, t in enumerate((x, r, w)):
        flat = t.reshape(-1)
        for i in range(0, flat.numel(), 5):
            keep = flat[i].item()
            flat[i] = keep + step
            up = loss(x, r, w)
            flat[i] = keep - step
            down = loss(x, r, w)
            flat[i] = keep
            assert abs((up - down) / (2 * step) - got[k].reshape(-1)[i].item()) < 2e-5 * 8


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("W", [1, 7, 64, 100, 512, 1000, 2560, 5120, 16392])
@pytest.mark.parametrize("rows", [1, 6, 1100])
def test_fp8_output(W, rows, dtype):
    rows = min(rows, 8_000_000 // W)
    x, r, w = _inputs((rows, W), dtype, W * 3 + rows)
    codes, scale, h = layers.add_rms_norm_fp8(x, r, w)
    assert codes.dtype is torch.float8_e4m3fn and scale.shape == (rows,)
    n64, _ = _norm64(x.double() + r.double(), w, 1e-6)
    top = n64.abs().amax(-1) / 448
    assert bool(((scale.double() - top).abs() <= (slack(W) + 2.0**-23) * top).all())
    got = codes.float().double() * scale.double()[:, None]
    # half a step of e4m3: 2^-4 of a normal value, 2^-10 scales of a subnormal one
    bound = (2.0**-4 * n64.abs()).maximum(2.0**-10 * scale.double()[:, None]) * (1 + 20 * (slack(W) + 2.0**-22))
    assert bool(((got - n64).abs() <= bound).all())
    _check(h, x.double() + r.double(), U[dtype], 2.0**-24)


def test_fp8_rows_of_zeros_and_extremes():
    x = torch.zeros((4, 512), device="cuda")
    r = torch.zeros_like(x)
    x[1] = 1e-30  # the norm divides by sqrt(eps): tiny, still above the smallest scale
    x[2, 3] = 3e15
    w = torch.ones(512, device="cuda")
    codes, scale, h = layers.add_rms_norm_fp8(x, r, w)
    assert scale[0] == 1 and not codes[0].float().any()
    n64, _ = _norm64(x.double(), w, 1e-6)
    assert bool((codes.float().double() * scale.double()[:, None] - n64).abs().max() <= 2.0**-4 * n64.abs().max())
    assert torch.equal(codes[1].float(), torch.full((512,), 448.0, device="cuda"))
    assert torch.equal(h, x)


@pytest.mark.parametrize("fp8", [False, True])
def test_non_finite_rows_stay_in_their_rows(fp8):
    x, r, w = _inputs((9, 768), torch.bfloat16)
    x[2, 5], r[4, 700], x[6, 0] = float("nan"), float("inf"), float("-inf")
    call = layers.add_rms_norm_fp8 if fp8 else layers.add_rms_norm
    got = call(x, r, w)
    keep = [0, 1, 3, 5, 7, 8]
    clean = call(x[keep], r[keep], w)
    for a, b in zip(got, clean):
        assert torch.equal(a[keep].float(), b.float())
    assert got[0][2].float().isnan().all()
    assert got[0][4, 700].float().isnan() and got[0][6, 0].float().isnan()  # inf * 0


def test_strides_leading_dims_and_views():
    base = torch.randn((2, 3, 5, 1280), device="cuda").to(torch.bfloat16)
    w = torch.randn((640,), device="cuda").to(torch.bfloat16)
    cases = [
        (base[..., :640], base[..., 640:]),          # rows 1,280 apart
        (base[..., 1:641], base[..., 3:643]),        # rows that start off 16 bytes
        (base.transpose(0, 1)[..., :640], base.transpose(0, 1)[..., 640:]),
        (base[:1, ..., :640].expand(4, 3, 5, 640), base[0, :1, :1, 640:].expand(4, 3, 5, 640)),
        (base[0, 0, 0, :640], base[0, 0, 0, 640:]),  # one row, rank 1
        (base[..., ::2], base[..., 1::2]),           # width not contiguous
    ]
    for x, r in cases:
        n, h = layers.add_rms_norm(x, r, w)
        n2, h2 = layers.add_rms_norm(x.contiguous(), r.contiguous(), w)
        assert n.shape == x.shape and torch.equal(h, h2)
        _check(n, _norm64(x.double() + r.double(), w, 1e-6)[0], U[torch.bfloat16], slack(640))
        _check(n2, n.double(), U[torch.bfloat16] * 2, 0.0)


def test_gradient_of_broadcast_addend():
    x = torch.randn((4, 6, 256), device="cuda", requires_grad=True)
    r = torch.randn((1, 6, 256), device="cuda", requires_grad=True)
    w = torch.ones(256, device="cuda")
    n, h = layers.add_rms_norm(x, r.expand(4, 6, 256), w)
    dx, dr = torch.autograd.grad((n * 2 + h).sum(), (x, r))
    assert dr.shape == r.shape
    assert bool(((dx.sum(0, keepdim=True) - dr).abs() <= 1e-5 * dx.abs().sum(0, keepdim=True)).all())


@pytest.mark.parametrize("W", [8, 3])
def test_more_rows_than_one_launch_takes(W):
    rows = 2**21 + 5
    x, r, w = _inputs((rows, W), torch.bfloat16)
    with torch.no_grad():
        n, h = layers.add_rms_norm(x, r, w)
        codes, scale, h8 = layers.add_rms_norm_fp8(x, r, w)
    h64 = x.double() + r.double()
    n64, _ = _norm64(h64, w, 1e-6)
    _check(h, h64, U[torch.bfloat16], 2.0**-24)
    _check(n, n64, U[torch.bfloat16], slack(W))
    assert torch.equal(h, h8)
    back = codes.double() * scale.double()[:, None]
    # e4m3: half a step of the value, or of the smallest step, 2^-9 of the scale.
    bound = n64.abs() * (2.0**-4 + slack(W)) + scale.double()[:, None] * (2.0**-10 + 448 * slack(W))
    assert bool(((back - n64).abs() <= bound).all())


def test_no_rows():
    x = torch.empty((0, 640), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(640, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    n, h = layers.add_rms_norm(x, x.detach(), w)
    assert n.shape == h.shape == (0, 640)
    dx, dw = torch.autograd.grad((n, h), (x, w), (torch.empty_like(n), torch.empty_like(h)))
    assert dx.shape == (0, 640) and not dw.any()
    codes, scale, _ = layers.add_rms_norm_fp8(x.detach(), x.detach(), w.detach())
    assert codes.shape == (0, 640) and scale.shape == (0,)


def test_runs_are_bitwise_the_same_on_any_stream():
    x, r, w = _inputs((3001, 2560), torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    dn = torch.randn((3001, 2560), device="cuda", dtype=torch.bfloat16)

    def step():
        n, h = layers.add_rms_norm(*leaves)
        return (n, h) + torch.autograd.grad((n, h), leaves, (dn, dn))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_and_replayed():
    x, r, w = _inputs((65, 5120), torch.bfloat16)
    dn = torch.randn((65, 5120), device="cuda", dtype=torch.bfloat16)
    from avgen_amd import block_ops

    def step():
        n, h = layers.add_rms_norm(x, r, w)
        dx, dw = block_ops.add_rms_norm_bwd(dn, dn, h, w, 1e-6)
        return (n, h, dx, dw) + tuple(layers.add_rms_norm_fp8(x, r, w))

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for k in range(4):
            x.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, step()):
                assert torch.equal(a.float(), b.float())


def test_ops_pass_opcheck_and_compile():
    from avgen_amd import block_ops

    x, r, w = _inputs((5, 96), torch.float32)
    x.requires_grad_(True)
    torch.library.opcheck(block_ops._add_rms_norm_op, (x, r, w, 1e-6))
    torch.library.opcheck(block_ops._add_rms_norm_fp8_op, (x.detach(), r, w, 1e-6))
    fn = torch.compile(lambda a, b, c: layers.add_rms_norm(a, b, c), fullgraph=True)
    for a, b in zip(fn(x, r, w), layers.add_rms_norm(x, r, w)):
        assert torch.equal(a, b)
