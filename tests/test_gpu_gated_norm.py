"""The gated residual step with its norms against float64, and its gradients
against the formulas' and against differences."""

from __future__ import annotations

import pytest
import torch

from avgen_amd import layers

pytestmark = pytest.mark.gpu

B16, F32 = torch.bfloat16, torch.float32
UNIT = 2.0**-24
NAMES = ("x", "r", "w", "gate", "scale", "shift", "p")
EPS = 1e-6


def half(dtype):
    return torch.finfo(dtype).eps / 2


def inputs(lead, W, dtype, modulation, post, gain, seed=0, vectors=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    vectors = dtype if vectors is None else vectors

    def rand(shape, spread, middle=0.0, t=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * spread + middle).to(t)

    st = dict.fromkeys(NAMES)
    st["x"], st["r"] = rand((*lead, W), 1.0), rand((*lead, W), 3.0)
    if gain:
        st["w"] = rand((W,), 0.2, 1.0, vectors)
    if post:
        st["p"] = rand((W,), 0.2, 1.0, vectors)
    shape = {"none": None, "shared": (W,), "batch": (lead[0],) + (1,) * (len(lead) - 1) + (W,),
             "token": (*lead, W)}[modulation]
    if shape is not None:
        st["gate"], st["scale"], st["shift"] = rand((*shape[:-1], 3 * W), 0.3, 0.0, vectors).chunk(3, -1)
    st["dn"], st["dh"] = rand((*lead, W), 1.0), rand((*lead, W), 1.0)
    return st


def call(st, alpha):
    return layers.gated_add_rms_norm(st["x"], st["r"], st["w"], gate=st["gate"], scale=st["scale"], shift=st["shift"],
                                     post_weight=st["p"], residual_scale=alpha, eps=EPS)


def plain(x, r, w, gate, scale, shift, p, alpha):
    """(norm, sum) in the inputs' precision."""
    if p is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * p
    h = alpha * r + (x if gate is None else gate * x)
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    if w is not None:
        n = n * w
    if scale is not None:
        n = n * (1 + scale)
    return n if shift is None else n + shift, h


def doubles(st):
    return [None if st[n] is None else st[n].detach().double() for n in NAMES]


def close(got, want, tol, label):
    diff = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((diff <= tol).all()), f"{label}: {float((diff / tol).max()):.3f} of the tolerance"


def check_forward(st, alpha, n, h):
    dtype = st["x"].dtype
    x, r, w, gate, scale, shift, p = doubles(st)
    want_n, want_h = plain(x, r, w, gate, scale, shift, p, alpha)
    # float32: a norm's factor is off by the rounding of the sum of its squares (W
    # of them in at most W / 64 steps and a tree) and some operations, every product
    # or sum by one rounding; of the sum's two terms, by their magnitudes.
    W = x.shape[-1]
    norm = (W / 64 + 24) * UNIT
    term = want_h - alpha * r
    err_h = (norm + 4 * UNIT) * term.abs() + 3 * UNIT * ((alpha * r).abs() + want_h.abs())
    close(h, want_h, half(dtype) * want_h.abs() + err_h + 1e-37, "sum")
    rh = torch.rsqrt((want_h * want_h).mean(-1, keepdim=True) + EPS)
    factor = rh * (1 if w is None else w) * (1 if scale is None else 1 + scale)
    scaled = want_h * factor
    # An error of h changes the row's factor by its relative size at most.
    row = ((err_h * err_h).sum(-1, keepdim=True) / (want_h * want_h).sum(-1, keepdim=True).clamp(min=1e-300)).sqrt()
    err_n = err_h * factor.abs() + (norm + row + 6 * UNIT) * scaled.abs() + 2 * UNIT * want_n.abs()
    close(n, want_n, half(dtype) * want_n.abs() + err_n + 1e-37, "norm")


def check_backward(st, alpha, grads, with_dh=True):
    """Against the formulas, from the unrounded sum."""
    dtype = st["x"].dtype
    x, r, w, gate, scale, shift, p = doubles(st)
    dn = st["dn"].double()
    dh = st["dh"].double() if with_dh else torch.zeros_like(r)
    one = torch.ones((), dtype=torch.float64, device="cuda")
    g, s = one if gate is None else gate, one if scale is None else 1 + scale
    wv, pv = one if w is None else w, one if p is None else p
    W = x.shape[-1]
    rx = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) if p is not None else one
    h = alpha * r + g * (x * rx * pv)
    rh = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    nx, nh, t = x * rx, h * rh, dn * wv * s
    d = dh + rh * (t - nh * (t * nh).mean(-1, keepdim=True))
    b = d * g * pv
    dx = b if p is None else rx * (b - nx * (b * nx).mean(-1, keepdim=True))
    # float32 terms of d and dx: (a row's sums in at most W / 64 steps and a tree)
    # times the sizes of the terms; h's is that of its two terms.
    unit = (W / 64 + 32) * UNIT
    size_h = (alpha * r).abs() + (g * nx * pv).abs()
    size_n = size_h * rh
    size_d = dh.abs() + rh * (t.abs() + size_n * (t.abs() * size_n).mean(-1, keepdim=True))
    size_b = size_d * (g * pv).abs()
    size_x = size_b if p is None else rx * (size_b + nx.abs() * (size_b * nx.abs()).mean(-1, keepdim=True) * 2)
    want = {"x": (dx, unit * size_x), "r": (alpha * d, unit * size_d * abs(alpha))}

    def total_of(terms, sizes, like):
        n = terms.numel() // like.numel()
        return terms.sum_to_size(like.shape), (sizes * (unit + (n + 8) * UNIT)).sum_to_size(like.shape)

    if w is not None:
        want["w"] = total_of(dn * s * nh, (dn * s).abs() * size_n, w)
    if gate is not None:
        want["gate"] = total_of(d * nx * pv, size_d * (nx * pv).abs(), gate)
    if scale is not None:
        want["scale"] = total_of(dn * nh * wv, (dn * wv).abs() * size_n, scale)
    if shift is not None:
        want["shift"] = total_of(dn, dn.abs(), shift)
    if p is not None:
        want["p"] = total_of(d * g * nx, size_d * (g * nx).abs(), p)
    for name, got in grads.items():
        value, err = want[name]
        assert got.dtype is st[name].dtype and got.shape == st[name].shape, name
        close(got, value, half(got.dtype) * value.abs() + err + 1e-37, "gradient of " + name)


def check(lead, W, dtype, modulation, post, gain, alpha=1.0, seed=0, vectors=None, drop=()):
    st = inputs(lead, W, dtype, modulation, post, gain, seed, vectors)
    for name in drop:
        st[name] = None
    with torch.no_grad():
        check_forward(st, alpha, *call(st, alpha))
    leaves = {n: st[n].detach().requires_grad_(True) for n in NAMES if st[n] is not None}
    n, h = call({**st, **leaves}, alpha)
    grads = torch.autograd.grad((n, h), list(leaves.values()), (st["dn"], st["dh"]))
    check_backward(st, alpha, dict(zip(leaves, grads)))
    return st


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("modulation", ["none", "shared", "batch", "token"])
@pytest.mark.parametrize("lead, W", [((2, 9), 64), ((3, 130), 520), ((2, 70), 1536), ((1, 40), 5120), ((8, 1), 2560)])
def test_shapes_and_modulations(lead, W, modulation, post, dtype):
    check(lead, W, dtype, modulation, post, True)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("modulation, post", [("none", False), ("batch", True), ("token", True)])
@pytest.mark.parametrize("W", [1, 2, 7, 8, 63, 129, 1001, 4097, 8192, 9000, 16384, 16392, 20001])
def test_widths(W, modulation, post, dtype):
    check((2, 5), W, dtype, modulation, post, True)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("drop", [("gate",), ("scale",), ("shift",), ("gate", "shift"), ("scale", "shift"),
                                  ("gate", "scale")])
@pytest.mark.parametrize("modulation", ["batch", "token"])
@pytest.mark.parametrize("post, gain, alpha", [(False, False, 0.5), (True, True, -1.0), (True, False, 0.0)])
def test_some_of_the_vectors(post, gain, alpha, modulation, drop, dtype):
    check((2, 33), 256, dtype, modulation, post, gain, alpha, drop=drop)


@pytest.mark.parametrize("modulation", ["shared", "batch", "token"])
def test_float32_vectors_of_bf16_rows(modulation):
    check((2, 50), 640, B16, modulation, True, True, vectors=F32)
    check((2, 50), 641, B16, modulation, True, True, vectors=F32)


@pytest.mark.parametrize("lead", [(1,), (5,), (2, 3, 4), (1, 1), (40, 3), (700, 2), (3, 1, 5)])
@pytest.mark.parametrize("modulation", ["none", "batch", "token"])
def test_leading_dimensions(lead, modulation):
    check(lead, 128, B16, modulation, True, True)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("W", [128, 2048])
@pytest.mark.parametrize("modulation", ["none", "batch", "token"])
def test_many_rows(modulation, W, dtype):
    """Several rows per worker, forward and backward."""
    check((3, 7001), W, dtype, modulation, True, True)


def test_modulations_of_different_shapes():
    st = inputs((2, 3, 20), 96, B16, "none", False, True)
    g = torch.Generator(device="cuda").manual_seed(5)
    gate, scale, shift = ((torch.randn(s, generator=g, device="cuda") * 0.3).to(B16).requires_grad_(True)
                          for s in ((96,), (2, 3, 1, 96), (2, 1, 1, 96)))
    x, r, w = (st[n].detach().requires_grad_(True) for n in ("x", "r", "w"))
    n, h = layers.gated_add_rms_norm(x, r, w, gate=gate, scale=scale, shift=shift)
    leaves = dict(x=x, r=r, w=w, gate=gate, scale=scale, shift=shift)
    grads = dict(zip(leaves, torch.autograd.grad((n, h), list(leaves.values()), (st["dn"], st["dh"]))))
    full = {**st, "gate": gate, "scale": scale, "shift": shift}
    check_forward(full, 1.0, n, h)
    # Summed by torch from the bf16 gradients of the widest shape: a rounding of
    # each of up to six of them more.
    st32 = {k: None if v is None else v.detach().float() for k, v in full.items()}
    want = [t.detach().double().requires_grad_(True) for t in leaves.values()]
    pn, ph = plain(*want, None, 1.0)
    exact = torch.autograd.grad((pn, ph), want, (st["dn"].double(), st["dh"].double()))
    for name, e in zip(leaves, exact):
        rel = float((grads[name].double() - e).norm() / e.norm())
        # output and partial roundings: four half steps
        assert rel <= 4 * half(B16), (name, rel)
    assert st32["gate"] is not None


@pytest.mark.parametrize("which", ["norm", "sum"])
@pytest.mark.parametrize("post", [False, True])
def test_one_output_used(which, post):
    st = inputs((2, 30), 320, F32, "batch", post, True)
    leaves = {n: st[n].detach().requires_grad_(True) for n in NAMES if st[n] is not None}
    n, h = call({**st, **leaves}, 0.5)
    if which == "norm":
        grads = torch.autograd.grad(n, list(leaves.values()), st["dn"])
        check_backward(st, 0.5, dict(zip(leaves, grads)), with_dh=False)
    else:
        names = [k for k in leaves if k in ("x", "r", "gate", "p")]
        grads = torch.autograd.grad(h, [leaves[k] for k in names], st["dh"])
        st["dn"] = torch.zeros_like(st["dn"])
        check_backward(st, 0.5, dict(zip(names, grads)))


@pytest.mark.parametrize("modulation", ["none", "batch", "token"])
@pytest.mark.parametrize("post", [False, True])
def test_gradient_against_differences(post, modulation):
    """float32 gradients along a direction against central differences in float64."""
    st = inputs((2, 6), 48, F32, modulation, post, True)
    names = [n for n in NAMES if st[n] is not None]
    leaves = {n: st[n].detach().requires_grad_(True) for n in names}
    n, h = call({**st, **leaves}, 0.7)
    grads = torch.autograd.grad((n, h), list(leaves.values()), (st["dn"], st["dh"]))
    g = torch.Generator(device="cuda").manual_seed(3)
    for name, grad in zip(names, grads):
        direction = torch.randn(grad.shape, generator=g, device="cuda").double()

        def at(step):
            args = [None if st[k] is None else st[k].double() + (step * direction if k == name else 0.0) for k in NAMES]
            n, h = plain(*args, 0.7)
            return (n * st["dn"].double()).sum() + (h * st["dh"].double()).sum()

        want = float((at(1e-5) - at(-1e-5)) / 2e-5)
        # float32 roundings of some hundred terms; differences are good to 1e-9.
        size = float((grad.double() * direction).abs().sum())
        assert abs(float((grad.double() * direction).sum()) - want) <= 2e-5 * size + 1e-6, name


@pytest.mark.parametrize("dtype", [B16, F32])
def test_strides(dtype):
    """Transposed, gapped and unaligned rows, expanded vectors."""
    st = inputs((4, 10), 64, dtype, "batch", True, True)
    want = call(st, 1.0)
    x = st["x"].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(4, 10, 65, dtype=dtype, device="cuda")
    wide[..., 1:] = st["r"]
    gaps = torch.zeros(64, 2, dtype=dtype, device="cuda")
    gaps[:, 0] = st["w"]
    got = call({**st, "x": x, "r": wide[..., 1:], "w": gaps[:, 0]}, 1.0)
    for a, b in zip(got, want):
        # Value by value the sums run in another order.
        assert bool(((a.double() - b.double()).abs() <= 2 * half(dtype) * b.double().abs() + 64 * UNIT * 8).all())
    same = {**st, "gate": st["gate"][:1].expand(4, 1, 64), "scale": st["scale"][:1].expand(4, 1, 64),
            "shift": st["shift"][:1].expand(4, 1, 64)}
    shared = {**st, "gate": st["gate"][0, 0], "scale": st["scale"][0, 0], "shift": st["shift"][0, 0]}
    assert all(torch.equal(a, b) for a, b in zip(call(same, 1.0), call(shared, 1.0)))


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
def test_no_rows(lead):
    st = inputs(lead, 16, B16, "none", True, True)
    leaves = {n: st[n].detach().requires_grad_(True) for n in NAMES if st[n] is not None}
    gate = torch.ones(16, dtype=B16, device="cuda", requires_grad=True)
    n, h = call({**st, **leaves, "gate": gate}, 1.0)
    assert n.shape == h.shape == (*lead, 16)
    grads = torch.autograd.grad((n, h), [*leaves.values(), gate], (st["dn"], st["dh"]))
    assert all(bool((g == 0).all()) for g in grads)


def test_rows_of_zeros_and_what_is_not_finite():
    st = inputs((1, 4), 128, F32, "none", True, True)
    st["x"][0, 0] = 0.0
    st["r"][0, 0] = 0.0
    st["x"][0, 1, 5] = float("inf")
    st["r"][0, 2, 7] = float("nan")
    n, h = call(st, 1.0)
    assert bool((n[0, 0] == 0).all() and (h[0, 0] == 0).all())
    assert bool(n[0, 1].isnan().all() and n[0, 2].isnan().all())
    assert bool(torch.isfinite(n[0, 3]).all())


def test_same_tensor_twice_and_repeatable():
    st = inputs((3, 700), 384, B16, "batch", True, True)
    leaves = {n: st[n].detach().requires_grad_(True) for n in NAMES if st[n] is not None}

    def grads():
        n, h = call({**st, **leaves}, 1.0)
        return torch.autograd.grad((n, h), list(leaves.values()), (st["dn"], st["dh"]))

    assert all(torch.equal(a, b) for a, b in zip(grads(), grads()))
    x = st["x"].detach().requires_grad_(True)
    n, h = layers.gated_add_rms_norm(x, x, gate=st["gate"])
    (got,) = torch.autograd.grad((n, h), x, (st["dn"], st["dh"]))
    two = [st["x"].detach().requires_grad_(True) for _ in range(2)]
    n2, h2 = layers.gated_add_rms_norm(*two, gate=st["gate"])
    a, b = torch.autograd.grad((n2, h2), two, (st["dn"], st["dh"]))
    assert torch.equal(h, h2) and torch.equal(got, a + b)


@pytest.mark.parametrize("dtype", [B16, F32])
@pytest.mark.parametrize("W", [1, 5, 8, 24, 33, 64, 65, 129, 200, 257, 512, 513, 777, 1025, 2056, 4097, 6152, 8191, 8200,
                               12288, 16381, 16384, 16392])
@pytest.mark.parametrize("lead, modulation", [((3, 37), "batch"), ((1, 600), "shared"), ((2, 9), "token"),
                                              ((70, 3), "batch")])
def test_every_way_of_sharing_a_row(lead, modulation, W, dtype):
    """Several rows in a wave, one in a wave or in a workgroup of any size, with and
    without whole 16-byte chunks, and rows of any width; one workgroup and many."""
    check(lead, W, dtype, modulation, W % 3 != 0, True, 0.5, seed=W)


def test_more_workgroups_than_a_launch_takes():
    """Groups of three rows of 8 values, 2^21 + 7 of them: a workgroup each in the
    backward, in two launches."""
    groups, W = 2**21 + 7, 8
    g = torch.Generator(device="cuda").manual_seed(8)
    x, r, dn, dh = (torch.randn(groups, 3, W, generator=g, device="cuda", dtype=F32) for _ in range(4))
    gate = torch.randn(groups, 1, W, generator=g, device="cuda", dtype=F32)
    leaves = [t.requires_grad_(True) for t in (x, r, gate)]
    n, h = layers.gated_add_rms_norm(x, r, gate=gate)
    grads = torch.autograd.grad((n, h), leaves, (dn, dh))
    at = torch.tensor([0, 1, 2**20, 2**21 - 1, 2**21, groups - 1], device="cuda")
    st = dict.fromkeys(NAMES)
    st.update({k: v.detach()[at] for k, v in dict(x=x, r=r, gate=gate, dn=dn, dh=dh).items()})
    check_forward(st, 1.0, n.detach()[at], h.detach()[at])
    check_backward(st, 1.0, {k: v[at] for k, v in zip(("x", "r", "gate"), grads)})
