"""Refusals of the block ops (rotation by positions, residual norm): every
check runs before any launch, so they are tested without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from avgen_amd import _lib, layers, rope
from avgen_amd.rope import PositionScaling, RotaryTables

T = RotaryTables(cos=torch.zeros(1, 1, 4, 8), sin=torch.zeros(1, 1, 4, 8))
X = torch.zeros(2, 3, 4, 32)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        rope.rotate_heads(X, T)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rope.build_position_tables(torch.arange(4), rotary_dim=16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.add_rms_norm(X, X, torch.zeros(32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.add_rms_norm_fp8(X, X, torch.zeros(32))


@pytest.mark.parametrize("call, error", [
    (lambda: rope.rotate_heads(X[0], T), ValueError),
    (lambda: rope.rotate_heads(X.half(), T), TypeError),
    (lambda: rope.rotate_heads(X[:, :, :3], T), ValueError),
    (lambda: rope.rotate_heads(X, T, start=17), ValueError),
    (lambda: rope.rotate_heads(X, T, start=-1), ValueError),
    (lambda: rope.rotate_heads(X[..., :14], T), ValueError),
    (lambda: rope.rotate_heads(X, T, layout="paired"), ValueError),
    (lambda: rope.rotate_heads(X, RotaryTables(T.cos.expand(3, 1, 4, 8), T.sin.expand(3, 1, 4, 8))), ValueError),
    (lambda: rope.rotate_heads(X, RotaryTables(T.cos.double(), T.sin.double())), TypeError),
    (lambda: rope.rotate_heads(X, RotaryTables(T.cos, T.sin[..., :4])), ValueError),
    (lambda: rope.rotate_query_key(X, X.bfloat16(), T), TypeError),
    (lambda: rope.rotate_query_key(X, X[..., :16], T), ValueError),
    (lambda: rope.rotate_query_key(X, X[:1], T), ValueError),
    (lambda: rope.build_position_tables(torch.zeros(1, 1, 4, dtype=torch.int64), rotary_dim=16), ValueError),
    (lambda: rope.build_position_tables(torch.zeros(4), rotary_dim=16), TypeError),
    (lambda: rope.build_position_tables(torch.arange(4), rotary_dim=15), ValueError),
    (lambda: rope.build_position_tables(torch.arange(4), rotary_dim=514), ValueError),
    (lambda: rope.build_position_tables(torch.arange(4), rotary_dim=16, theta=0.0), ValueError),
    (lambda: PositionScaling("cubic"), ValueError),
    (lambda: PositionScaling("linear", 0.0), ValueError),
    (lambda: PositionScaling("yarn", 2.0), ValueError),
    (lambda: PositionScaling("yarn", 2.0, 100, 1.0, 1.0), ValueError),
    (lambda: PositionScaling("yarn", 2.0, 100, attention_factor=-1.0), ValueError),
    (lambda: layers.add_rms_norm(X, X[..., :16], torch.zeros(32)), ValueError),
    (lambda: layers.add_rms_norm(X, X.bfloat16(), torch.zeros(32)), TypeError),
    (lambda: layers.add_rms_norm(X.half(), X.half(), torch.zeros(32)), TypeError),
    (lambda: layers.add_rms_norm(X, X, torch.zeros(31)), ValueError),
    (lambda: layers.add_rms_norm(X, X, torch.zeros(32).bfloat16()), TypeError),
    (lambda: layers.add_rms_norm(X, X, torch.zeros(32), eps=-1.0), ValueError),
    (lambda: layers.add_rms_norm(X, X, torch.zeros(32), eps=float("nan")), ValueError),
    (lambda: layers.add_rms_norm(X[..., :0], X[..., :0], torch.zeros(0)), ValueError),
    (lambda: layers.add_rms_norm_fp8(X.requires_grad_(False), X, torch.zeros(32, requires_grad=True)), RuntimeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake-pointer validation tests run only without a GPU")


@cpu_only
def test_c_entry_points_refuse():
    lib = _lib.load()
    p, s = 4096, _lib.i64_array([64, 64, 64])
    f = (ctypes.c_double * 4)(1.0, 0.5, 0.25, 0.125)
    fp = ctypes.cast(f, ctypes.c_void_p)
    bad = (ctypes.c_double * 4)(1.0, float("inf"), 0.25, 0.125)

    def tables(pos=p, i64=1, stride=0, B=1, L=8, P=4, freq=fp, amp=1.0, cos=p, sin=p):
        return lib.avattn_position_tables(pos, i64, stride, B, L, P, freq, amp, cos, sin, None)

    assert tables(P=0) == 2 and tables(P=257) == 2 and tables(B=-1) == 2
    assert tables(freq=None) == 1 and tables(pos=None) == 1 and tables(cos=None) == 1
    assert tables(pos=p + 4) == 5 and tables(sin=p + 2) == 5
    assert tables(stride=7) == 9 and tables(amp=float("nan")) == 9
    assert tables(freq=ctypes.cast(bad, ctypes.c_void_p)) == 9
    assert tables(L=0) == 0

    def rot(q=p, qs=s, H=2, qo=p, qos=s, k=None, ks=None, Hk=0, ko=None, kos=None, B=1, L=4, D=64, P=8, start=0,
            f32=0, c=p, n=p, tsb=0):
        return lib.avattn_rotate(q, qs, H, qo, qos, k, ks, Hk, ko, kos, B, L, D, P, start, 1, f32, c, n, tsb, 0, None)

    assert rot(P=33) == 2 and rot(start=49) == 2 and rot(start=-1) == 2 and rot(P=0) == 2 and rot(D=1) == 2
    assert rot(D=65538) == 2 and rot(H=1 << 25) == 8
    assert rot(q=None) == 1 and rot(qos=None) == 1 and rot(c=None) == 1 and rot(Hk=1) == 1
    assert rot(q=p + 1) == 5 and rot(q=p + 2, f32=1) == 5 and rot(n=p + 2) == 5
    assert rot(tsb=31) == 9 and rot(B=0) == 0

    def norm(x=p, r=p, w=p, w32=0, rows=3, W=64, f32=0, eps=1e-6, h=p, n=p, sc=None):
        return lib.avattn_add_rms_norm(x, 64, r, 64, w, w32, rows, W, f32, eps, h, n, sc, None)

    assert norm(rows=-1) == 2 and norm(W=0) == 2 and norm(rows=1 << 31) == 8
    assert norm(eps=-1.0) == 9 and norm(f32=1) == 9
    assert norm(x=None) == 1 and norm(n=None) == 1 and norm(x=p + 1) == 5 and norm(sc=p + 2) == 5
    assert norm(rows=0, x=None) == 0

    def back(dn=p, h=p, w=p, rows=3, W=64, f32=0, w32=0, dx=p, dw=p, ws=p, nb=1 << 20, eps=0.0):
        return lib.avattn_add_rms_norm_bwd(dn, 64, None, 0, h, 64, w, w32, rows, W, f32, eps, dx, dw, ws, nb, None)

    assert back(W=0) == 2 and back(eps=float("inf")) == 9 and back(f32=1) == 9
    assert back(dw=None) == 1 and back(dn=None) == 1 and back(dx=None) == 1 and back(h=p + 1) == 5
    assert back(ws=None) == 6 and back(nb=4 * 64 * 4 - 1) == 6 and back(ws=p + 4) == 6
    assert lib.avattn_add_rms_norm_bwd_workspace_size(3, 64) == 4 * 64 * 4
    assert lib.avattn_add_rms_norm_bwd_workspace_size(5000, 64) == 4096 * 64 * 4
    assert lib.avattn_add_rms_norm_bwd_workspace_size(5000, 1025) == 1024 * 1025 * 4
    assert lib.avattn_add_rms_norm_bwd_workspace_size(5, 0) == 0
