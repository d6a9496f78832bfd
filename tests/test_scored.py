"""Attention with changed scores without a GPU: refusals of every layer (all of
them before any launch) and the windows of documents."""

from __future__ import annotations

import ctypes

import pytest
import torch

from avgen_amd import _lib, scored_ops
from avgen_amd import attention as A

B16, F32 = torch.bfloat16, torch.float32
Q, K = torch.zeros(2, 4, 5, 64, dtype=B16), torch.zeros(2, 2, 7, 64, dtype=B16)
QF, KF = Q.float(), K.float()
LO, HI = torch.zeros(5, dtype=torch.int32), torch.full((5,), 7, dtype=torch.int32)
SLOPES = torch.ones(4)


def scored(q=Q, k=K, v=None, **kw):
    return A.scored_attention(q, k, k if v is None else v, **{"enable_gqa": True, **kw})


@pytest.mark.parametrize("call", [scored, lambda: scored(QF, KF), lambda: scored(softcap=30.0),
                                  lambda: scored(distance_slopes=SLOPES, window_lo=LO, window_hi=HI)])
def test_no_cpu_path(call):
    with pytest.raises(RuntimeError, match="no CPU path"):
        call()


@pytest.mark.parametrize("call, error", [
    (lambda: scored(Q[0]), ValueError),
    (lambda: scored(Q.half(), K.half()), TypeError),
    (lambda: scored(Q, KF), TypeError),
    (lambda: scored(v=K[:, :, :6]), ValueError),
    (lambda: scored(Q[:1]), ValueError),
    (lambda: scored(Q[..., :32], K[..., :32]), ValueError),
    (lambda: scored(Q[:, :3]), ValueError),
    (lambda: scored(enable_gqa=False), ValueError),
    (lambda: scored(softcap=0.0), ValueError),
    (lambda: scored(softcap=-1.0), ValueError),
    (lambda: scored(softcap=float("nan")), ValueError),
    (lambda: scored(softcap=float("inf")), ValueError),
    (lambda: scored(softcap=1025.0), ValueError),
    (lambda: scored(scale=0.0), ValueError),
    (lambda: scored(scale=float("nan")), ValueError),
    (lambda: scored(distance_slopes=SLOPES[:2]), ValueError),
    (lambda: scored(distance_slopes=SLOPES.double()), TypeError),
    (lambda: scored(distance_slopes=SLOPES.clone().requires_grad_(True)), NotImplementedError),
    (lambda: scored(Q[:, :1].expand(-1, 130, -1, -1), K, distance_slopes=torch.ones(130)), ValueError),
    (lambda: scored(query_offset=(1 << 30) + 1), ValueError),
    (lambda: scored(query_offset=-(1 << 30) - 1), ValueError),
    (lambda: scored(query_offset=1.0), TypeError),
    (lambda: scored(query_offset=torch.zeros(3, dtype=torch.int32)), ValueError),
    (lambda: scored(query_offset=torch.zeros((), dtype=torch.int32)), ValueError),
    (lambda: scored(query_offset=torch.zeros(2, dtype=torch.int64)), TypeError),
    (lambda: scored(window_lo=LO), ValueError),
    (lambda: scored(window_lo=LO, window_hi=HI.long()), TypeError),
    (lambda: scored(window_lo=LO[:4], window_hi=HI[:4]), ValueError),
    (lambda: scored(attn_mask=torch.ones(2, 1, 1, 6, dtype=torch.bool)), ValueError),
    (lambda: scored(attn_mask=torch.ones(2, 1, 5, 7, dtype=torch.bool)), NotImplementedError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


@pytest.mark.parametrize("change, error", [
    (dict(dout=Q[:, :, :4]), ValueError), (dict(dout=QF), ValueError), (dict(out=Q[:, :2]), ValueError),
    (dict(lse=torch.zeros(2, 4, 4)), ValueError), (dict(lse=torch.zeros(2, 4, 5, dtype=B16)), ValueError),
])
def test_backward_refusals(change, error, monkeypatch):
    # Past the device checks, which on a CPU tensor would come first.
    monkeypatch.setattr(scored_ops, "_one_device", lambda *a: None)
    t = {"dout": Q, "out": Q, "lse": torch.zeros(2, 4, 5), **change}
    with pytest.raises(error):
        scored_ops._bwd_impl(t["dout"], Q, K, K, t["out"], t["lse"], None, None, None, None, None, 0.125, 5.0, 0, False)


@pytest.mark.parametrize("capturing, error, match", [(False, ValueError, "non-decreasing"),
                                                     (True, RuntimeError, "monotone=True")])
@pytest.mark.parametrize("lo, hi", [
    (LO, torch.tensor([1, 3, 2, 4, 5], dtype=torch.int32)),
    (torch.tensor([[0, 0, 0, 0, 0], [0, 0, 2, 1, 3]], dtype=torch.int32), HI.expand(2, -1)),
])
def test_backward_refuses_windows_out_of_order(lo, hi, capturing, error, match, monkeypatch):
    monkeypatch.setattr(scored_ops, "_one_device", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    with pytest.raises(error, match=match):
        scored_ops._bwd_impl(Q, Q, K, K, Q, torch.zeros(2, 4, 5), lo, hi, None, None, None, 0.125, 5.0, 0, False)


def allowed(lo, hi, L):
    j = torch.arange(L)
    return (j >= lo[:, None]) & (j < hi[:, None])


@pytest.mark.parametrize("cu", [[0, 9], [0, 4, 5, 9], [0, 3, 3, 7], [0], [0, 0, 11], [0, 1]])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("prefix", [0, 2, 100, "each"])
def test_document_windows(cu, causal, prefix):
    L = 11
    n = len(cu) - 1
    each = [(3 * s + 1) % 5 for s in range(n)] if prefix == "each" else [prefix] * n
    if prefix == "each":
        prefix = torch.tensor(each, dtype=torch.int64)
    lo, hi = A.document_windows(torch.tensor(cu), L, causal=causal, prefix_lengths=prefix)
    assert lo.dtype is hi.dtype is torch.int32
    assert bool((lo[1:] >= lo[:-1]).all()) and bool((hi[1:] >= hi[:-1]).all())
    want = torch.zeros(L, L, dtype=torch.bool)
    for s in range(n):
        for i in range(cu[s], cu[s + 1]):
            for j in range(cu[s], cu[s + 1]):
                want[i, j] = not causal or j <= i or j - cu[s] < each[s]
    assert torch.equal(allowed(lo, hi, L), want)


cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake-pointer validation tests run only without a GPU")


@cpu_only
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("Lq", [1, 5000])  # the few-row kernels and the others
def test_c_entry_points_refuse(f32, Lq):
    lib = _lib.load()
    p, s = 4096, _lib.i64_array([64, 64, 64])
    odd = _lib.i64_array([64, 64, 66])
    Lk = 5000

    def fwd(q=p, k=p, v=p, qs=s, ks=s, vs=s, B=1, Hq=4, Hkv=2, Lq=Lq, Lk=Lk, D=64, mask=None, msb=0, lo=None, hi=None,
            wsb=0, scale=0.125, cap=10.0, slopes=None, offs=None, off=0, flags=0, out=p, os=s, lse=p, ws=p, nb=1 << 40):
        return lib.avattn_fwd_scored(q, k, v, qs, ks, vs, B, Hq, Hkv, Lq, Lk, D, f32, mask, msb, lo, hi, wsb, scale,
                                     cap, slopes, offs, off, flags, out, os, lse, ws, nb, None)

    assert fwd(B=-1) == 2 and fwd(D=96) == 3 and fwd(Hkv=3) == 4 and fwd(Hq=0) == 4
    assert fwd(qs=None) == 1 and fwd(os=None) == 1
    for bad in (dict(scale=0.0), dict(scale=float("nan")), dict(cap=-1.0), dict(cap=float("inf")), dict(flags=2),
                dict(off=(1 << 30) + 1), dict(off=-(1 << 30) - 1), dict(mask=p, msb=Lk - 1),
                dict(cap=1e-44), dict(lo=p, hi=p, wsb=-1)):
        assert fwd(**bad) == 9, bad
    if not f32:
        assert fwd(cap=1025.0) == 9
    assert fwd(lo=p) == 1 and fwd(hi=p) == 1
    assert fwd(lo=p + 2, hi=p) == 5 and fwd(slopes=p + 2) == 5 and fwd(offs=p + 1) == 5
    assert fwd(Hq=130, slopes=p) == 8
    for name in ("q", "k", "v", "out", "lse"):
        assert fwd(**{name: None}) == 1, name
    for name in ("q", "k", "v", "out"):
        assert fwd(**{name: p + 8}) == 5, name
    for name in ("qs", "ks", "vs", "os"):
        assert fwd(**{name: odd}) == 5, name
    need = lib.avattn_fwd_scored_workspace_size(1, 4, 2, Lq, Lk, 64, f32)
    assert need > 0
    assert fwd(ws=None) == 6 and fwd(nb=need - 1) == 6 and fwd(ws=p + 8) == 6
    assert fwd(B=0) == 0 and fwd(Lq=0) == 0
    if Lq == 1:
        far = _lib.i64_array([64, 64, 1 << 23])
        assert fwd(ks=far) == 5 and fwd(vs=far) == 5
    assert lib.avattn_fwd_scored_workspace_size(1, 4, 3, Lq, Lk, 64, f32) == 0
    assert lib.avattn_fwd_scored_workspace_size(1, 4, 2, Lq, 0, 64, f32) == 0

    def bwd(dout=p, q=p, k=p, v=p, out=p, lse=p, dos=s, qs=s, ks=s, vs=s, os=s, B=1, Hq=4, Hkv=2, Lq=Lq, Lk=Lk, D=64,
            mask=None, msb=0, lo=None, hi=None, wsb=0, table=None, tsb=0, units=0, scale=0.125, cap=10.0, slopes=None,
            offs=None, off=0, dq=p, dqs=s, dk=p, dks=s, dv=p, dvs=s, ws=p, nb=1 << 40):
        return lib.avattn_bwd_scored(dout, q, k, v, out, lse, dos, qs, ks, vs, os, B, Hq, Hkv, Lq, Lk, D, f32, mask,
                                     msb, lo, hi, wsb, table, tsb, units, scale, cap, slopes, offs, off, dq, dqs, dk,
                                     dks, dv, dvs, ws, nb, None)

    assert bwd(B=-1) == 2 and bwd(D=96) == 3 and bwd(Hkv=3) == 4
    for bad in (dict(scale=0.0), dict(cap=-1.0), dict(cap=float("nan")), dict(off=(1 << 30) + 1),
                dict(mask=p, msb=Lk - 1), dict(cap=1e-44), dict(lo=p, hi=p, wsb=-1)):
        assert bwd(**bad) == 9, bad
    if f32:
        assert bwd(table=p, lo=p, hi=p, units=1) == 9
    assert bwd(lo=p) == 1 and bwd(slopes=p + 2) == 5 and bwd(Hq=130, slopes=p) == 8
    for name in ("dout", "q", "k", "v", "out", "lse", "dq", "dk", "dv"):
        assert bwd(**{name: None}) == 1, name
    for name in ("dout", "q", "k", "v", "out", "dq", "dk", "dv"):
        assert bwd(**{name: p + 8}) == 5, name
    for name in ("dos", "qs", "ks", "vs", "os", "dqs", "dks", "dvs"):
        assert bwd(**{name: odd}) == 5, name
        assert bwd(**{name: None}) == 1, name
    assert bwd(ws=None) == 6 and bwd(nb=16) == 6
    assert bwd(B=0) == 0
    for windowed in (0, 1):
        assert lib.avattn_bwd_scored_workspace_size(1, 4, 2, Lq, Lk, 64, f32, windowed) > 0
        assert lib.avattn_bwd_scored_workspace_size(1, 4, 2, Lq, 0, 64, f32, windowed) == 0


def test_few_rows_workspace_is_that_of_the_split():
    """One query per sequence: parts of 128 keys or more over at most one
    round of the chip, 4 rows of D + 2 floats (rounded up) each."""
    lib = _lib.load()
    small = lib.avattn_fwd_scored_workspace_size(1, 8, 2, 1, 64, 128, 0)
    assert small == 0  # one part: straight to the output
    one = lib.avattn_fwd_scored_workspace_size(1, 8, 2, 1, 100000, 128, 0)
    assert 0 < one <= 256 * (4 * 128 + 64) * 4
    assert ctypes.sizeof(ctypes.c_size_t) == 8
