"""Refusals of the paged cache and of the gated residual norm: every check runs
before any launch, so they are tested without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from avgen_amd import _lib, cache, cache_ops, gated_ops, layers
from avgen_amd.cache import PagedCache, append_paged, paged_attention
from avgen_amd.rope import RotaryTables

B16, F8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


class OffGpu:
    """What a PagedCache holds, on the CPU (which a PagedCache refuses)."""

    _plan = None

    def __init__(self, dtype=B16, pages=6, heads=2, page=16, dim=64):
        self.key, self.value = (torch.zeros(pages, heads, page, dim).to(dtype) for _ in range(2))
        coded = dtype is F8
        self.key_exponent, self.value_exponent = (torch.zeros(pages, heads, dtype=torch.int8) if coded else None
                                                  for _ in range(2))


POOL, CODED = OffGpu(), OffGpu(F8)
Q = torch.zeros(3, 4, 5, 64, dtype=B16)
K = Q[:, :2]
TABLE = torch.zeros(3, 2, dtype=I32)
LEN = torch.full((3,), 5, dtype=I32)
T = RotaryTables(cos=torch.zeros(1, 1, 5, 8), sin=torch.zeros(1, 1, 5, 8))


def pool(**changed):
    p = OffGpu()
    for name, t in changed.items():
        setattr(p, name, t)
    return p


def made(**changed):
    given = dict(key=POOL.key, value=POOL.value)
    given.update(changed)
    return PagedCache(**given)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        made()
    for p in (POOL, CODED):
        with pytest.raises(RuntimeError, match="no CPU path"):
            append_paged(p, K, K, TABLE, LEN)
        with pytest.raises(RuntimeError, match="no CPU path"):
            paged_attention(Q, p, TABLE, LEN)
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.gated_add_rms_norm(Q, Q)


@pytest.mark.parametrize("call, error", [
    (lambda: made(value=POOL.value[:5]), ValueError),
    (lambda: made(key=POOL.key[0], value=POOL.value[0]), ValueError),
    (lambda: made(value=POOL.value.float()), TypeError),
    (lambda: made(key=POOL.key.float(), value=POOL.value.float()), TypeError),
    (lambda: made(key=CODED.key, value=CODED.value), ValueError),
    (lambda: made(key_exponent=CODED.key_exponent, value_exponent=CODED.value_exponent), ValueError),
    (lambda: made(key=CODED.key, value=CODED.value, key_exponent=CODED.key_exponent[:5],
                  value_exponent=CODED.value_exponent), ValueError),
    (lambda: made(key=CODED.key, value=CODED.value, key_exponent=CODED.key_exponent.int(),
                  value_exponent=CODED.value_exponent), TypeError),
    (lambda: made(key=CODED.key, value=CODED.value, key_exponent=CODED.key_exponent.t().contiguous().t(),
                  value_exponent=CODED.value_exponent), ValueError),
    (lambda: made(key=POOL.key[:, :, :8], value=POOL.value[:, :, :8]), ValueError),  # page size
    (lambda: made(key=torch.zeros(2, 2, 512, 64, dtype=B16), value=torch.zeros(2, 2, 512, 64, dtype=B16)), ValueError),
    (lambda: made(key=torch.zeros(2, 2, 48, 64, dtype=B16), value=torch.zeros(2, 2, 48, 64, dtype=B16)), ValueError),
    (lambda: made(key=POOL.key[..., :32], value=POOL.value[..., :32]), ValueError),  # head_dim
    (lambda: made(key=POOL.key[:, :0], value=POOL.value[:, :0]), ValueError),
    (lambda: made(key=POOL.key.transpose(2, 3).contiguous().transpose(2, 3)), ValueError),  # slots not rows
    (lambda: made(key=POOL.key.transpose(1, 2).contiguous().transpose(1, 2)), ValueError),  # slots apart
    (lambda: made(key=POOL.key[:1].expand(6, 2, 16, 64)), ValueError),  # pages in one place
    (lambda: made(key=POOL.key.as_strided((6, 2, 16, 64), (1024, 1024, 64, 1))), ValueError),
    (lambda: made(key=torch.zeros(6 * 2 * 1024 + 1, dtype=B16)[1:].view(6, 2, 16, 64)), ValueError),  # unaligned
    (lambda: append_paged(POOL, K[0], K, TABLE, LEN), ValueError),
    (lambda: append_paged(POOL, K, K[:, :, :4], TABLE, LEN), ValueError),
    (lambda: append_paged(POOL, Q, Q, TABLE, LEN), ValueError),  # heads
    (lambda: append_paged(POOL, K.float(), K, TABLE, LEN), TypeError),
    (lambda: append_paged(POOL, K, K.float(), TABLE, LEN), TypeError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, tables=T, query=Q.float()), TypeError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, tables=T, query=Q[:, :, :4]), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, tables=T, start=49), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, tables=T, start=-1), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, tables=T, layout="paired"), ValueError),
    (lambda: append_paged(POOL, K[:, :, :4], K[:, :, :4], TABLE, LEN, tables=T), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, tables=RotaryTables(T.cos.double(), T.sin.double())), TypeError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN,
                          tables=RotaryTables(T.cos.expand(2, 1, 5, 8), T.sin.expand(2, 1, 5, 8))), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE[:2], LEN), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE[0], LEN), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE.long(), LEN), TypeError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN[:2]), ValueError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN.long()), TypeError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, counts=LEN.long()), TypeError),
    (lambda: append_paged(POOL, K, K, TABLE, LEN, counts=LEN[:1]), ValueError),
    (lambda: append_paged(POOL, K.clone().requires_grad_(True), K, TABLE, LEN), RuntimeError),
    (lambda: paged_attention(Q[0], POOL, TABLE, LEN), ValueError),
    (lambda: paged_attention(Q[..., :32], POOL, TABLE, LEN), ValueError),
    (lambda: paged_attention(Q.float(), POOL, TABLE, LEN), TypeError),
    (lambda: paged_attention(Q[:, :3], POOL, TABLE, LEN), ValueError),
    (lambda: paged_attention(Q[:, :0], POOL, TABLE, LEN), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE[:2], LEN), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE.long(), LEN), TypeError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN.long()), TypeError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, window=0), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, window=(1 << 30) + 1), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, softcap=0.0), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, softcap=1025.0), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, scale=0.0), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, scale=float("nan")), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, distance_slopes=torch.zeros(3)), ValueError),
    (lambda: paged_attention(Q, POOL, TABLE, LEN, distance_slopes=torch.zeros(4).double()), TypeError),
    (lambda: paged_attention(torch.zeros(3, 130, 5, 64, dtype=B16), POOL, TABLE, LEN,
                             distance_slopes=torch.zeros(130)), ValueError),
    (lambda: paged_attention(Q.clone().requires_grad_(True), POOL, TABLE, LEN), RuntimeError),
    (lambda: cache_ops.page_values(CODED.key, CODED.value, CODED.key_exponent, None), ValueError),
])
def test_paged_refusals(call, error):
    with pytest.raises(error):
        call()


X, W, S = torch.zeros(2, 3, 32), torch.zeros(32), torch.zeros(6, 2)


def gated(x=X, r=X, w=W, **more):
    return layers.gated_add_rms_norm(x, r, w, **more)


@pytest.mark.parametrize("call, error", [
    (lambda: gated(r=X[..., :16]), ValueError),
    (lambda: gated(r=X.bfloat16()), TypeError),
    (lambda: gated(x=X.half(), r=X.half()), TypeError),
    (lambda: gated(w=W[:31]), ValueError),
    (lambda: gated(w=W.bfloat16()), TypeError),
    (lambda: gated(post_weight=W[:31]), ValueError),
    (lambda: gated(post_weight=W.half()), TypeError),
    (lambda: gated(gate=W[:31]), ValueError),
    (lambda: gated(gate=X[:, :2]), ValueError),
    (lambda: gated(gate=torch.zeros(3, 1, 32)), ValueError),
    (lambda: gated(gate=torch.zeros(1, 2, 3, 32)), ValueError),
    (lambda: gated(gate=torch.zeros(())), ValueError),
    (lambda: gated(scale=W.bfloat16()), TypeError),
    (lambda: gated(scale=W, shift=W.bfloat16()), TypeError),
    (lambda: gated(eps=-1.0), ValueError),
    (lambda: gated(eps=float("inf")), ValueError),
    (lambda: gated(residual_scale=float("nan")), ValueError),
    (lambda: gated(x=X[..., :0], r=X[..., :0], w=W[:0]), ValueError),
    (lambda: gated_ops.gated_add_rms_norm(X, X, W, None, torch.zeros(4, 32), None, None, 1.0, 1e-6), ValueError),
    (lambda: gated_ops.gated_add_rms_norm(X, X, W, None, torch.zeros(2, 32), torch.zeros(3, 32), None, 1.0, 1e-6),
     ValueError),
    (lambda: gated_ops.gated_add_rms_norm_bwd(X[:1], None, X, X, S, W, None, W, None, None, 1.0, 1e-6), ValueError),
    (lambda: gated_ops.gated_add_rms_norm_bwd(X, None, X, X[:1], S, W, None, W, None, None, 1.0, 1e-6), ValueError),
    (lambda: gated_ops.gated_add_rms_norm_bwd(X, X.bfloat16(), X, X, S, W, None, W, None, None, 1.0, 1e-6), ValueError),
    (lambda: gated_ops.gated_add_rms_norm_bwd(X, None, X, X, S[:5], W, None, W, None, None, 1.0, 1e-6), ValueError),
])
def test_gated_refusals(call, error):
    with pytest.raises(error):
        call()


def test_modulations_take_one_shape():
    one = layers._one_modulation
    x = (2, 3, 4, 8)
    shapes = lambda *t: [None if y is None else tuple(y.shape) for y in one(x, *t)]  # noqa: E731
    z = torch.zeros
    assert shapes(z(8), None, z(8)) == [(8,), None, (8,)]
    assert shapes(z(2, 1, 1, 8), z(8), None) == [(2, 1, 1, 8), (2, 1, 1, 8), None]
    assert shapes(z(8), z(2, 3, 1, 8), z(2, 1, 1, 8)) == [(2, 3, 1, 8)] * 3
    assert shapes(z(4, 8), None, None) == [(2, 3, 4, 8), None, None]
    assert shapes(z(1, 1, 1, 8), z(8), None) == [(1, 1, 1, 8), (1, 1, 1, 8), None]
    assert shapes(None, None, None) == [None] * 3


# ---------------------------------------------------------------------------
# The C entry points: fake addresses, refused before any launch
# ---------------------------------------------------------------------------

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake-pointer tests run only without a GPU")
P = 1 << 20  # an aligned address that nothing reads
S3 = ctypes.c_int64 * 3


def strides(*s):
    return S3(*s)


def append_args(**c):
    a = dict(k=P, ks=strides(640, 64, 128), v=P, vs=strides(640, 64, 128), q=P, qs=strides(1280, 64, 256), hq=4, qo=P,
             qos=strides(1280, 64, 256), B=2, H=2, L=5, D=64, cos=P, sin=P, tsb=0, pairs=8, start=0, half=0, table=P,
             bts=3, blocks=3, lengths=P, counts=None, kp=P, kps=strides(2048, 1024, 64), vp=P,
             vps=strides(2048, 1024, 64), ke=None, kes=0, ve=None, ves=0, pages=6, page=16, stream=None)
    assert set(c) <= set(a)
    a.update(c)
    return list(a.values())


def attend_args(**c):
    a = dict(q=P, qs=strides(1280, 64, 256), B=2, Hq=4, H=2, L=5, D=64, table=P, bts=3, blocks=3, lengths=P,
             counts=None, kp=P, kps=strides(2048, 1024, 64), vp=P, vps=strides(2048, 1024, 64), ke=None, kes=0, ve=None,
             ves=0, pages=6, page=16, window=0, scale=0.125, cap=0.0, slopes=None, out=P, os=strides(1280, 64, 256),
             lse=P, ws=P, wsb=1 << 30, stream=None)
    assert set(c) <= set(a)
    a.update(c)
    return list(a.values())


@cpu_only
@pytest.mark.parametrize("changed, status", [
    (dict(B=-1), _lib.ERR_BAD_SHAPE), (dict(L=-1), _lib.ERR_BAD_SHAPE), (dict(H=0), _lib.ERR_BAD_SHAPE),
    (dict(hq=-1), _lib.ERR_BAD_SHAPE), (dict(D=32), _lib.ERR_HEAD_DIM), (dict(page=8), _lib.ERR_BAD_SHAPE),
    (dict(page=24), _lib.ERR_BAD_SHAPE), (dict(page=512), _lib.ERR_BAD_SHAPE), (dict(pages=-1), _lib.ERR_BAD_SHAPE),
    (dict(kp=None), _lib.ERR_NULL_POINTER), (dict(vps=None), _lib.ERR_NULL_POINTER),
    (dict(kp=P + 8), _lib.ERR_LAYOUT), (dict(kps=strides(2052, 1024, 64)), _lib.ERR_LAYOUT),
    (dict(vps=strides(2048, -1024, 64)), _lib.ERR_LAYOUT), (dict(ke=P), _lib.ERR_ARGUMENT),
    (dict(ke=P, ve=P, kes=-1), _lib.ERR_LAYOUT), (dict(ke=P, ve=P, kps=strides(2056, 1024, 64)), _lib.ERR_LAYOUT),
    (dict(blocks=-1), _lib.ERR_BAD_SHAPE), (dict(table=None), _lib.ERR_NULL_POINTER),
    (dict(lengths=None), _lib.ERR_NULL_POINTER), (dict(table=P + 2), _lib.ERR_LAYOUT), (dict(bts=2), _lib.ERR_ARGUMENT),
    (dict(sin=None), _lib.ERR_ARGUMENT), (dict(pairs=0), _lib.ERR_BAD_SHAPE), (dict(start=49), _lib.ERR_BAD_SHAPE),
    (dict(cos=P + 2), _lib.ERR_LAYOUT), (dict(tsb=39), _lib.ERR_ARGUMENT), (dict(k=None), _lib.ERR_NULL_POINTER),
    (dict(v=P + 1), _lib.ERR_LAYOUT), (dict(qo=None), _lib.ERR_NULL_POINTER), (dict(q=P + 1), _lib.ERR_LAYOUT),
    (dict(B=1 << 15, L=1 << 15, bts=0), _lib.ERR_TOO_LARGE),
    (dict(B=0), _lib.OK), (dict(L=0), _lib.OK),
])
def test_append_status(changed, status):
    assert _lib.load().avattn_append_paged(*append_args(**changed)) == status


@cpu_only
@pytest.mark.parametrize("changed, status", [
    (dict(B=-1), _lib.ERR_BAD_SHAPE), (dict(Hq=3), _lib.ERR_GQA), (dict(D=96), _lib.ERR_HEAD_DIM),
    (dict(page=20), _lib.ERR_BAD_SHAPE), (dict(H=0, Hq=0), _lib.ERR_BAD_SHAPE), (dict(qs=None), _lib.ERR_NULL_POINTER),
    (dict(q=None), _lib.ERR_NULL_POINTER), (dict(lse=None), _lib.ERR_NULL_POINTER), (dict(q=P + 8), _lib.ERR_LAYOUT),
    (dict(qs=strides(1280, 60, 256)), _lib.ERR_LAYOUT), (dict(out=P + 2), _lib.ERR_LAYOUT),
    (dict(window=-1), _lib.ERR_ARGUMENT), (dict(scale=0.0), _lib.ERR_ARGUMENT),
    (dict(scale=float("inf")), _lib.ERR_ARGUMENT), (dict(cap=-1.0), _lib.ERR_ARGUMENT),
    (dict(cap=2000.0), _lib.ERR_ARGUMENT), (dict(slopes=P + 2), _lib.ERR_LAYOUT),
    (dict(blocks=1 << 27, bts=1 << 27), _lib.ERR_TOO_LARGE), (dict(blocks=1 << 21, bts=1 << 21), _lib.ERR_TOO_LARGE),
    (dict(lengths=None), _lib.ERR_NULL_POINTER), (dict(counts=P + 1), _lib.ERR_LAYOUT),
    (dict(L=4000, Hq=64, ws=None, qs=strides(4096 * 4000, 64, 4096)), _lib.ERR_WORKSPACE),
    (dict(L=4000, Hq=64, wsb=1000, qs=strides(4096 * 4000, 64, 4096)), _lib.ERR_WORKSPACE),
    (dict(blocks=300, bts=300, ws=P + 8), _lib.ERR_WORKSPACE), (dict(blocks=300, bts=300, wsb=8), _lib.ERR_WORKSPACE),
    (dict(B=0), _lib.OK), (dict(L=0), _lib.OK),
])
def test_attention_status(changed, status):
    assert _lib.load().avattn_paged_attention(*attend_args(**changed)) == status


def norm_args(**c):
    a = dict(x=P, xs=32, r=P, rs=32, w=P, w32=0, p=P, p32=0, g=P, gs=96, s=P, ss=96, t=P, ts=96, m32=0, rows=6, W=32,
             R=3, f32=0, alpha=1.0, eps=1e-6, h=P, n=P, stats=P, stream=None)
    assert set(c) <= set(a)
    a.update(c)
    return list(a.values())


def norm_bwd_args(**c):
    a = dict(dn=P, dns=32, dh=P, dhs=32, x=P, xs=32, r=P, rs=32, stats=P, w=P, w32=0, p=P, p32=0, g=P, gs=96, s=P, ss=96, t=P,
             ts=96, m32=0, rows=6, W=32, R=3, f32=0, alpha=1.0, eps=1e-6, dx=P, dr=P, dw=P, dp=P, dg=P, ds=P, dt=P,
             ws=P, wsb=1 << 20, stream=None)
    assert set(c) <= set(a)
    a.update(c)
    return list(a.values())


SHARED = [
    (dict(rows=-1), _lib.ERR_BAD_SHAPE), (dict(W=0), _lib.ERR_BAD_SHAPE), (dict(R=0), _lib.ERR_BAD_SHAPE),
    (dict(R=4), _lib.ERR_BAD_SHAPE), (dict(rows=1 << 31, R=1 << 31), _lib.ERR_TOO_LARGE),
    (dict(eps=-1.0), _lib.ERR_ARGUMENT), (dict(alpha=float("inf")), _lib.ERR_ARGUMENT),
    (dict(f32=1), _lib.ERR_ARGUMENT), (dict(w=P + 1), _lib.ERR_LAYOUT), (dict(g=P + 1), _lib.ERR_LAYOUT),
    (dict(m32=1, s=P + 2), _lib.ERR_LAYOUT), (dict(x=P + 1), _lib.ERR_LAYOUT),
]


@cpu_only
@pytest.mark.parametrize("changed, status", SHARED + [
    (dict(x=None), _lib.ERR_NULL_POINTER), (dict(n=None), _lib.ERR_NULL_POINTER), (dict(h=P + 1), _lib.ERR_LAYOUT),
    (dict(stats=P + 4), _lib.ERR_LAYOUT),
    (dict(rows=0), _lib.OK),
])
def test_norm_status(changed, status):
    assert _lib.load().avattn_gated_add_rms_norm(*norm_args(**changed)) == status


@cpu_only
@pytest.mark.parametrize("changed, status", SHARED + [
    (dict(rows=0), _lib.ERR_BAD_SHAPE), (dict(x=None), _lib.ERR_NULL_POINTER), (dict(stats=None), _lib.ERR_NULL_POINTER),
    (dict(r=None), _lib.ERR_NULL_POINTER), (dict(stats=P + 4), _lib.ERR_LAYOUT), (dict(dr=None), _lib.ERR_NULL_POINTER),
    (dict(dx=None), _lib.ERR_NULL_POINTER), (dict(w=None), _lib.ERR_ARGUMENT), (dict(g=None), _lib.ERR_ARGUMENT),
    (dict(ws=None), _lib.ERR_WORKSPACE), (dict(wsb=100), _lib.ERR_WORKSPACE), (dict(ws=P + 4), _lib.ERR_WORKSPACE),
    (dict(dg=P + 1), _lib.ERR_LAYOUT), (dict(dw=P + 1), _lib.ERR_LAYOUT), (dict(dh=P + 1), _lib.ERR_LAYOUT),
])
def test_norm_bwd_status(changed, status):
    assert _lib.load().avattn_gated_add_rms_norm_bwd(*norm_bwd_args(**changed)) == status
