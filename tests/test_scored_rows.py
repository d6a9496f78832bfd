"""The row statistic of biased scores without a GPU: refusals of the C entry
points and of the backward."""

from __future__ import annotations

import math

import pytest
import torch

from avgen_amd import _lib, ops, scored_ops

B16 = torch.bfloat16
cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake-pointer validation tests run only without a GPU")


@cpu_only
@pytest.mark.parametrize("f32", [0, 1])
@pytest.mark.parametrize("Lq", [1, 5000])
def test_c_entry_points_refuse(f32, Lq):
    lib = _lib.load()
    p, s, odd = 4096, _lib.i64_array([64, 64, 64]), _lib.i64_array([64, 64, 66])
    Lk = 5000

    def fwd(slopes=p, flags=4, B=1, lse=p):
        return lib.avattn_fwd_scored(p, p, p, s, s, s, B, 4, 2, Lq, Lk, 64, f32, None, 0, None, None, 0, 0.125, 10.0,
                                     slopes, None, 0, flags, p, s, lse, p, 1 << 40, None)

    assert _lib.SCORED_ROW_LSE == 4
    assert fwd(slopes=None) == 9 and fwd(flags=8) == 9 and fwd(flags=2) == 9
    assert fwd(lse=None) == 1
    assert fwd(B=0) == 0 and fwd(B=0, flags=5) == 0

    def bwd(lse=p, dqs=s, ws=p, scale=0.125, B=1, slopes=p):
        return lib.avattn_bwd_scored_row_lse(p, p, p, p, p, lse, s, s, s, s, s, B, 4, 2, Lq, Lk, 64, f32, None, 0, None,
                                             None, 0, None, 0, 0, scale, 10.0, slopes, None, 0, p, dqs, p, s, p, s, ws,
                                             1 << 40, None)

    assert bwd(lse=None) == 1 and bwd(dqs=None) == 1 and bwd(dqs=odd) == 5 and bwd(ws=None) == 6
    assert bwd(scale=0.0) == 9 and bwd(slopes=p + 2) == 5
    assert bwd(B=0) == 0 and bwd(B=-1) == 2


@pytest.mark.parametrize("row_lse", [torch.zeros(2, 4, 4), torch.zeros(2, 4, 5, dtype=B16), torch.zeros(2, 2, 5)])
def test_backward_refuses_another_row_statistic(row_lse, monkeypatch):
    monkeypatch.setattr(scored_ops, "_one_device", lambda *a: None)
    q, k = torch.zeros(2, 4, 5, 64, dtype=B16), torch.zeros(2, 2, 7, 64, dtype=B16)
    with pytest.raises(ValueError, match="logsumexp"):
        scored_ops._bwd_impl(q, q, k, k, q, torch.zeros(2, 4, 5), None, None, None, torch.ones(4), None, 0.125, 5.0, 0,
                             False, row_lse)


@pytest.mark.parametrize("f32", [False, True])
def test_strides_of_sizes_of_one_are_rounded(f32):
    """What the C entry points would refuse in a size that is stepped by, they
    get in whole units where the size is one."""
    t = torch.zeros(100_000, dtype=torch.float32 if f32 else B16)
    one = t.as_strided((1, 3, 5, 64), (12_345, 320, 64, 1))
    laid, strides = scored_ops._laid_out(one, f32)
    assert laid.data_ptr() == one.data_ptr() and list(strides) == [12_352, 320, 64]
    one = t.as_strided((2, 1, 1, 64), (640, 77, 67, 1))
    laid, strides = scored_ops._laid_out(one, f32)
    assert laid.data_ptr() == one.data_ptr() and list(strides) == [640, 80, 72]
    two = t.as_strided((2, 3, 5, 64), (12_345, 320, 64, 1))
    laid, strides = scored_ops._laid_out(two, f32)
    assert laid.data_ptr() != two.data_ptr() and list(strides) == [960, 320, 64]


@pytest.mark.parametrize("f32", [False, True])
def test_unaligned_rows_are_copied(f32):
    """Also where they are contiguous, one row of one head among them."""
    dtype = torch.float32 if f32 else B16
    ready = ops._f32_ready if f32 else ops._kernel_ready
    flat = torch.arange(3000, dtype=torch.float32).to(dtype)
    for shape in ((2, 3, 5, 64), (1, 1, 1, 64)):
        t = flat[1:1 + math.prod(shape)].view(shape)
        assert t.is_contiguous() and t.data_ptr() % 16 != 0
        for got in (ready(t), scored_ops._laid_out(t, f32)[0]):
            assert got.data_ptr() % 16 == 0 and torch.equal(got, t)
