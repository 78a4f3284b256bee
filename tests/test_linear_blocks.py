"""Refusals of the block-scaled and grouped products, and of the quantiser, before any device work
(CPU): each names its argument and none touches a device. Pointers are never dereferenced here."""
import pytest

import tsfm_b200 as tb
from helpers import has_gpu

F32, F16, BF16 = 0, 1, 2
P = 1 << 20  # an aligned address that no refused call reads


def name(st):
    return tb.STATUS_NAMES[st]


def quantize(**kw):
    a = dict(x=P, x_dtype=BF16, rows=4, cols=200, ldx=200, block_rows=1, q=P, ldq=208, scale=P, ld_scale=2, stream=None)
    a.update(kw)
    return name(tb.lib.tsfm_kernel_quantize_e4m3(*a.values()))


def e4m3(**kw):
    a = dict(x=P, xs=P, ld_xs=2, w=P, ws=P, ld_ws=2, bias=None, y=P, y_dtype=BF16, accumulate=0, act=0, M=4, N=256,
             K=200, ldx=208, ldw=208, ldy=256, stream=None)
    a.update(kw)
    return name(tb.lib.tsfm_kernel_linear_e4m3(*a.values()))


def grouped(**kw):
    a = dict(x=P, x_dtype=BF16, w=P, w_dtype=BF16, bias=None, y=P, y_dtype=BF16, accumulate=0, act=0, offsets=P,
             groups=3, M=4, N=256, K=200, ldx=200, ldw=200, w_group=256 * 200, ldy=256, stream=None)
    a.update(kw)
    return name(tb.lib.tsfm_kernel_linear_grouped(*a.values()))


def grouped_e4m3(**kw):
    a = dict(x=P, xs=P, ld_xs=2, w=P, ws=P, ld_ws=2, ws_group=4, bias=None, y=P, y_dtype=BF16, accumulate=0, act=0,
             offsets=P, groups=3, M=4, N=256, K=200, ldx=208, ldw=208, w_group=256 * 208, ldy=256, stream=None)
    a.update(kw)
    return name(tb.lib.tsfm_kernel_linear_grouped_e4m3(*a.values()))


@pytest.mark.parametrize("kw", [dict(x=None), dict(q=None), dict(scale=None), dict(rows=-1), dict(cols=0),
                                dict(ldx=199), dict(ldq=199), dict(ld_scale=1), dict(block_rows=64),
                                dict(x=P + 1), dict(scale=P + 2), dict(x_dtype=F32, x=P + 2), dict(rows=1 << 31)])
def test_quantize_refusals(kw):
    assert quantize(**kw) == "INVALID_ARGUMENT"


def test_quantize_dtype_and_empty():
    assert quantize(x_dtype=3) == "UNSUPPORTED_DTYPE"
    assert quantize(rows=0) == "OK"


COMMON = [dict(x=None), dict(w=None), dict(y=None), dict(M=-1), dict(N=0), dict(K=0), dict(K=1 << 31, ldx=1 << 31, ldw=1 << 31),
          dict(act=2), dict(accumulate=2), dict(accumulate=1), dict(act=3, N=128), dict(act=3, bias=P),
          dict(act=3, y_dtype=F32), dict(ldx=192), dict(ldw=192), dict(ldy=255), dict(x=P + 8), dict(w=P + 8),
          dict(ldx=201), dict(ldw=201), dict(y=P + 1), dict(bias=P + 2)]
SCALES = [dict(xs=None), dict(ws=None), dict(ld_xs=1), dict(ld_ws=1), dict(xs=P + 2), dict(ws=P + 1)]
GROUPS = [dict(offsets=None), dict(groups=0), dict(groups=-1), dict(w_group=100), dict(offsets=P + 2)]


@pytest.mark.parametrize("kw", COMMON + SCALES)
def test_linear_e4m3_refusals(kw):
    assert e4m3(**kw) == "INVALID_ARGUMENT"


@pytest.mark.parametrize("kw", COMMON + GROUPS + [dict(w_group=256 * 200 + 4)])
def test_linear_grouped_refusals(kw):
    assert grouped(**kw) == "INVALID_ARGUMENT"


@pytest.mark.parametrize("kw", COMMON + SCALES + GROUPS + [dict(ws_group=3), dict(w_group=256 * 208 + 8)])
def test_linear_grouped_e4m3_refusals(kw):
    assert grouped_e4m3(**kw) == "INVALID_ARGUMENT"


def test_dtypes_groups_and_empty_batches():
    assert e4m3(y_dtype=7) == "UNSUPPORTED_DTYPE"
    assert grouped(x_dtype=F16) == "UNSUPPORTED_DTYPE"
    assert grouped(x_dtype=F32, w_dtype=F32) == "UNSUPPORTED_DTYPE"
    assert grouped(groups=1025) == "UNSUPPORTED" and grouped_e4m3(groups=1025) == "UNSUPPORTED"
    assert e4m3(M=0) == "OK" and grouped(M=0) == "OK" and grouped_e4m3(M=0) == "OK"
    assert "1024 groups" in (grouped(groups=1025), tb.last_error())[1]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_empty_batches_may_have_null_addresses(dtype):
    # a tensor without rows has no storage: its x, y, codes and scales are null; weights and offsets are not
    for block_rows in (1, 128):
        assert quantize(rows=0, x_dtype=dtype, block_rows=block_rows, x=None, q=None, scale=None) == "OK"
    assert e4m3(M=0, x=None, xs=None, y=None, y_dtype=dtype) == "OK"
    assert grouped(M=0, x=None, y=None, y_dtype=dtype) == "OK"
    assert grouped_e4m3(M=0, x=None, xs=None, y=None, y_dtype=dtype) == "OK"
    assert e4m3(M=0, w=None) == grouped(M=0, w=None) == grouped(M=0, offsets=None) == "INVALID_ARGUMENT"
    assert e4m3(M=0, ws=None) == grouped_e4m3(M=0, offsets=None) == "INVALID_ARGUMENT"
    assert e4m3(M=0, x=None, y=None, act=2) == quantize(rows=0, x=None, cols=0) == "INVALID_ARGUMENT"


def test_groups_are_counted_before_anything_else():
    assert grouped(groups=1025, M=0) == grouped_e4m3(groups=1025, M=0) == "UNSUPPORTED"


def test_kernel_status_needs_a_device():
    # without a device the error word that every product records in cannot be had, and that is an error
    assert name(tb.lib.tsfm_kernel_status(None)) == ("OK" if has_gpu() else "NO_DEVICE")
