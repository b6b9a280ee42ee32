"""Calls that the fp8 entry points refuse before they touch the GPU."""
import ctypes

import numpy as np
import pytest

import fp8_util as U
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, MLK_Q8, NativeError

P = 1 << 20  # stands for an address; the refusals below never look at it


def quantize(dtype=MLK_F32, x=P, rows=4, cols=256, block_rows=1, q=P, s=P):
    native.quantize_fp8(dtype, x, rows, cols, block_rows, q, s)


def norm(dtype=MLK_F32, x=P, norm_w=P, rows=4, cols=256, q=P, s=P, **more):
    native.rmsnorm_fp8(dtype, x, norm_w, rows, cols, q, s, **more)


def swiglu(dtype=MLK_F32, x=P, rows=4, width=256, q=P, s=P):
    native.swiglu_fp8(dtype, x, rows, width, q, s)


def matmul(dtype=MLK_F32, w=P, ws=P, x=P, xs=P, y=P, out=64, inp=256, rows=4, resid=None):
    native.matmul_fp8(dtype, w, ws, x, xs, y, out, inp, rows, resid=resid)


def grouped(dtype=MLK_F32, w=P, ws=P, x=P, xs=P, y=P, out=64, inp=256, groups=3, offsets=P,
            entries=4, **more):
    native.matmul_fp8_grouped(dtype, w, ws, x, xs, y, out, inp, groups, offsets, entries, **more)


@pytest.mark.parametrize("call,bad,says", [
    (quantize, dict(dtype=MLK_Q8), "type"),
    (quantize, dict(dtype=-1), "type"),
    (quantize, dict(rows=-1), "rows"),
    (quantize, dict(cols=0), "cols"),
    (quantize, dict(block_rows=64), "block_rows"),
    (quantize, dict(cols=(1 << 30) + 1), "cols"),
    (norm, dict(cols=(1 << 31) - 1), "cols"),
    (swiglu, dict(width=(1 << 31) - 1), "width"),
    (matmul, dict(inp=(1 << 30) + 1), "in_width"),
    (matmul, dict(out=(1 << 31) - 1), "out_width"),
    (grouped, dict(inp=(1 << 31) - 1), "in_width"),
    (grouped, dict(out=0), "out_width"),
    (quantize, dict(x=None), "x is null"),
    (quantize, dict(q=None), "q is null"),
    (quantize, dict(s=None), "s is null"),
    (quantize, dict(x=P + 2), "x is not aligned"),
    (quantize, dict(dtype=MLK_BF16, x=P + 1), "x is not aligned"),
    (quantize, dict(s=P + 1), "s is not aligned"),
    (norm, dict(dtype=4), "type"),
    (norm, dict(rows=-2), "rows"),
    (norm, dict(cols=-1), "cols"),
    (norm, dict(eps=-1e-6), "eps"),
    (norm, dict(eps=float("nan")), "eps"),
    (norm, dict(eps=float("inf")), "eps"),
    (norm, dict(norm_w=None), "norm_w is null"),
    (norm, dict(x=None), "x is null"),
    (norm, dict(resid=P + 2), "resid is not aligned"),
    (norm, dict(total=P + 3), "sum is not aligned"),
    (swiglu, dict(dtype=2), "type"),
    (swiglu, dict(width=0), "width"),
    (swiglu, dict(rows=-1), "rows"),
    (swiglu, dict(x=None), "gate_up is null"),
    (matmul, dict(dtype=MLK_Q8), "type"),
    (matmul, dict(out=0), "out_width"),
    (matmul, dict(inp=-3), "in_width"),
    (matmul, dict(rows=-1), "rows"),
    (matmul, dict(w=None), "w is null"),
    (matmul, dict(ws=None), "ws is null"),
    (matmul, dict(xs=P + 2), "xs is not aligned"),
    (matmul, dict(y=P + 2), "y is not aligned"),
    (matmul, dict(dtype=MLK_BF16, resid=P + 1), "resid is not aligned"),
    (grouped, dict(groups=0), "groups"),
    (grouped, dict(entries=-1), "entries"),
    (grouped, dict(x_rows=-1), "x_rows"),
    (grouped, dict(x_rows=3), "row for each entry"),
    (grouped, dict(x_rows=0, row_ids=P), "no rows"),
    (grouped, dict(offsets=None), "offsets is null"),
    (grouped, dict(offsets=P + 1), "offsets is not aligned"),
    (grouped, dict(row_ids=P + 2), "row_ids is not aligned"),
])
def test_refused(call, bad, says):
    with pytest.raises(NativeError, match=says):
        call(**bad)


@pytest.mark.parametrize("call,empty", [
    (quantize, dict(rows=0, x=None, q=None, s=None)),
    (norm, dict(rows=0, x=None, norm_w=None, q=None, s=None)),
    (swiglu, dict(rows=0, x=None, q=None, s=None)),
    (matmul, dict(rows=0, x=None, xs=None, y=None)),
    (grouped, dict(entries=0, x=None, xs=None, y=None)),
])
def test_nothing_to_do(call, empty):
    call(**empty)


@pytest.mark.parametrize("call", [quantize, norm, swiglu, matmul, grouped])
def test_without_a_device(call):
    """A full call reports the missing GPU, or the address that is none of its memory."""
    with pytest.raises(NativeError, match="no HIP device|not device memory"):
        call()


@pytest.mark.gpu
def test_host_memory_is_refused(device):
    x = np.zeros((4, 256), np.float32)
    q, s = native.DeviceBuffer(1024), native.DeviceBuffer(32)
    with pytest.raises(NativeError, match="x is not device memory"):
        quantize(x=x.ctypes.data, q=q, s=s)
    buf = ctypes.create_string_buffer(4 * 4 * 64 + 16)
    at = ctypes.addressof(buf) + -ctypes.addressof(buf) % 16
    d = native.DeviceBuffer(1 << 16)
    with pytest.raises(NativeError, match="y is not device memory"):
        matmul(w=d, ws=d, x=d, xs=d, y=at)


def test_codes_of_the_oracle():
    """The numpy codec agrees with itself: every code's value has that code, midpoints go
    to the even neighbour."""
    codes = np.array([c for c in range(256) if c & 0x7f != 0x7f], np.uint8)
    assert np.array_equal(U.encode(U.decode(codes)), codes)
    mags = U.decode(np.arange(127, dtype=np.uint8))
    mid = U.encode((mags[:-1] + mags[1:]) / 2)
    assert np.all(mid % 2 == 0) and mags.max() == 448.0
    assert U.step(448.0) == 32.0 and U.step(2.0 ** -9) == 2.0 ** -9
