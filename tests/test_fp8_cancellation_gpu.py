"""fp8 products whose loud columns cancel: what is left of the quiet ones beside them."""
import numpy as np
import pytest

import fp8_util as U
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32
from test_fp8_gpu import Out, put

pytestmark = pytest.mark.gpu

F32 = np.float32


def cancelling(rng, rows, out, inp):
    """x, xs, w, ws: in one of the eights of columns of each output +448 * 448 and
    -448 * 448 meet beside six products of 1 to 32; scales are powers of two."""
    eights = inp // 8
    x = U.encode(rng.integers(1, 9, (rows, inp)).astype(float))
    x[:, :8 * eights].reshape(rows, eights, 8)[:, :, :2] = 0x7e
    w = np.zeros((out, inp), np.uint8)
    at = (np.arange(out) * 7 + rng.integers(eights)) % eights
    w[np.arange(out)[:, None], 8 * at[:, None] + np.arange(8)] = np.concatenate(
        [np.tile([0x7e, 0xfe], (out, 1)), U.encode(rng.integers(1, 5, (out, 6)).astype(float))], 1)
    xs = 2.0 ** rng.integers(-3, 4, (rows, U.blocks(inp)))
    ws = 2.0 ** rng.integers(-3, 4, (U.blocks(out), U.blocks(inp)))
    return x, xs.astype(F32), w, ws.astype(F32)


def run(dtype, rows, out, inp):
    """(y, what it should be, the magnitudes added, the sum of the eights' largest) of a
    few rows."""
    rng = np.random.default_rng(rows + out + inp)
    x, xs, w, ws = cancelling(rng, rows, out, inp)
    bufs = [put(a) for a in (w, ws, x, xs)]
    y = Out(rows * out * (2 if dtype == MLK_BF16 else 4))
    native.matmul_fp8(dtype, *[b[1] for b in bufs], y.ptr, out, inp, rows)
    got = y.get(np.uint16 if dtype == MLK_BF16 else F32, (rows, out))
    got = (U.from_bf16(got) if dtype == MLK_BF16 else got).astype(np.float64)
    at = np.union1d(rng.integers(0, rows, min(rows, 6)), [0, rows - 1])
    return got[at], *U.product(x[at], xs[at], w, ws)


# by the kernel choice's model of their times: streams, then the tiles of 64 x 64,
# 128 x 128 and (bf16 outputs) 256 x 256, with and without whole 16-byte pieces
FEW = [(1, 272, 528), (5, 272, 2064), (16, 300, 525), (40, 640, 11264)]
MANY = [(700, 900, 528), (1600, 2100, 532), (1746, 3278, 144), (1746, 3278, 149), (2550, 6150, 528)]


@pytest.mark.parametrize("rows,out,inp", FEW + MANY)
def test_f32_outputs_keep_f32_sums(device, rows, out, inp):
    got, want, mass, top = run(MLK_F32, rows, out, inp)
    off = np.abs(got - want)
    assert np.all(off <= U.product_tolerance(want, mass, top, inp, False)), off.max()


@pytest.mark.parametrize("rows,out,inp", FEW)
def test_bf16_outputs_of_few_rows_keep_f32_sums(device, rows, out, inp):
    got, want, mass, top = run(MLK_BF16, rows, out, inp)
    room = U.product_tolerance(want, mass, top, inp, False)
    room = room + U.HALF_BF16 * (np.abs(want) + room)
    assert np.all(np.abs(got - want) <= room)


@pytest.mark.parametrize("rows,out,inp", MANY)
def test_bf16_outputs_of_many_rows_lose_no_more_than_told(device, rows, out, inp):
    """2^-10 of the sum of the largest product of each eight columns, beside the f32 sums'
    own error and the rounding."""
    got, want, mass, top = run(MLK_BF16, rows, out, inp)
    room = U.product_tolerance(want, mass, top, inp, False) + 2.0 ** -10 * top
    room = room + U.HALF_BF16 * (np.abs(want) + room)
    assert np.all(np.abs(got - want) <= room)
