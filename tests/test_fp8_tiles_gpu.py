"""The tile kernels of the fp8 products where the small products do not take them: many
steps of columns, gathered and malformed rows, values that are not finite, rows past 32
bits.  By the kernel choice's model of their times the sizes here run on the tiles that
are named beside them (bf16 / f32 outputs where they differ)."""
import numpy as np
import pytest

import fp8_util as U
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32
from test_fp8_gpu import Out, check_matmul, fp8_matrix, put, run_grouped, zeros

pytestmark = pytest.mark.gpu

F32 = np.float32
TYPES = pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])


# ---- more columns than two groups of 8 steps of scales -------------------------------


@TYPES
@pytest.mark.parametrize("rows,out,inp", [
    (900, 900, 2064),     # 64 x 64 (f32: a stream of 64 x 64)
    (1000, 1200, 2071),   # 64 x 64 through registers
    (1746, 3278, 2064),   # 128 x 128
    (2550, 6150, 2064),   # 256 x 256 / 128 x 128
    (2550, 6150, 2071),   # 128 x 128 through registers
    (2550, 6150, 1024),   # 8 steps: the last group of scales ends with the columns
    (2550, 6150, 1152)])  # 9
def test_scale_groups(device, dtype, rows, out, inp):
    check_matmul(dtype, rows, out, inp, with_resid=inp == 2064)


@TYPES
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts,out,inp", [
    ([700, 0, 301, 999], 1000, 2064),     # 64 x 64
    ([1500, 2, 700, 798], 900, 2071),     # 64 x 64 through registers
    ([4000, 1, 4999], 1030, 2064),        # 256 x 256 / 128 x 128
    ([3000, 257, 0, 2743], 1200, 2071)])  # 128 x 128 through registers
def test_scale_groups_of_grouped_products(device, dtype, gather, counts, out, inp):
    run_grouped(np.random.default_rng(out + inp), dtype, counts, out, inp, gather, spare=3)


# ---- rows that are not there ---------------------------------------------------------

# 64 x 64, the same through registers, 128 x 128, 256 x 256 / 128 x 128
GROUPED = [([150, 0, 450], 640, 256), ([1300, 700, 1000], 640, 258), ([2000, 1, 1999], 1100, 400),
           ([4000, 1, 4999], 1030, 2064)]


@TYPES
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts,out,inp", GROUPED)
def test_grouped_from_a_later_row(device, dtype, gather, counts, out, inp):
    run_grouped(np.random.default_rng(5), dtype, counts, out, inp, gather, first=6, spare=3)


@TYPES
@pytest.mark.parametrize("counts,out,inp", GROUPED)
def test_grouped_row_ids_out_of_range_are_nan(device, dtype, counts, out, inp):
    rng = np.random.default_rng(6)
    n = sum(counts)
    ids = rng.integers(0, n // 3, n)
    bad = np.union1d(rng.integers(0, n, 20), [0, 3, n - 1])
    ids[bad] = rng.choice([-1, n // 3, 2 ** 31 - 1, -2 ** 31], bad.size)
    got = run_grouped(rng, dtype, counts, out, inp, True, ids=ids)
    assert np.isnan(got[bad]).all() and np.isfinite(np.delete(got, bad, 0)).all()


@TYPES
@pytest.mark.parametrize("counts,out,inp", GROUPED)
@pytest.mark.parametrize("offsets", [
    [0.0, 1.0, 0.0, 1.0], [0.0, 0.7, 0.3, 0.5], [-0.1, 0.3, 0.6, 1.0], [0.0, 0.3, 9.0, 9.0],
    [1.0, 0.6, 0.3, 0.0], [1.3, 1.3, 1.3, 1.3], None])
def test_grouped_bad_offsets_stay_in_range(device, dtype, counts, out, inp, offsets):
    """Groups that overlap, decrease or leave the entries: nothing outside y is written
    (the guards), whatever its rows become."""
    n, rng = sum(counts), np.random.default_rng(7)
    ends = [-(1 << 31), (1 << 31) - 1, 0, n] if offsets is None else [int(o * n) for o in offsets]
    bufs = [put(rng.integers(0, 0x70, shape, np.uint8)) for shape in ((3, out, inp), (n, inp))]
    scales = [put(np.ones(shape, F32)) for shape in ((3, U.blocks(out), U.blocks(inp)),
                                                     (n, U.blocks(inp)))]
    at = put(np.array(ends, np.int32))
    y = Out(n * out * (2 if dtype == MLK_BF16 else 4))
    native.matmul_fp8_grouped(dtype, bufs[0][1], scales[0][1], bufs[1][1], scales[1][1], y.ptr,
                              out, inp, 3, at[1], n)
    y.get(np.uint8, -1)


# ---- values that are not finite ------------------------------------------------------


@TYPES
@pytest.mark.parametrize("lead", [0, 5])
@pytest.mark.parametrize("rows,out,inp", [(700, 900, 528), (1746, 3278, 144), (2550, 6150, 528)])
def test_nan_stays_in_its_row(device, dtype, rows, out, inp, lead):
    """NaN codes, and a scale of infinity, reach the outputs of their row or column only
    (64 x 64, 128 x 128, 256 x 256 / 128 x 128, each through registers too)."""
    rng = np.random.default_rng(3)
    w, ws = fp8_matrix(rng, out, inp, block_rows=128)
    x, xs = fp8_matrix(rng, rows, inp, block_rows=1)
    x[2, inp - 1], x[rows - 1, 0], w[out - 2, 0], w[5, 17] = 0x7f, 0xff, 0xff, 0x7f
    xs[300, 1] = np.inf
    bufs = [put(a, k) for a, k in ((w, lead), (ws, 0), (x, lead), (xs, 0))]
    y = Out(rows * out * (2 if dtype == MLK_BF16 else 4))
    native.matmul_fp8(dtype, *[b[1] for b in bufs], y.ptr, out, inp, rows)
    got = y.get(np.uint16 if dtype == MLK_BF16 else F32, (rows, out))
    got = U.from_bf16(got) if dtype == MLK_BF16 else got
    bad = np.zeros(got.shape, bool)
    bad[[2, 300, rows - 1]], bad[:, [5, out - 2]] = True, True
    assert not np.isfinite(got[bad]).any() and np.isfinite(got[~bad]).all()


# ---- past 32 bits --------------------------------------------------------------------


@TYPES
@pytest.mark.parametrize("x_rows", [1_900_000, 2_200_000])  # 64 x 64; through registers
def test_gathered_rows_past_32_bits(device, dtype, x_rows):
    inp, out, entries = 2048, 96, 20_000
    rng = np.random.default_rng(x_rows)
    where = np.array([0, 1 << 20, (1 << 20) + 1, x_rows - 2, x_rows - 1])
    rows, scales = fp8_matrix(rng, 5, inp, block_rows=1)
    w, ws = fp8_matrix(rng, 2, out, inp, block_rows=128)
    x, xs = zeros(x_rows * inp), zeros(x_rows * U.blocks(inp) * 4)
    for i, r in enumerate(where):
        x.upload(rows[i], int(r) * inp)
        xs.upload(scales[i], int(r) * U.blocks(inp) * 4)
    take = rng.integers(0, 5, entries)
    ends = np.array([0, entries // 3, entries], np.int32)
    bufs = [put(a) for a in (w, ws, ends, where[take].astype(np.int32))]
    y = Out(entries * out * (2 if dtype == MLK_BF16 else 4))
    native.matmul_fp8_grouped(dtype, bufs[0][1], bufs[1][1], x.ptr, xs.ptr, y.ptr, out, inp, 2,
                              bufs[2][1], entries, row_ids=bufs[3][1], x_rows=x_rows)
    got = y.get(np.uint16 if dtype == MLK_BF16 else F32, (entries, out))
    got = (U.from_bf16(got) if dtype == MLK_BF16 else got).astype(np.float64)
    for g in range(2):
        at = slice(ends[g], ends[g + 1])
        want, *parts = U.product(rows, scales, w[g], ws[g])
        room = U.product_tolerance(want, *parts, inp, dtype == MLK_BF16)
        assert np.all(np.abs(got[at] - want[take[at]]) <= room[take[at]])
