"""The fp8 entry points against their formulas in 64 bits."""
import threading

import numpy as np
import pytest

import fp8_util as U
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, DeviceBuffer

pytestmark = pytest.mark.gpu

F32 = np.float32
GUARD = 64  # bytes behind an output that stay as they are


class Out:
    """An output of `nbytes` behind `lead` bytes, and guards on both sides."""

    def __init__(self, nbytes, lead=0, fill=0xA5):
        self.n, self.lead, self.fill = nbytes, lead + GUARD, fill
        self.buf = DeviceBuffer.from_array(np.full(nbytes + lead + 2 * GUARD, fill, np.uint8))
        self.ptr = self.buf.ptr + self.lead

    def get(self, dtype, shape):
        raw = self.buf.download(np.uint8)
        assert np.all(raw[:self.lead] == self.fill) and np.all(raw[self.lead + self.n:] == self.fill)
        return raw[self.lead:self.lead + self.n].copy().view(dtype).reshape(shape)


def put(array, lead=0):
    """(buffer, address) of an array `lead` bytes into an allocation."""
    array = np.ascontiguousarray(array)
    buf = DeviceBuffer(array.nbytes + lead)
    if array.nbytes:
        buf.upload(array.view(np.uint8).reshape(-1), lead)
    return buf, buf.ptr + lead


def typed(dtype, v):
    """Values as `dtype` holds them: (what is uploaded, the same as f32)."""
    if dtype == MLK_BF16:
        bits = U.to_bf16(v)
        return bits, U.from_bf16(bits)
    return v.astype(F32), v.astype(F32)


def rows_of(rng, rows, cols, loud=30.0):
    v = rng.standard_normal((rows, cols))
    return v * np.where(rng.random(cols) < 0.01, loud, 1.0)


# ---- quantising -----------------------------------------------------------------


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,cols,lead", [
    (1, 1, 0), (1, 127, 0), (3, 128, 0), (5, 129, 0), (130, 304, 0), (257, 2048, 0),
    (16, 136, 4), (1, 20001, 0), (300, 8, 0), (128, 128, 16)])
def test_quantize(device, dtype, block_rows, rows, cols, lead):
    rng = np.random.default_rng(rows * 1000 + cols)
    raw, v = typed(dtype, rows_of(rng, rows, cols))
    buf, at = put(raw, lead)
    q, s = Out(rows * cols, lead), Out(4 * (rows if block_rows == 1 else U.blocks(rows)) * U.blocks(cols))
    native.quantize_fp8(dtype, at, rows, cols, block_rows, q.ptr, s.ptr)
    code, scale = U.quantize(v, block_rows)
    np.testing.assert_array_equal(s.get(F32, scale.shape), scale)
    np.testing.assert_array_equal(q.get(np.uint8, (rows, cols)), code)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(device, block_rows):
    """Blocks of zeros, subnormals, huge values, values next to the borders of codes,
    a NaN (it alone) and an infinity (its whole block)."""
    v = np.zeros((6, 256), F32)
    v[0, 3] = -0.0
    v[1, :128] = np.linspace(1e-44, 1e-41, 128)
    v[1, 128:] = np.linspace(-3.4e38, 3.4e38, 128)
    mags = U.decode(np.arange(127, dtype=np.uint8))
    mid = ((mags[:-1] + mags[1:]) / 2).astype(F32)
    v[2, :126], v[2, 127] = mid, 448.0
    v[2, 128:254], v[2, 255] = np.nextafter(mid, F32(0)), 448.0
    v[3, :126], v[3, 127] = -np.nextafter(mid, F32(1e9)), 448.0
    v[4] = 1.0
    v[4, 7] = np.nan
    v[5] = 2.0
    v[5, 130] = -np.inf
    if block_rows == 128:
        v = np.concatenate([np.pad(r[None], ((0, 127), (0, 0))) for r in v])
    rows, cols = v.shape
    buf, at = put(v)
    q, s = Out(v.size), Out(4 * (rows // block_rows) * 2)
    native.quantize_fp8(MLK_F32, at, rows, cols, block_rows, q.ptr, s.ptr)
    want_code, want_scale = U.quantize(v, block_rows)
    code, scale = q.get(np.uint8, v.shape), s.get(F32, want_scale.shape)
    np.testing.assert_array_equal(scale, want_scale)
    got, want = U.decode(code), U.decode(want_code)
    np.testing.assert_array_equal(got, want)  # (NaN equal to NaN, of either sign)
    with np.errstate(invalid="ignore"):
        back = got * U.spread(scale, rows, cols, block_rows)
    r4, r5 = 4 * block_rows, 5 * block_rows
    assert np.isnan(back[r4, 7]) and np.isfinite(np.delete(back[r4], 7)).all()
    assert np.isnan(back[r5, 128:]).all() and np.isfinite(back[r5, :128]).all()


# ---- norm -----------------------------------------------------------------------


@pytest.mark.parametrize("keep", ["no", "apart", "x", "resid"])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 100), (3, 2048), (2, 2056), (5, 4100), (3, 8192),
                                       (2, 8200), (3, 16384), (2, 20001), (300, 640)])
def test_rmsnorm(device, dtype, rows, cols, keep):
    rng = np.random.default_rng(rows + 7 * cols)
    size = 2 if dtype == MLK_BF16 else 4
    with_resid = keep != "no" or cols % 2 == 0
    xr, x = typed(dtype, rng.standard_normal((rows, cols)))
    rr, r = typed(dtype, rows_of(rng, rows, cols))
    w = (1.0 + 0.2 * rng.standard_normal(cols)).astype(F32)
    xb, rb = Out(rows * cols * size), Out(rows * cols * size)
    xb.buf.upload(xr.view(np.uint8).reshape(-1), xb.lead)
    rb.buf.upload(rr.view(np.uint8).reshape(-1), rb.lead)
    wb, wat = put(w)
    q, s, total = Out(rows * cols), Out(4 * rows * U.blocks(cols)), Out(rows * cols * size)
    into = {"no": None, "apart": total, "x": xb, "resid": rb}[keep]
    native.rmsnorm_fp8(dtype, xb.ptr, wat, rows, cols, q.ptr, s.ptr,
                       resid=rb.ptr if with_resid else None, total=into and into.ptr, eps=1e-5)
    h = x + r if with_resid else x
    raw = U.to_bf16(h) if dtype == MLK_BF16 else h
    if into:
        np.testing.assert_array_equal(into.get(raw.dtype, raw.shape), raw)
    h = (U.from_bf16(raw) if dtype == MLK_BF16 else raw).astype(np.float64)
    v = h / np.sqrt((h * h).mean(1, keepdims=True) + F32(1e-5).astype(np.float64)) * w
    # the sum of squares: at most cols / 256 + 10 f32 additions deep, halved by the root;
    # the mean, eps, root, quotient and two products: 6 roundings
    delta = ((cols / 256 + 18) / 2 + 6) * U.HALF_F32
    U.check_codes(q.get(np.uint8, (rows, cols)), s.get(F32, (rows, U.blocks(cols))), v, delta)


def test_rmsnorm_special_rows(device):
    """A row of zeros, one with a NaN, one with an infinity, one too small to square."""
    h = np.ones((4, 300), F32)
    h[0] = 0.0
    h[1, 5] = np.nan
    h[2, 290] = np.inf
    h[3] = 1e-30
    (xb, x), (wb, w) = put(h), put(np.ones(300, F32))
    q, s = Out(1200), Out(4 * 4 * 3)
    native.rmsnorm_fp8(MLK_F32, x, w, 4, 300, q.ptr, s.ptr, eps=1e-6)
    v = U.decode(q.get(np.uint8, (4, 300))) * U.spread(s.get(F32, (4, 3)).astype(float), 4, 300, 1)
    assert np.all(v[0] == 0) and np.isnan(v[1]).all()
    assert np.isnan(v[2, 290]) and np.all(v[2, :256] == 0)
    np.testing.assert_allclose(v[3], 1e-27, rtol=2.0 ** -4)


# ---- SwiGLU -----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 127), (2, 128), (37, 1408), (5, 1001), (700, 24)])
def test_swiglu(device, dtype, rows, width):
    rng = np.random.default_rng(rows * width)
    raw, v = typed(dtype, 3.0 * rng.standard_normal((rows, 2 * width)))
    buf, at = put(raw)
    q, s = Out(rows * width), Out(4 * rows * U.blocks(width))
    native.swiglu_fp8(dtype, at, rows, width, q.ptr, s.ptr)
    g, u = v[:, :width].astype(np.float64), v[:, width:].astype(np.float64)
    # half places: 2^t 2 (one last place), its rest's product and sum 2, 1 + exp 1, the
    # reciprocal 2, the two products 2
    U.check_codes(q.get(np.uint8, (rows, width)), s.get(F32, (rows, U.blocks(width))),
                  g / (1.0 + np.exp(-g)) * u, 9 * U.HALF_F32)


def test_swiglu_far_gates(device):
    """Gates so far below zero that exp overflows give zeros, far above the up values;
    up values that g * u would take out of range stay finite."""
    g = np.array([[-1e4, -100.0, 100.0, 1e4, 3e38, -3e38, 2.0, 0.0]], F32)
    u = np.array([[1e30, 1e30, 1.0, 1.0, 1e-10, 1e-10, 1.5, 7.0]], F32)
    buf, at = put(np.concatenate([g, u], 1))
    q, s = Out(8), Out(4)
    native.swiglu_fp8(MLK_F32, at, 1, 8, q.ptr, s.ptr)
    v = U.decode(q.get(np.uint8, (1, 8))) * s.get(F32, (1, 1))
    want = np.array([[0, 0, 100, 1e4, 3e28, 0, 0, 0]])
    np.testing.assert_allclose(v, np.where(want < 1e20, 0, want), rtol=2.0 ** -4)


# ---- products ---------------------------------------------------------------------


def fp8_matrix(rng, *shape, block_rows, loud=30.0):
    """Codes and scales of normal values; a few columns of rows are loud."""
    *lead, rows, cols = shape
    v = rng.standard_normal(shape)
    if block_rows == 1:
        v = v * np.where(rng.random(cols) < 0.01, loud, 1.0)
    flat = v.reshape(-1, rows, cols)
    made = [U.quantize(m, block_rows) for m in flat]
    code = np.stack([m[0] for m in made]).reshape(shape)
    scale = np.stack([m[1] for m in made])
    return code, scale.reshape(*lead, *scale.shape[1:])


SHAPES = [
    (1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 300, 2048), (4, 2048, 1408), (5, 33, 4096),
    (15, 130, 272), (16, 128, 64), (17, 129, 1000), (31, 576, 512), (33, 64, 130), (64, 64, 128),
    (65, 257, 384), (100, 1000, 999), (127, 256, 1280), (128, 128, 256), (129, 384, 144),
    (200, 640, 1408), (256, 512, 640), (300, 272, 2064), (513, 260, 512), (1, 4096, 11264),
    (40, 48, 11264), (1000, 136, 264)]


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,out,inp", SHAPES)
def test_matmul(device, dtype, rows, out, inp):
    check_matmul(dtype, rows, out, inp, with_resid=(rows + out) % 2 == 0)


# By the kernel choice's model of their times each of these is the fastest on another
# shape of tile or stream; the last on one that bf16 outputs alone have.
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,out,inp", [
    (314, 401, 73), (20, 8200, 1000), (202, 2358, 66), (1095, 3766, 1039), (421, 200, 528),
    (1144, 215, 656), (686, 749, 4016), (40, 8200, 144), (1746, 3278, 144), (2550, 6150, 528)])
def test_matmul_of_each_kernel(device, dtype, rows, out, inp):
    check_matmul(dtype, rows, out, inp, with_resid=out < 800)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("lead_w,lead_x,lead_y", [(1, 0, 0), (0, 3, 0), (8, 8, 0), (0, 0, 4)])
@pytest.mark.parametrize("rows,out,inp", [(1, 64, 256), (20, 96, 512), (150, 260, 384)])
def test_matmul_unaligned(device, dtype, lead_w, lead_x, lead_y, rows, out, inp):
    check_matmul(dtype, rows, out, inp, True, lead_w, lead_x, lead_y)


def some_rows(rng, rows, size):
    """The rows that are checked: all, or of large products the last and some by chance."""
    if rows * size <= 5e8:
        return np.arange(rows)
    return np.union1d(rng.integers(0, rows, max(4, int(3e8 / size))), [0, rows - 1])


def check_matmul(dtype, rows, out, inp, with_resid, lead_w=0, lead_x=0, lead_y=0):
    rng = np.random.default_rng(rows * 7 + out * 3 + inp)
    w, ws = fp8_matrix(rng, out, inp, block_rows=128)
    x, xs = fp8_matrix(rng, rows, inp, block_rows=1)
    size = 2 if dtype == MLK_BF16 else 4
    (wb, wat), (xb, xat), (wsb, wsat), (xsb, xsat) = put(w, lead_w), put(x, lead_x), put(ws), put(xs)
    resid, rb, rat = None, None, None
    if with_resid:
        raw, resid = typed(dtype, 10.0 * rng.standard_normal((rows, out)))
        rb, rat = put(raw, lead_y)
        resid = resid.astype(np.float64)
    y = Out(rows * out * size, lead_y)
    native.matmul_fp8(dtype, wat, wsat, xat, xsat, y.ptr, out, inp, rows, resid=rat)
    got = y.get(np.uint16 if dtype == MLK_BF16 else F32, (rows, out))
    again = Out(rows * out * size, lead_y)
    native.matmul_fp8(dtype, wat, wsat, xat, xsat, again.ptr, out, inp, rows, resid=rat)
    np.testing.assert_array_equal(again.get(got.dtype, got.shape), got)
    if with_resid:  # y in the residual's own memory
        native.matmul_fp8(dtype, wat, wsat, xat, xsat, rat, out, inp, rows, resid=rat)
        np.testing.assert_array_equal(
            rb.download(np.uint8)[lead_y:].view(got.dtype).reshape(got.shape), got)
    got = (U.from_bf16(got) if dtype == MLK_BF16 else got).astype(np.float64)
    assert np.isfinite(got).all()
    at = some_rows(rng, rows, out * inp)
    resid = None if resid is None else resid[at]
    want, *parts = U.product(x[at], xs[at], w, ws)
    room = U.product_tolerance(want, *parts, inp, dtype == MLK_BF16, resid)
    off = np.abs(got[at] - (want if resid is None else want + resid))
    assert np.all(off <= room), (np.max(off / room), np.argmax(off / room))


def test_matmul_nan_stays_in_its_row(device):
    """NaN codes, and a scale of infinity, reach the outputs of their row or column only."""
    rng = np.random.default_rng(3)
    for rows in (5, 200):
        w, ws = fp8_matrix(rng, 260, 300, block_rows=128)
        x, xs = fp8_matrix(rng, rows, 300, block_rows=1)
        x[2, 299], w[258, 0] = 0x7f, 0xff
        xs[4, 1] = np.inf
        bufs = [put(a) for a in (w, ws, x, xs)]
        y = Out(rows * 260 * 4)
        native.matmul_fp8(MLK_F32, *[b[1] for b in bufs], y.ptr, 260, 300, rows)
        got = y.get(F32, (rows, 260))
        bad = np.zeros_like(got, bool)
        bad[2], bad[4], bad[:, 258] = True, True, True
        assert not np.isfinite(got[bad]).any() and np.isfinite(got[~bad]).all()


# ---- grouped products ---------------------------------------------------------------


def run_grouped(rng, dtype, counts, out, inp, gather, first=0, spare=0, ids=None, lead=0,
                offsets=None):
    """One call on groups of `counts` rows, and its check."""
    groups, n = len(counts), int(np.sum(counts))
    ends = first + np.concatenate([[0], np.cumsum(counts)])
    entries = first + n + spare
    x_rows = max(1, n // 3) if gather else max(entries, 1)
    w, ws = fp8_matrix(rng, groups, out, inp, block_rows=128)
    x, xs = fp8_matrix(rng, x_rows, inp, block_rows=1)
    if gather and ids is None:
        ids = rng.integers(0, x_rows, entries)
    size = 2 if dtype == MLK_BF16 else 4
    bufs = [put(a, k) for a, k in ((w, lead), (ws, 0), (x, lead), (xs, 0))]
    ob = put(np.asarray(ends if offsets is None else offsets, np.int32))
    ib = put(np.asarray(ids, np.int32)) if gather else (None, None)
    y = Out(entries * out * size, fill=0x5A)
    native.matmul_fp8_grouped(dtype, *[b[1] for b in bufs], y.ptr, out, inp, groups, ob[1],
                              entries, row_ids=ib[1], x_rows=x_rows)
    raw = y.get(np.uint16 if dtype == MLK_BF16 else F32, (entries, out))
    got = (U.from_bf16(raw) if dtype == MLK_BF16 else raw).astype(np.float64)
    if offsets is not None:
        return got
    outside = np.concatenate([raw[:first], raw[first + n:]])
    assert np.all(outside.view(np.uint8) == 0x5A)
    for g in range(groups):
        at = ends[g] + some_rows(rng, counts[g], out * inp * groups)
        src = np.asarray(ids)[at] if gather else at
        ok = (src >= 0) & (src < x_rows)
        assert np.isnan(got[at[~ok]]).all()
        at, src = at[ok], src[ok]
        want, *parts = U.product(x[src], xs[src], w[g], ws[g])
        room = U.product_tolerance(want, *parts, inp, dtype == MLK_BF16)
        off = np.abs(got[at] - want)
        assert np.all(off <= room), (g, np.max(off / room))
    return got


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("counts,out,inp,spare", [
    ([1], 16, 128, 0), ([0, 0, 3, 0], 48, 256, 5), ([1, 1, 1, 1, 1], 130, 2048, 0),
    ([16, 0, 17, 1], 128, 129, 0), ([40, 3, 0, 64, 65], 272, 512, 7),
    ([128, 129, 1, 0, 255], 256, 384, 0), ([300, 2], 640, 144, 1), ([0, 0], 32, 64, 4),
    ([5] * 70, 64, 256, 0), ([0] * 130 + [9], 32, 128, 0), ([33] * 20, 160, 1000, 2)])
def test_grouped(device, dtype, counts, out, inp, spare, gather):
    rng = np.random.default_rng(len(counts) * 31 + out)
    run_grouped(rng, dtype, counts, out, inp, gather, spare=spare)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("groups,each,out,inp", [
    (5, 167, 545, 65), (8, 424, 1116, 272), (8, 167, 362, 1984), (4, 372, 150, 1088),
    (5, 900, 835, 1222), (32, 230, 2048, 272), (270, 60, 130, 64), (300, 40, 130, 66)])
def test_grouped_of_each_kernel(device, dtype, groups, each, out, inp, gather):
    rng = np.random.default_rng(groups + each)
    counts = rng.multinomial(groups * each, np.full(groups, 1.0 / groups))
    run_grouped(rng, dtype, list(counts), out, inp, gather, spare=3)


@pytest.mark.parametrize("counts", [[4, 0, 9], [70, 150, 3]])
def test_grouped_from_a_later_row(device, counts):
    """Rows before offsets[0] stay as they are, as those behind the last group."""
    run_grouped(np.random.default_rng(5), MLK_F32, counts, 144, 256, True, first=6, spare=3)


@pytest.mark.parametrize("counts", [[4, 0, 9], [70, 150, 3]])
@pytest.mark.parametrize("lead", [0, 5])
def test_grouped_row_ids_out_of_range_are_nan(device, counts, lead):
    rng = np.random.default_rng(6)
    n = sum(counts)
    ids = rng.integers(0, n // 3, n)
    ids[0], ids[3], ids[n - 1] = -1, n // 3, 2 ** 31 - 1
    run_grouped(rng, MLK_F32, counts, 144, 256, True, ids=ids, lead=lead)


@pytest.mark.parametrize("offsets", [
    [0, 50, 20, 30], [-5, 10, 20, 30], [0, 10, 1 << 30, 1 << 30], [30, 20, 10, 0],
    [-(1 << 31), (1 << 31) - 1, 0, 30], [40, 40, 40, 40],
    [5, -(1 << 31), 20, 30]])
def test_grouped_bad_offsets_stay_in_range(device, offsets):
    """Offsets that decrease or leave the entries: nothing outside y is written (the
    guards), whatever rows are left out."""
    run_grouped(np.random.default_rng(7), MLK_F32, [10, 10, 10], 64, 256, False, offsets=offsets)


# ---- past 32 bits -------------------------------------------------------------------


def zeros(nbytes):
    buf = DeviceBuffer(nbytes)
    buf.zero()
    return buf


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("x_rows", [1_900_000, 2_200_000])  # codes up to 3.9e9 and 4.5e9 bytes in
@pytest.mark.parametrize("entries", [5, 300])
def test_grouped_rows_past_32_bits(device, dtype, x_rows, entries):
    inp, out = 2048, 96
    rng = np.random.default_rng(x_rows + entries)
    where = np.array([0, 1 << 20, (1 << 20) + 1, x_rows - 2, x_rows - 1])
    rows, scales = fp8_matrix(rng, 5, inp, block_rows=1)
    w, ws = fp8_matrix(rng, 2, out, inp, block_rows=128)
    x, xs = zeros(x_rows * inp), zeros(x_rows * U.blocks(inp) * 4)
    for i, r in enumerate(where):
        x.upload(rows[i], int(r) * inp)
        xs.upload(scales[i], int(r) * U.blocks(inp) * 4)
    take = rng.integers(0, 5, entries)
    ends = np.array([0, entries // 2, entries], np.int32)
    bufs = [put(a) for a in (w, ws, ends, where[take].astype(np.int32))]
    size = 2 if dtype == MLK_BF16 else 4
    y = Out(entries * out * size)
    native.matmul_fp8_grouped(dtype, bufs[0][1], bufs[1][1], x.ptr, xs.ptr, y.ptr, out, inp, 2,
                              bufs[2][1], entries, row_ids=bufs[3][1], x_rows=x_rows)
    got = y.get(np.uint16 if dtype == MLK_BF16 else F32, (entries, out))
    got = (U.from_bf16(got) if dtype == MLK_BF16 else got).astype(np.float64)
    for g in range(2):
        at = slice(ends[g], ends[g + 1])
        want, *parts = U.product(rows[take[at]], scales[take[at]], w[g], ws[g])
        assert np.all(np.abs(got[at] - want) <=
                      U.product_tolerance(want, *parts, inp, dtype == MLK_BF16))


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
def test_matmul_outputs_past_32_bits(device, dtype):
    rows, out, inp = 800_000, 4096, 16  # 3.3e9 outputs
    size = 2 if dtype == MLK_BF16 else 4
    rng = np.random.default_rng(8)
    where = np.array([0, (1 << 19) - 1, 1 << 19, rows - 1])
    x, xs = fp8_matrix(rng, 4, inp, block_rows=1)
    w, ws = fp8_matrix(rng, out, inp, block_rows=128)
    xb, xsb, y = zeros(rows * inp), zeros(rows * 4), zeros(rows * out * size)
    for i, r in enumerate(where):
        xb.upload(x[i], int(r) * inp)
        xsb.upload(xs[i], int(r) * 4)
    (wb, wat), (wsb, wsat) = put(w), put(ws)
    native.matmul_fp8(dtype, wat, wsat, xb.ptr, xsb.ptr, y.ptr, out, inp, rows)
    want, *parts = U.product(x, xs, w, ws)
    room = U.product_tolerance(want, *parts, inp, dtype == MLK_BF16)
    for i, r in enumerate(where):
        got = y.download(np.uint16 if dtype == MLK_BF16 else F32, out, int(r) * out * size)
        got = (U.from_bf16(got) if dtype == MLK_BF16 else got).astype(np.float64)
        assert np.all(np.abs(got - want[i]) <= room[i])
    for r in (1, rows - 2):  # rows of zeros between them
        assert not y.download(np.uint8, out * size, r * out * size).any()


@pytest.mark.parametrize("what", ["rows", "matrix", "norm", "swiglu"])
def test_rows_past_32_bits(device, what):
    rows, cols = 640_000, 4096  # 2.6e9 values, 5.2e9 bytes of bf16
    rng = np.random.default_rng(9)
    width = cols * (2 if what == "swiglu" else 1)
    where = np.array([0, (1 << 19) - 1, 1 << 19, rows - 1])
    raw, v = typed(MLK_BF16, rows_of(rng, 4, width))
    x, q = zeros(rows * width * 2), DeviceBuffer(rows * cols)
    per = U.blocks(cols)
    s = DeviceBuffer((U.blocks(rows) if what == "matrix" else rows) * per * 4)
    for i, r in enumerate(where):
        x.upload(raw[i], int(r) * width * 2)
    norm = put(np.ones(cols, F32))
    if what == "rows":
        native.quantize_fp8(MLK_BF16, x.ptr, rows, cols, 1, q.ptr, s.ptr)
    elif what == "matrix":
        native.quantize_fp8(MLK_BF16, x.ptr, rows, cols, 128, q.ptr, s.ptr)
    elif what == "norm":
        native.rmsnorm_fp8(MLK_BF16, x.ptr, norm[1], rows, cols, q.ptr, s.ptr)
    else:
        native.swiglu_fp8(MLK_BF16, x.ptr, rows, cols, q.ptr, s.ptr)
    v = v.astype(np.float64)
    for i, r in enumerate(where):
        code = q.download(np.uint8, cols, int(r) * cols)[None]
        at = int(r) // (128 if what == "matrix" else 1)
        scale = s.download(F32, per, at * per * 4)[None]
        if what == "rows":
            one, sc = U.quantize(v[i:i + 1].astype(F32), 1)
            np.testing.assert_array_equal(code, one)
            np.testing.assert_array_equal(scale, sc)
        elif what == "matrix":  # the rows of one block are one below the other
            near = v[(where // 128) == at].astype(F32)
            one, sc = U.quantize(near, 128)
            np.testing.assert_array_equal(scale, sc)
            mine = np.flatnonzero(where[where // 128 == at] == r)[0]
            np.testing.assert_array_equal(code[0], one[mine])
        elif what == "norm":
            h = v[i:i + 1]
            h = h / np.sqrt((h * h).mean(1, keepdims=True) + F32(1e-5).astype(np.float64))
            U.check_codes(code, scale, h, ((cols / 256 + 18) / 2 + 6) * U.HALF_F32)  # as above
        else:
            g, u = v[i:i + 1, :cols], v[i:i + 1, cols:]
            U.check_codes(code, scale, g / (1.0 + np.exp(-g)) * u, 9 * U.HALF_F32)


# ---- calls at once, and the operators one after the other ---------------------------


def test_calls_of_two_threads(device):
    rng = np.random.default_rng(9)
    jobs = []
    for rows in (3, 150):
        w, ws = fp8_matrix(rng, 320, 512, block_rows=128)
        x, xs = fp8_matrix(rng, rows, 512, block_rows=1)
        bufs = [put(a) for a in (w, ws, x, xs)]
        jobs.append((rows, bufs, [Out(rows * 320 * 4) for _ in range(20)], U.product(x, xs, w, ws)))

    def go(rows, bufs, outs):
        for y in outs:
            native.matmul_fp8(MLK_F32, *[b[1] for b in bufs], y.ptr, 320, 512, rows)

    threads = [threading.Thread(target=go, args=j[:3]) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for rows, _, outs, (want, *parts) in jobs:
        room = U.product_tolerance(want, *parts, 512, False)
        for y in outs:
            assert np.all(np.abs(y.get(F32, (rows, 320)) - want) <= room)


def softmax_top(rng, tokens, experts, top_k):
    score = rng.random((tokens, experts))
    ids = np.argsort(-score, 1, kind="stable")[:, :top_k]
    weight = np.take_along_axis(score, ids, 1)
    return ids, weight / weight.sum(1, keepdims=True)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("tokens", [1, 7, 150])
def test_expert_layer(device, dtype, tokens):
    """The operators as a layer runs them: packed weights, the norm of the residual sum,
    the gathered gate and up products, SwiGLU, the down products, and a dense product
    onto the residual stream.  Every stage is checked on the codes that the one before
    left, the whole against the layer in 64 bits without fp8."""
    hidden, inter, experts, top_k = 256, 160, 6, 2
    rng = np.random.default_rng(tokens)
    size, kind = (2, np.uint16) if dtype == MLK_BF16 else (4, F32)

    def value(raw):
        return (U.from_bf16(raw) if dtype == MLK_BF16 else raw).astype(np.float64)

    def pack(m):
        out, inp = m.shape[-2:]
        raw = m.reshape(-1, out, inp).astype(F32)
        codes, scales = [], []
        for one in raw:
            src, at = put(one)
            q, s = Out(out * inp), Out(4 * U.blocks(out) * U.blocks(inp))
            native.quantize_fp8(MLK_F32, at, out, inp, 128, q.ptr, s.ptr)
            codes.append(q.get(np.uint8, (out, inp)))
            scales.append(s.get(F32, (U.blocks(out), U.blocks(inp))))
        return np.stack(codes), np.stack(scales)

    gate_up = 0.06 * rng.standard_normal((experts, 2 * inter, hidden))
    down = 0.08 * rng.standard_normal((experts, hidden, inter))
    proj = 0.06 * rng.standard_normal((1, hidden, hidden))
    packed = [pack(m) for m in (gate_up, down, proj)]
    dev = [[put(a) for a in p] for p in packed]
    xr, x = typed(dtype, rng.standard_normal((tokens, hidden)))
    rr, r = typed(dtype, rows_of(rng, tokens, hidden, 5.0))
    norm = (1.0 + 0.1 * rng.standard_normal(hidden)).astype(F32)
    ids, weight = softmax_top(rng, tokens, experts, top_k)
    order = np.argsort(ids.reshape(-1), kind="stable")
    counts = np.bincount(ids.reshape(-1), minlength=experts)
    ends = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n = tokens * top_k
    (xb, xat), (rb, rat), (nb, nat), (ob, oat), (ib, iat) = (
        put(a) for a in (xr, rr, norm, ends, (order // top_k).astype(np.int32)))
    hb = U.blocks(hidden)
    total, xq, xs = Out(tokens * hidden * size), Out(tokens * hidden), Out(4 * tokens * hb)
    gu, hq, hs = Out(n * 2 * inter * size), Out(n * inter), Out(4 * n * U.blocks(inter))
    dn, y = Out(n * hidden * size), Out(tokens * hidden * size)
    native.rmsnorm_fp8(dtype, xat, nat, tokens, hidden, xq.ptr, xs.ptr, resid=rat, total=total.ptr)
    native.matmul_fp8_grouped(dtype, dev[0][0][1], dev[0][1][1], xq.ptr, xs.ptr, gu.ptr, 2 * inter,
                              hidden, experts, oat, n, row_ids=iat, x_rows=tokens)
    native.swiglu_fp8(dtype, gu.ptr, n, inter, hq.ptr, hs.ptr)
    native.matmul_fp8_grouped(dtype, dev[1][0][1], dev[1][1][1], hq.ptr, hs.ptr, dn.ptr, hidden,
                              inter, experts, oat, n)
    native.matmul_fp8(dtype, dev[2][0][1], dev[2][1][1], xq.ptr, xs.ptr, y.ptr, hidden, hidden,
                      tokens, resid=total.ptr)
    h = value(total.get(kind, (tokens, hidden)))
    xc, xsc = xq.get(np.uint8, (tokens, hidden)), xs.get(F32, (tokens, hb))
    gate_up_out = value(gu.get(kind, (n, 2 * inter)))
    hc, hsc = hq.get(np.uint8, (n, inter)), hs.get(F32, (n, U.blocks(inter)))
    down_out = value(dn.get(kind, (n, hidden)))
    bf16 = dtype == MLK_BF16
    for e in range(experts):
        at = slice(ends[e], ends[e + 1])
        src = (order // top_k)[at]
        want, *parts = U.product(xc[src], xsc[src], packed[0][0][e], packed[0][1][e])
        assert np.all(np.abs(gate_up_out[at] - want) <=
                      U.product_tolerance(want, *parts, hidden, bf16))
        want, *parts = U.product(hc[at], hsc[at], packed[1][0][e], packed[1][1][e])
        assert np.all(np.abs(down_out[at] - want) <= U.product_tolerance(want, *parts, inter, bf16))
    g, u = gate_up_out[:, :inter], gate_up_out[:, inter:]
    U.check_codes(hc, hsc, g / (1.0 + np.exp(-g)) * u, 9 * U.HALF_F32)
    want, *parts = U.product(xc, xsc, packed[2][0][0], packed[2][1][0])
    got = value(y.get(kind, (tokens, hidden)))
    assert np.all(np.abs(got - want - h) <= U.product_tolerance(want, *parts, hidden, bf16, h))
    # the layer without fp8: a code is off by at most 2^-4 of its value, in the rows and
    # matrices of three products in a row; sums of many such errors of either sign are
    # far below 4 x 2^-4 of the whole
    full = (x + r).astype(np.float64)
    full = U.from_bf16(U.to_bf16(full)).astype(np.float64) if bf16 else full
    v = full / np.sqrt((full * full).mean(1, keepdims=True) + 1e-5) * norm
    layer, got_layer = np.zeros((tokens, hidden)), np.zeros((tokens, hidden))
    for j, entry in enumerate(order):
        t, e = entry // top_k, ids.reshape(-1)[entry]
        gu_full = gate_up[e] @ v[t]
        act = gu_full[:inter] / (1.0 + np.exp(-gu_full[:inter])) * gu_full[inter:]
        layer[t] += weight.reshape(-1)[entry] * (down[e] @ act)
        got_layer[t] += weight.reshape(-1)[entry] * down_out[j]
    assert np.linalg.norm(got_layer - layer) <= 4 * 2.0 ** -4 * np.linalg.norm(layer)
