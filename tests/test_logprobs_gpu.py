"""mlk_token_logprobs against its formulas in 64 bits."""
import numpy as np
import pytest

import fp8_util as U
import latent_util as L
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, DeviceBuffer
from test_fp8_gpu import Out, put

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64


def run(dtype, x, tokens, top, stride=None, lead=0, entropy=True):
    """x [rows, vocab] as f64 values of `dtype`; (logprobs, entropy, ids, top logprobs)."""
    rows, vocab = x.shape
    stride = vocab if stride is None else stride
    wide = np.full((rows, stride), 1e30)
    wide[:, :vocab] = x
    raw, _ = L.typed(dtype, wide)
    xb, at = put(raw, lead)
    tb, tat = put(np.asarray(tokens, np.int32))
    lp, h = Out(4 * rows), Out(4 * rows)
    ids, tops = Out(4 * rows * top), Out(4 * rows * top)
    space = DeviceBuffer(max(native.token_logprobs_workspace(rows, vocab, top), 16))
    native.token_logprobs(dtype, at, rows, vocab, tat, lp.ptr, space, stride=stride,
                          entropy=h.ptr if entropy else None, top=top, top_ids=ids.ptr if top else None,
                          top_logprobs=tops.ptr if top else None)
    if not entropy:
        assert np.all(h.get(np.uint8, 4 * rows) == h.fill)
    return (lp.get(F32, rows), h.get(F32, rows), ids.get(np.int32, (rows, top)), tops.get(F32, (rows, top)))


def exact(x, tokens, top):
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        m = x.max(1, keepdims=True)
        e = np.exp(x - m)
        z = e.sum(1)
        lp = x - m - np.log(z)[:, None]
        h = np.log(z) - np.where(e > 0, e * (x - m), 0.0).sum(1) / z
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return lp[np.arange(len(x)), tokens], h, ids, np.take_along_axis(lp, ids, 1)


def check(dtype, x, tokens, top, **more):
    _, x = L.typed(dtype, x)
    lp, h, ids, tops = run(dtype, x, tokens, top, **more)
    want = exact(x, tokens, top)
    np.testing.assert_array_equal(ids, want[2])
    # exp(d) = 2^(d log2 e): d is rounded (2^-24 of at most 104, past which exp is 0), its
    # product by log2 e (2^-24 of it, in log2 e units of the exponent) and log2 e itself (less
    # than 2^-26 of it), and 2 last places of the power: each term within 104 * 2.25 + 4 =
    # 238 * 2^-24 of itself, with up to 7 f32 additions 252; so is their sum less the largest
    # term, which is exact, and log Z by that times (Z - 1) / Z.  The result is rounded once.
    z = np.exp(x - x.max(1, keepdims=True)).sum(1)
    off = 252 * U.HALF_F32 * (z - 1) / z + 1e-13
    for got, ref in ((lp, want[0]), (tops, want[3])):
        room = U.HALF_F32 * np.abs(np.where(np.isinf(ref), 0, ref)) + (off if ref.ndim == 1 else off[:, None])
        same = np.isinf(ref) & (got == ref)
        with np.errstate(invalid="ignore"):
            assert np.all(same | (np.abs(got - ref) <= room)), np.nanmax(np.abs(got - ref) / room)
    if more.get("entropy", True):
        # T = sum (x - m) exp(x - m): 2 more roundings a term and up to 8 additions in f32
        with np.errstate(invalid="ignore"):
            d = x - x.max(1, keepdims=True)
            mean = np.where(np.exp(d) > 0, -d * np.exp(d), 0.0).sum(1) / z
        room = off * (1 + mean) + 270 * U.HALF_F32 * mean + U.HALF_F32 * want[1]
        assert np.all(np.abs(h - want[1]) <= room)
    return lp, h, ids, tops


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 0), (1, 1, 1), (3, 2, 2), (2, 7, 5), (5, 255, 32), (4, 256, 1), (3, 2047, 20), (2, 2048, 20),
    (2, 2049, 32), (1, 8193, 8), (1, 163840, 20), (2, 163840, 0), (40, 163840, 5), (700, 300, 3),
    (600, 8200, 20), (513, 8192, 32), (9, 50021, 20)])
def test_logprobs(device, dtype, rows, vocab, top):
    rng = np.random.default_rng(rows + vocab)
    x = 2.5 * rng.standard_normal((rows, vocab)) + 6.0 * (rng.random((rows, vocab)) < 0.002)
    check(dtype, x, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
def test_strided_unaligned_rows_without_entropy(device, dtype):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, 4099))
    check(dtype, x, [0, 4098, 7, 1, 2], 9, stride=4103, lead=L.item_size(dtype), entropy=False)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,vocab", [(3, 5000), (600, 3000)])
def test_equal_and_masked_logits(device, dtype, rows, vocab):
    """Ties over a whole row, in rising and falling order, zeros of both signs, rows that a
    mask leaves one or a few tokens of."""
    rng = np.random.default_rng(4)
    for kind in range(7):
        x = rng.standard_normal((rows, vocab))
        if kind == 0:
            x[:] = 1.5
        elif kind == 1:
            x[:] = np.sort(x, 1)
        elif kind == 2:
            x[:] = -np.sort(x, 1)
        elif kind == 3:
            x[:] = np.where(rng.random(x.shape) < 0.5, 0.0, -0.0)
        elif kind == 4:
            x[:] = np.round(x)
        elif kind == 5:
            x[:] = -np.inf
            x[:, vocab - 3] = 2.0
        else:
            keep = rng.random(x.shape) < 0.002
            keep[:, 17] = True
            x[~keep] = -np.inf
        check(dtype, x, rng.integers(0, vocab, rows), 12)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
def test_likely_tokens_keep_their_small_log_probabilities(device, dtype):
    """One token far above the others, by 5 to 60: log p down to -1e-21 or so is told to the
    precision of the sum of the others."""
    rng = np.random.default_rng(5)
    for above in (5, 12, 20, 30, 45):
        for vocab in (900, 70000):
            x = np.round(8 * rng.standard_normal((3, vocab))) / 8
            at = rng.integers(0, vocab, 3)
            x[np.arange(3), at] = x.max(1) + above
            lp, _, _, _ = check(dtype, x, at, 4)
            want = exact(L.typed(dtype, x)[1], at, 4)[0]
            if above <= 30:
                np.testing.assert_allclose(lp, want, rtol=1e-3)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,vocab", [(4, 700), (4, 30000), (600, 9000)])
def test_rows_that_have_no_softmax(device, dtype, rows, vocab):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((rows, vocab))
    x[0, 5] = np.nan
    x[1, vocab - 1] = np.inf
    x[2] = -np.inf
    lp, h, ids, tops = run(dtype, x, [7] * rows, 3)
    assert np.isnan(lp[:3]).all() and np.isnan(h[:3]).all() and np.isnan(tops[:3]).all()
    assert ids[1, 0] == vocab - 1 and list(ids[2]) == [0, 1, 2] and 5 not in ids[0]
    assert np.isfinite(lp[3:]).all() and np.isfinite(tops[3:]).all()
    x = np.full((2, 4), np.nan)
    x[1, 2] = 1.0
    _, _, ids, _ = run(dtype, x, [0, 0], 3)
    assert list(ids[0]) == [-1, -1, -1] and list(ids[1]) == [2, -1, -1]


def test_tokens_out_of_range(device):
    rng = np.random.default_rng(7)
    x = rng.standard_normal((4, 900))
    lp, h, _, _ = run(MLK_F32, x, [-1, 900, 3, 1 << 30], 0, stride=1000)
    assert np.isnan(lp[[0, 1, 3]]).all() and np.isfinite(lp[2]) and np.isfinite(h).all()


def test_rows_past_32_bits(device):
    """Rows more than 2^32 bytes behind the first."""
    rows, vocab, stride = 3, 1000, (1 << 31) + 12
    rng = np.random.default_rng(8)
    _, x = L.typed(MLK_BF16, rng.standard_normal((rows, vocab)))
    raw = U.to_bf16(x.astype(F32))
    data = DeviceBuffer(2 * (stride * (rows - 1) + vocab))
    for r in range(rows):
        data.upload(raw[r].view(np.uint8), 2 * stride * r)
    tb, tat = put(np.array([1, 2, 3], np.int32))
    lp, ids, tops = Out(12), Out(24), Out(24)
    space = DeviceBuffer(max(native.token_logprobs_workspace(rows, vocab, 2), 16))
    native.token_logprobs(MLK_BF16, data, rows, vocab, tat, lp.ptr, space, stride=stride, top=2,
                          top_ids=ids.ptr, top_logprobs=tops.ptr)
    want = exact(x, [1, 2, 3], 2)
    np.testing.assert_allclose(lp.get(F32, 3), want[0], rtol=1e-6)
    np.testing.assert_array_equal(ids.get(np.int32, (3, 2)), want[2])


def test_greedy_sampler_takes_the_first(device):
    """What mlk_sample picks at temperature 0 is the first alternative."""
    rng = np.random.default_rng(9)
    x = np.round(4 * rng.standard_normal((1, 163840))) / 4  # many equal largest
    x[0, rng.integers(0, 163840, 5)] = 30.0
    _, _, ids, _ = check(MLK_F32, x, [0], 5)
    xb, at = put(x.astype(F32))
    assert native.sample(at, 163840, 0.0, 1.0, 0.0) == ids[0, 0]


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("most,vocab", [(40, 50021), (13, 163840), (300, 8200)])
def test_one_workspace_for_batches_that_shrink(device, dtype, most, vocab):
    """The largest batch's workspace serves fewer rows, by whichever pieces these are taken."""
    rng = np.random.default_rng(10)
    top = 20
    space = DeviceBuffer(native.token_logprobs_workspace(most, vocab, top))
    raw, x = L.typed(dtype, rng.standard_normal((most, vocab)))
    tokens = rng.integers(0, vocab, most)
    xb, xat = put(raw)
    tb, tat = put(tokens.astype(np.int32))
    for rows in [r for r in (most, 255, 36, 12, 3, 1) if r <= most]:
        lp, ids, tops = Out(4 * rows), Out(4 * rows * top), Out(4 * rows * top)
        native.token_logprobs(dtype, xat, rows, vocab, tat, lp.ptr, space, top=top, top_ids=ids.ptr,
                              top_logprobs=tops.ptr)
        want = exact(x[:rows], tokens[:rows], top)
        np.testing.assert_array_equal(ids.get(np.int32, (rows, top)), want[2])
        # as in check(): log p is off by half a last place of it and 252 * 2^-24
        for got, ref in ((lp.get(F32, rows), want[0]), (tops.get(F32, (rows, top)), want[3])):
            assert np.all(np.abs(got - ref) <= U.HALF_F32 * (np.abs(ref) + 252) + 1e-13)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 2000000), (1, 2088960), (2, 1000001), (1, 1 << 22), (3, 1 << 21)])
def test_widest_vocabularies_with_most_alternatives(device, dtype, rows, vocab):
    """Up to 1020 small pieces, or 512 large ones, whose likely tokens are put in order together;
    many of them are equal."""
    rng = np.random.default_rng(11)
    x = np.round(8 * 2.5 * rng.standard_normal((rows, vocab))) / 8
    check(dtype, x, rng.integers(0, vocab, rows), 32)
    x[:] = -1.0
    x[:, ::5] = 2.0
    check(dtype, x, rng.integers(0, vocab, rows), 32)
