"""The latent cache entry points against their formulas in 64 bits."""
import threading

import numpy as np
import pytest

import fp8_util as U
import latent_util as L
from conftest import rel_l2
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, MLK_FP4, DeviceBuffer
from test_fp8_gpu import Out, put

pytestmark = pytest.mark.gpu

F32, F64 = np.float32, np.float64
FREQ = (50000.0 ** (-np.arange(0, 64, 2) / 64)).astype(F32)


def freq(rope):
    return (50000.0 ** (-np.arange(0, rope, 2) / rope)).astype(F32)


@pytest.fixture(scope="module")
def workspace(device):
    return DeviceBuffer(native.latent_attend_workspace())


# ---- append ---------------------------------------------------------------------


def run_append(rng, cache, dtype, heads=3, head=None, extra=0, norm=True, query=True, lead=0, kv=None):
    """Appends random rows; checks every byte of the pages and every value of q."""
    latent, rope, rows = cache.latent, cache.rope, cache.rows
    head = rope + 5 if head is None else head
    size = L.item_size(dtype)
    width = latent + rope
    v = rng.standard_normal((rows, width + extra)) * 3 if kv is None else kv
    raw, v = L.typed(dtype, v)
    w = (1 + 0.2 * rng.standard_normal(latent)).astype(F32) if norm else None
    qr, qv = L.typed(dtype, rng.standard_normal((rows, heads * head + extra)))
    f = freq(rope)
    batch = cache.upload()
    kvb, kvat = put(raw, lead)
    wb, wat = put(w if norm else np.zeros(1, F32))
    fb, fat = put(f)
    qb, qat = put(qr, lead)
    out = Out(rows * heads * width * size, lead)
    native.latent_append(batch, dtype, kvat, rows, wat if norm else None, fat, eps=1e-5,
                         stride=width + extra, query=qat if query else None,
                         query_stride=heads * head + extra, heads=heads, head_width=head,
                         q=out.ptr if query else None)
    got = cache.download()
    q = out.get(np.uint8, (rows, heads, width * size))
    untouched = np.full(width * size, out.fill, np.uint8)
    wrote = np.zeros(cache.pool.shape[:2], bool)
    turned = set()
    for r, s, j in cache.each_row():
        if j < 0:
            continue
        page = cache.tables[s, j // cache.page] if j // cache.page < cache.width else -1
        if query:
            turned.add(r)
            want = L.rotate(qv[r, :heads * head].reshape(heads, head)[:, head - rope:], j, f)
            have = L.values(dtype, q[r][:, latent * size:].copy()).reshape(heads, rope)
            half = U.HALF_BF16 if dtype == MLK_BF16 else U.HALF_F32
            assert np.all(np.abs(have - want) <= half * np.abs(want) * (1 + 1e-6) + 1e-30), r
            assert np.all(q[r][:, :latent * size] == out.fill)
        if not 0 <= page < cache.pages:
            continue
        key = np.concatenate([L.normed(v[r, :latent], w, 1e-5), L.rotate(v[r, latent:width], j, f)])
        want = L.encode_row(key, cache.type, latent)
        have = got[page, j % cache.page]
        assert L.same_rows(have, want, cache.type, latent), (r, s, j)
        wrote[page, j % cache.page] = True
    for r in range(rows):
        if r not in turned:
            assert np.all(q[r] == np.broadcast_to(untouched, q[r].shape)), r
    assert np.array_equal(got[~wrote], cache.pool[~wrote])
    return got


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("latent,rope,page,pairs,lead,extra", [
    (512, 64, 16, [(1, 1)], 0, 0),
    (512, 64, 16, [(40, 3), (0, 1), (17, 17), (5, 0), (2, 4)], 0, 7),
    (512, 64, 1, [(3, 2), (1, 1)], 4, 1),
    (64, 16, 7, [(9, 9), (30, 1)], 8, 0),
    (128, 32, 200, [(300, 70)], 4, 3),
    (448, 48, 64, [(65, 2), (64, 1)], 0, 0)])
def test_append(device, dtype, cache_type, latent, rope, page, pairs, lead, extra):
    rng = np.random.default_rng(latent + page + len(pairs))
    cache = L.Cache(rng, cache_type, pairs, latent, rope, page, rows_behind=2)
    run_append(rng, cache, dtype, lead=lead, extra=extra)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
def test_append_many_sequences_one_row_each(device, cache_type):
    rng = np.random.default_rng(4)
    cache = L.Cache(rng, cache_type, [(int(n), 1) for n in rng.integers(0, 40, 150)], starts=False)
    run_append(rng, cache, MLK_F32, heads=1)


@pytest.mark.parametrize("seqs", [64, 65, 128, 300])
def test_rows_of_many_sequences(device, workspace, seqs):
    """Appended, read back and attended to by starts of more sequences than a wave has lanes,
    some of them without rows, the last ones among them."""
    rng = np.random.default_rng(seqs)
    counts = rng.integers(0, 4, seqs)
    counts[-3:] = 0
    pairs = [(int(n) + int(rng.integers(0, 9)), int(n)) for n in counts]
    cache = L.Cache(rng, MLK_FP4, pairs, 64, 16, 4, rows_behind=3)
    run_append(rng, cache, MLK_F32, heads=1)
    cache.fill(rng)
    out = Out(cache.rows * 80 * 4)
    native.latent_gather(cache.upload(), MLK_F32, out.ptr, cache.rows)
    got = out.get(F32, (cache.rows, 80))
    for r, s, j in cache.each_row():
        np.testing.assert_array_equal(got[r], cache.get(s, j))
    assert np.all(got[cache.starts[-1]:].view(np.uint8) == out.fill)
    check_attend(rng, cache, MLK_F32, 2, workspace)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
def test_append_without_norm_or_queries(device, cache_type):
    rng = np.random.default_rng(5)
    cache = L.Cache(rng, cache_type, [(4, 4), (9, 1)], 64, 16)
    run_append(rng, cache, MLK_F32, norm=False, query=False)


def test_append_borders_of_codes(device):
    """Ties, the neighbours of ties, scales at their borders, zeros, values too small and
    too large for a scale, NaN and infinities."""
    rng = np.random.default_rng(6)
    rows = np.zeros((12, 80), F32)
    mid = ((L.MAGNITUDES[:-1] + L.MAGNITUDES[1:]) / 2).astype(F32)
    for r, sign in ((0, 1), (1, -1)):
        rows[r, :7], rows[r, 7:14], rows[r, 14:21] = mid, np.nextafter(mid, F32(0)), np.nextafter(mid, F32(9))
        rows[r, 21:32] = 6.0
        rows[r, 32:64] = rows[r, :32] * F32(2.0 ** -90)
        rows[r] *= sign
    rows[2, :32], rows[2, 32:64] = 6.0, np.nextafter(F32(6), F32(7))
    rows[3, 0], rows[3, 32] = F32(2.0 ** -99), F32(2.0 ** -103)
    rows[4, :64] = -0.0
    rows[5, 3] = np.nan
    rows[6, 40] = -np.inf
    rows[7, 0], rows[7, 32] = F32(2.0 ** 127), np.nextafter(F32(2.0 ** 127), F32(0))
    rows[8, :64] = np.linspace(-3.4e38, 3.4e38, 64)
    rows[9, :64] = F32(1e-45)
    rows[10, :64] = np.linspace(-4, 4, 64) * F32(6 * 2.0 ** -100)
    rows[11, :64] = np.geomspace(1e-6, 1, 64)
    for cache_type in (MLK_FP4, MLK_BF16):
        cache = L.Cache(rng, cache_type, [(12, 12)], 64, 16)
        run_append(rng, cache, MLK_F32, norm=False, query=False, kv=rows)


def test_append_far_positions(device):
    """Angles of positions near 2^31: pages of 512 rows, of which the table names a few."""
    rng = np.random.default_rng(7)
    cache = L.Cache(rng, MLK_BF16, [(5, 3), (600, 2)], 64, 16, 512, spare=3)
    far = np.full((2, 1 << 22), -1, np.int32)
    cache.lengths[:] = [(1 << 31) - 1, (1 << 30) + 1]
    far[0, (1 << 22) - 1] = cache.pages - 1
    far[1, (1 << 21) - 1:(1 << 21) + 1] = [0, 1]
    cache.tables, cache.width = far, far.shape[1]
    run_append(rng, cache, MLK_F32)


def test_append_pages_out_of_range(device):
    """A page that is none of the cache's, and a position behind the table."""
    rng = np.random.default_rng(8)
    cache = L.Cache(rng, MLK_FP4, [(40, 30), (50, 5)], 64, 16, 16)
    cache.tables[0, 1], cache.tables[0, 2] = cache.pages, -7
    cache.lengths[1] = cache.width * 16 + 2
    run_append(rng, cache, MLK_BF16)


def test_rows_of_malformed_starts(device, workspace):
    """Starts that decrease or leave the rows give their sequences no rows; nothing is
    written for them."""
    rng = np.random.default_rng(9)
    for starts in ([0, 3, 2, 4], [0, 2, 9, 12], [-4, -1, 1, 4], [5, 5, 5, 5], [0, -1, 2, 1 << 30]):
        cache = L.Cache(rng, MLK_BF16, [(8, 1), (8, 1), (8, 2)], 64, 16).fill(rng)
        cache.starts = np.array(starts, np.int32)
        batch = cache.upload()
        buf, at = put(np.zeros((4, 2, 80), F32))
        fb, fat = put(freq(16))
        q = Out(4 * 2 * 80 * 4)
        native.latent_append(batch, MLK_F32, at, 4, None, fat, query=at, heads=1, head_width=80, q=q.ptr,
                             query_stride=80)
        out = Out(4 * 2 * 64 * 4)
        native.latent_attend(batch, MLK_F32, at, out.ptr, 4, 2, 0.1, workspace)
        back = Out(4 * 80 * 4)
        native.latent_gather(batch, MLK_F32, back.ptr, 4)
        good = {r for a, b in zip(starts, starts[1:]) if 0 <= a < b <= 4 for r in range(a, b)}
        raw = out.get(np.uint8, (4, 512)), back.get(np.uint8, (4, 320)), q.get(np.uint8, (4, 640))
        for r in set(range(4)) - good:
            assert np.all(raw[0][r] == out.fill), (starts, r)
        if starts[0] >= 4:
            assert all(np.all(x == out.fill) for x in raw)
            assert np.array_equal(cache.download(), cache.pool)


# ---- gather ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("latent,rope,page,pairs,lead", [
    (512, 64, 16, [(37, 37), (0, 0), (1, 1), (20, 4), (3, 5)], 0),
    (512, 64, 5, [(70, 70)], 4),
    (64, 16, 1, [(3, 3), (2, 2)], 8),
    (192, 48, 33, [(40, 40)], 0)])
def test_gather(device, dtype, cache_type, latent, rope, page, pairs, lead):
    rng = np.random.default_rng(latent + page)
    cache = L.Cache(rng, cache_type, pairs, latent, rope, page, rows_behind=1).fill(rng)
    size = L.item_size(dtype)
    out = Out(cache.rows * (latent + rope) * size, lead)
    native.latent_gather(cache.upload(), dtype, out.ptr, cache.rows)
    got = out.get(np.uint8, (cache.rows, (latent + rope) * size))
    for r, s, j in cache.each_row():
        want = cache.get(s, j) if j >= 0 else np.zeros(latent + rope)
        np.testing.assert_array_equal(L.values(dtype, got[r].copy()), want)
    assert np.all(got[cache.starts[-1]:] == out.fill)


def test_gather_pages_out_of_range(device):
    rng = np.random.default_rng(11)
    cache = L.Cache(rng, MLK_FP4, [(40, 40)], 64, 16, 16).fill(rng)
    cache.tables[0, 1] = cache.pages
    out = Out(40 * 80 * 4)
    native.latent_gather(cache.upload(), MLK_F32, out.ptr, 40)
    got = out.get(F32, (40, 80))
    assert np.isnan(got[16:32]).all()
    cache.tables[0, 1] = 0
    for j in list(range(16)) + list(range(32, 40)):
        np.testing.assert_array_equal(got[j], cache.get(0, j))


# ---- attend ---------------------------------------------------------------------


def run_attend(rng, cache, dtype, heads, workspace, scale=None, sharp=1.0, lead=0, q=None):
    latent, width = cache.latent, cache.latent + cache.rope
    scale = 192 ** -0.5 if scale is None else scale
    if q is None:
        q = rng.standard_normal((cache.rows, heads, width)) * np.where(rng.random((heads, 1)) < 0.3, 3, 0.7)
        q = q * sharp
    raw, v = L.typed(dtype, q)
    size = L.item_size(dtype)
    qb, qat = put(raw, lead)
    out = Out(cache.rows * heads * latent * size, lead)
    native.latent_attend(cache.upload(), dtype, qat, out.ptr, cache.rows, heads, scale, workspace)
    got = out.get(np.uint8, (cache.rows, heads * latent * size))
    assert np.all(got[cache.starts[-1]:] == out.fill)
    got = L.values(dtype, got.copy()).reshape(cache.rows, heads, latent)[:cache.starts[-1]]
    return got, v, F64(F32(scale))


def check_attend(rng, cache, dtype, heads, workspace, **more):
    got, q, scale = run_attend(rng, cache, dtype, heads, workspace, **more)
    want, mass, score = L.attend(cache, q, heads, scale)
    want, mass, score = (x[:cache.starts[-1]] for x in (want, mass, score))
    room = L.attend_tolerance(cache, want, mass, score, dtype)
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    assert np.all(off <= room), (off / np.maximum(room, 1e-300)).max()
    # the errors of a result's many terms are of either sign: far below their sum
    if np.linalg.norm(want) > 0:
        assert rel_l2(got, want) < (2.0 ** -8 if dtype == MLK_BF16 else 1e-5)
    return got


CASES = [
    # latent, rope, page, heads, pairs
    (512, 64, 16, 16, [(1, 1)]),
    (512, 64, 16, 16, [(15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1)]),
    (512, 64, 64, 16, [(700, 1)]),
    (512, 64, 128, 16, [(0, 1), (300, 1), (0, 1), (5, 1)]),
    (512, 64, 7, 1, [(33, 1), (100, 1)]),
    (512, 64, 1, 5, [(129, 7)]),
    (512, 64, 16, 3, [(50, 50), (4, 6), (0, 3), (130, 9)]),
    (512, 64, 100, 40, [(90, 2), (1, 1)]),
    (512, 64, 16, 128, [(70, 1), (20, 2)]),
    (64, 16, 16, 4, [(200, 3), (1, 1)]),
    (128, 32, 33, 17, [(77, 2)]),
    (256, 64, 16, 16, [(140, 1), (3, 3)]),
    (448, 48, 64, 8, [(65, 5)]),
]


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("latent,rope,page,heads,pairs", CASES)
def test_attend(device, workspace, dtype, cache_type, latent, rope, page, heads, pairs):
    rng = np.random.default_rng(latent + page + heads)
    cache = L.Cache(rng, cache_type, pairs, latent, rope, page, rows_behind=1).fill(rng)
    check_attend(rng, cache, dtype, heads, workspace)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("page,heads,pairs,lead", [
    (16, 16, [(64, 64), (130, 66)], 0),
    (16, 128, [(4, 4), (9, 9), (700, 5)], 16),
    (64, 16, [(127, 45), (128, 40), (129, 38), (0, 0), (1, 1), (63, 20)], 0),
    (100, 5, [(300, 293), (140, 140)], 0),
    (1, 128, [(65, 1), (600, 16)], 0),
    (7, 40, [(2, 3), (90, 52), (0, 4)], 0),
    (128, 16, [(1500, 90), (700, 38), (30, 30), (1100, 1)], 0),
    (16, 1, [(650, 650), (1600, 1450)], 0),
    (16, 128, [(4000, 16)], 0),
    (16, 16, [(140, 130)], 2)])
def test_attend_many_pairs_a_sequence(device, workspace, cache_type, page, heads, pairs, lead):
    """Prompts in chunks, many heads; beside single rows and empty sequences."""
    rng = np.random.default_rng(page + heads + len(pairs))
    cache = L.Cache(rng, cache_type, pairs, page_size=page, rows_behind=1, table_extra=512 // page + 1).fill(rng)
    check_attend(rng, cache, MLK_BF16, heads, workspace, lead=lead)


@pytest.mark.parametrize("dtype,cache_type,latent,rope,heads,pairs", [
    (MLK_F32, MLK_FP4, 64, 16, 128, [(300, 290), (20, 10)]),
    (MLK_BF16, MLK_BF16, 64, 16, 128, [(300, 290), (20, 10)]),
    (MLK_BF16, MLK_BF16, 512, 64, 128, [(70, 600), (90, 500)])])
def test_attend_more_tiles_than_records(device, workspace, dtype, cache_type, latent, rope, heads, pairs):
    rng = np.random.default_rng(28)
    cache = L.Cache(rng, cache_type, pairs, latent, rope, table_extra=40).fill(rng)
    q = rng.standard_normal((cache.rows, heads, latent + rope), dtype=F32)
    check_attend(rng, cache, dtype, heads, workspace, q=q)


@pytest.mark.parametrize("dtype,cache_type,latent,rope,rows", [
    (MLK_F32, MLK_FP4, 64, 16, 4), (MLK_BF16, MLK_BF16, 512, 64, 40)])
def test_attend_tables_of_2_to_the_31_keys(device, workspace, dtype, cache_type, latent, rope, rows):
    """Steps of all keys that such tables hold are more than 32 bits count."""
    rng = np.random.default_rng(29)
    cache = L.Cache(rng, cache_type, [(100, rows), (70, 1)], latent, rope, 1 << 15, spare=0,
                    table_extra=(1 << 16) - 1).fill(rng)
    check_attend(rng, cache, dtype, 128, workspace)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
def test_attend_sequences_that_share_pages(device, workspace, cache_type):
    """A prefix that three sequences have in common, and a page twice in a table."""
    rng = np.random.default_rng(33)
    for heads, rows in ((16, 1), (16, 70)):
        cache = L.Cache(rng, cache_type, [(96, rows)] * 3, table_extra=32).fill(rng)
        cache.tables[1, :3] = cache.tables[2, :3] = cache.tables[0, :3]
        cache.tables[1, 4] = cache.tables[1, 3]
        check_attend(rng, cache, MLK_BF16, heads, workspace)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
def test_attend_joined_over_workgroups(device, workspace, dtype, cache_type):
    """Sequences whose keys fall to many workgroups, beside short ones and empty slots."""
    rng = np.random.default_rng(20)
    pairs = [(2500, 1), (1, 1), (0, 1), (1300, 2), (64, 1), (65, 1)]
    cache = L.Cache(rng, cache_type, pairs, page_size=48).fill(rng)
    check_attend(rng, cache, dtype, 16, workspace)


def test_attend_many_short_sequences(device, workspace):
    """More sequences than a workgroup has threads, one row each, without row_starts."""
    rng = np.random.default_rng(21)
    pairs = [(int(n), 1) for n in rng.integers(0, 9, 700)]
    cache = L.Cache(rng, MLK_BF16, pairs, 64, 16, 4, starts=False).fill(rng)
    check_attend(rng, cache, MLK_F32, 2, workspace)


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
def test_attend_sharp_and_flat_scores(device, workspace, dtype):
    """Scores in the hundreds, whose maximum moves late; all scores equal; a negative scale."""
    rng = np.random.default_rng(22)
    cache = L.Cache(rng, MLK_BF16, [(400, 1)], table_extra=32).fill(rng)
    for j in range(400):  # ever larger rows
        cache.put(0, j, cache.get(0, j) * (0.2 + j / 200))
    check_attend(rng, cache, dtype, 16, workspace, scale=0.5)
    check_attend(rng, cache, dtype, 16, workspace, scale=-0.3)
    check_attend(rng, cache, dtype, 16, workspace, scale=0.0)
    cache.starts = np.array([0, 70], np.int32)
    cache.rows = 70
    for scale in (0.5, -0.3, 0.0):
        check_attend(rng, cache, dtype, 16, workspace, scale=scale)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
def test_attend_unaligned_rows(device, workspace, dtype, cache_type):
    rng = np.random.default_rng(23)
    cache = L.Cache(rng, cache_type, [(90, 3)]).fill(rng)
    check_attend(rng, cache, dtype, 16, workspace, lead=L.item_size(dtype))


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("heads", [3, 160])
def test_attend_values_that_are_not_finite(device, workspace, dtype, cache_type, bad, heads):
    """A key with such a value reaches the rows that see it, and those alone, in the
    latent row or in the rope row; so does a query."""
    rng = np.random.default_rng(24)
    for column in (100, 540):
        for at in (0, 20, 93, 99):
            cache = L.Cache(rng, cache_type, [(100, 12), (40, 1)], table_extra=32).fill(rng)
            clean = cache.get(0, at)
            v = clean.copy()
            v[column] = bad
            cache.put(0, at, v)
            got, q, scale = run_attend(rng, cache, dtype, heads, workspace)
            sees = np.array([s == 0 and j >= at for _, s, j in cache.each_row()])
            assert np.isfinite(got[~sees]).all(), (column, at)
            cache.put(0, at, clean)
            want, mass, score = L.attend(cache, q, heads, scale)
            room = L.attend_tolerance(cache, want, mass, score, dtype)
            assert np.all(np.abs(got - want)[~sees] <= room[~sees]), (column, at)
            told = ~np.isfinite(got[sees]).all((1, 2))
            # (an infinity in the rope row may make a score of -inf: the key has no weight)
            assert told.all() or (column == 540 and np.isinf(bad))
    cache = L.Cache(rng, cache_type, [(100, 12), (40, 1)], table_extra=32).fill(rng)
    q = rng.standard_normal((13, heads, 576))
    q[4, 1, 7] = bad
    got, _, _ = run_attend(rng, cache, dtype, heads, workspace, q=q)
    fine = np.ones((13, heads), bool)
    fine[4, 1] = False
    assert np.isfinite(got[fine]).all() and np.isnan(got[4, 1]).all()


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("heads", [3, 160])
def test_attend_pages_out_of_range(device, workspace, dtype, cache_type, heads):
    """Rows that read a key without a page are NaN, the others as they were; so with keys
    behind the table."""
    rng = np.random.default_rng(25)
    cache = L.Cache(rng, cache_type, [(100, 30), (200, 1), (50, 2)], page_size=16, table_extra=32).fill(rng)
    good = cache.tables.copy()
    cache.tables[0, 5] = cache.pages       # keys 80 .. 95
    cache.tables[1, 3] = -1
    got, q, scale = run_attend(rng, cache, dtype, heads, workspace)
    cache.tables = good
    want, mass, score = L.attend(cache, q, heads, scale)
    room = L.attend_tolerance(cache, want, mass, score, dtype)
    sees = np.array([s == 1 or (s == 0 and j >= 80) for _, s, j in cache.each_row()])
    assert np.isnan(got[sees]).all()
    assert np.all(np.abs(got - want)[~sees] <= room[~sees])
    # a table that ends after 512 keys: the last row, key 512, sees one more
    cache = L.Cache(rng, cache_type, [(512, 13)], page_size=16, table_extra=0).fill(rng)
    cache.lengths[0] = 513
    got, q, scale = run_attend(rng, cache, dtype, heads, workspace)
    cache.lengths[0] = 512
    cache.starts = np.array([0, 12], np.int32)
    want, mass, score = L.attend(cache, q, heads, scale)
    room = L.attend_tolerance(cache, want, mass, score, dtype)
    assert np.all(np.abs(got - want)[:12] <= room[:12]) and np.isnan(got[12]).all()


@pytest.mark.parametrize("dtype,pairs", [(MLK_F32, [(900, 1), (3, 1), (400, 2)]),
                                         (MLK_BF16, [(900, 100), (3, 1), (400, 60)])])
def test_attend_repeats_itself(device, workspace, dtype, pairs):
    """The same call gives the same bits, whatever the workspace holds."""
    rng = np.random.default_rng(26)
    cache = L.Cache(rng, MLK_FP4, pairs).fill(rng)
    q = rng.standard_normal((cache.rows, 16, 576))
    first, _, _ = run_attend(rng, cache, dtype, 16, workspace, q=q)
    for fill in (0xFF, 0x00, 0x7F):
        workspace.upload(np.full(workspace.nbytes, fill, np.uint8))
        again, _, _ = run_attend(rng, cache, dtype, 16, workspace, q=q)
        assert np.array_equal(first, again)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
def test_past_32_bits(device, workspace, cache_type):
    """Pages more than 2^32 bytes into the cache: written, read back and attended to."""
    rng = np.random.default_rng(27)
    row = native.latent_row_bytes(cache_type, 512, 64)
    page, pages = 1024, (1 << 32) // (1024 * row) + 40
    data = DeviceBuffer(pages * page * row)
    tables = np.array([[pages - 1, 3, pages - 20]], np.int32)
    tb, lb = DeviceBuffer.from_array(tables), DeviceBuffer.from_array(np.array([2600], np.int32))
    sb = DeviceBuffer.from_array(np.array([0, 2600], np.int32))
    every = native.LatentBatch(cache_type, data, 512, 64, pages, page, 1, tb, 3, lb, sb)
    v = rng.standard_normal((2600, 576)).astype(F32)
    fb, ft = put(FREQ)
    kb, kt = put(v)
    native.latent_append(every, MLK_F32, kt, 2600, None, ft)
    back = Out(2600 * 576 * 4)
    native.latent_gather(every, MLK_F32, back.ptr, 2600)
    got = back.get(F32, (2600, 576)).astype(F64)
    cache = L.Cache(rng, cache_type, [(2600, 1)], page_size=1024)
    for j in range(2600):
        cache.put(0, j, np.concatenate([v[j, :512].astype(F64), L.rotate(v[j, 512:].astype(F64), j, FREQ)]))
        np.testing.assert_array_equal(got[j], cache.get(0, j))
    one = native.LatentBatch(cache_type, data, 512, 64, pages, page, 1, tb, 3, lb)
    raw, q = L.typed(MLK_F32, rng.standard_normal((1, 16, 576)))
    qb, qt = put(raw)
    out = Out(16 * 512 * 4)
    native.latent_attend(one, MLK_F32, qt, out.ptr, 1, 16, 0.07, workspace)
    want, mass, score = L.attend(cache, q, 16, F64(F32(0.07)))
    assert np.all(np.abs(out.get(F32, (1, 16, 512)) - want) <= L.attend_tolerance(cache, want, mass, score, MLK_F32))


# ---- together -------------------------------------------------------------------


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
def test_steps_of_a_batch(device, workspace, dtype, cache_type):
    """A prompt chunk and four decoding steps of three requests, one of which joins late and
    one of which leaves: append, attend and read back, against the same with dense rows."""
    rng = np.random.default_rng(30)
    heads, nope, latent, rope, page = 4, 24, 128, 32, 8
    width, head = latent + rope, nope + rope
    f, w = freq(rope), (1 + 0.1 * rng.standard_normal(latent)).astype(F32)
    fb, ft = put(f)
    wb, wt = put(w)
    row = native.latent_row_bytes(cache_type, latent, rope)
    pages = 24
    data = DeviceBuffer.from_array(np.full(pages * page * row, 0xFF, np.uint8))
    free = list(rng.permutation(pages))
    tables = np.full((3, 8), -1, np.int32)
    lengths = np.zeros(3, np.int32)
    dense = [[], [], []]
    tb, lb, sb = DeviceBuffer(3 * 8 * 4), DeviceBuffer(12), DeviceBuffer(16)
    batch = native.LatentBatch(cache_type, data, latent, rope, pages, page, 3, tb, 8, lb, sb)
    size = L.item_size(dtype)
    for step, counts in enumerate([(11, 3, 0), (1, 1, 9), (1, 1, 1), (2, 0, 1), (1, 0, 1)]):
        if step == 3:  # request 1 is done: its slot is empty
            lengths[1] = 0
        for s, n in enumerate(counts):
            lengths[s] += n
            while n and np.sum(tables[s] >= 0) * page < lengths[s]:
                tables[s, np.sum(tables[s] >= 0)] = free.pop()
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        rows = int(starts[-1])
        tb.upload(tables), lb.upload(lengths), sb.upload(starts)
        raw, both = L.typed(dtype, rng.standard_normal((rows, heads * head + width)))
        absorbed_raw, absorbed = L.typed(dtype, rng.standard_normal((rows, heads, width)))
        bb, bt = put(raw)
        qb, qt = put(absorbed_raw)
        native.latent_append(batch, dtype, bt + heads * head * size, rows, wt, ft,
                             stride=raw.shape[1], query=bt, query_stride=raw.shape[1], heads=heads,
                             head_width=head, q=qt)
        out, back = Out(rows * heads * latent * size), Out(rows * width * size)
        native.latent_attend(batch, dtype, qt, out.ptr, rows, heads, 0.1, workspace)
        native.latent_gather(batch, dtype, back.ptr, rows)
        got = L.values(dtype, out.get(np.uint8, (rows, heads * latent * size))).reshape(rows, heads, latent)
        kept = L.values(dtype, back.get(np.uint8, (rows, width * size))).reshape(rows, width)
        for s, n in enumerate(counts):
            for i in range(n):
                r = starts[s] + i
                j = len(dense[s])
                kv = both[r, heads * head:]
                key = np.concatenate([L.normed(kv[:latent], w, 1e-5), L.rotate(kv[latent:], j, f)])
                key = L.decode_row(L.encode_row(key, cache_type, latent), cache_type, latent)
                np.testing.assert_array_equal(kept[r], key)
                dense[s].append(key)
                q = absorbed[r].copy()
                turned = L.rotate(both[r, :heads * head].reshape(heads, head)[:, nope:], j, f)
                q[:, latent:] = L.typed(dtype, turned)[1]
                k = np.stack(dense[s])
                x = q @ k.T * F64(F32(0.1))
                p = np.exp(x - x.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                # as in attend_tolerance, for at most 20 keys and scores below 20
                bound = (2.0 ** -6 if dtype == MLK_BF16 else 2e-3) * (p @ np.abs(k[:, :latent]))
                assert np.all(np.abs(got[r] - p @ k[:, :latent]) <= bound), (step, s, i)
        if step == 3:
            assert lengths[1] == 0


def test_calls_from_two_threads(device):
    """Each with a workspace of its own."""
    rng = np.random.default_rng(31)
    caches = [L.Cache(rng, MLK_BF16, [(600, 1), (90, 1)]).fill(rng) for _ in range(2)]
    failed = []

    def work(k):
        try:
            mine = np.random.default_rng(40 + k)
            space = DeviceBuffer(native.latent_attend_workspace())
            for _ in range(6):
                check_attend(mine, caches[k], MLK_F32, 16, space)
        except BaseException as e:  # noqa: BLE001 (told by the main thread)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def with_bad_key(cache, s, at, column, bad):
    v = cache.get(s, at)
    v[column] = bad
    cache.put(s, at, v)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("heads,rows", [(3, 2), (16, 70)])
def test_attend_keys_that_are_not_finite_are_told_by_every_head(device, workspace, dtype, cache_type, bad, heads, rows):
    """Whatever the sign of a head's score: all of its results are NaN where a row sees the key, in
    the latent row or the rope row, at a sequence's beginning, middle and end; the others are right."""
    rng = np.random.default_rng(34)
    pairs = [(700, rows), (1, 1), (0, 1), (90, rows)]
    cache = L.Cache(rng, cache_type, pairs, table_extra=32).fill(rng)
    q = rng.standard_normal((cache.rows, heads, 576))
    _, v = L.typed(dtype, q)
    scale = F64(F32(192 ** -0.5))
    want, mass, score = L.attend(cache, v, heads, scale)
    room = L.attend_tolerance(cache, want, mass, score, dtype)
    for column in (100, 512, 540, 575):
        for s, at in ((0, 0), (0, 330), (0, 698), (0, 699), (1, 0), (3, 89)):
            clean = cache.pool[cache.place(s, at)].copy()
            with_bad_key(cache, s, at, column, bad)
            got, _, _ = run_attend(rng, cache, dtype, heads, workspace, q=q)
            cache.pool[cache.place(s, at)] = clean
            sees = np.array([t == s and j >= at for _, t, j in cache.each_row()])
            assert np.isnan(got[sees]).all(), (column, s, at)
            assert np.all(np.abs(got - want)[~sees] <= room[~sees]), (column, s, at)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows", [1, 70])
def test_attend_queries_that_are_not_finite(device, workspace, dtype, cache_type, bad, rows):
    """Such a query's results are NaN, over one key as over many; a row that sees none is zero."""
    rng = np.random.default_rng(35)
    cache = L.Cache(rng, cache_type, [(700, rows), (1, 1), (0, 1)], table_extra=32).fill(rng)
    for column in (7, 520):
        q = rng.standard_normal((cache.rows, 16, 576))
        fine = np.ones((cache.rows, 16), bool)
        for r, h in ((0, 1), (rows - 1, 15), (rows, 0), (rows, 9), (rows + 1, 4)):
            q[r, h, column] = bad
            fine[r, h] = r == rows + 1
        got, _, _ = run_attend(rng, cache, dtype, 16, workspace, q=q)
        assert np.isfinite(got[fine]).all() and np.isnan(got[~fine]).all()
        assert np.all(got[rows + 1] == 0)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("power", [20, 27, 34, 50, 90])
def test_attend_scores_far_above_a_last_place(device, workspace, dtype, cache_type, rows, power):
    """Scores of 2^power and more, whose last place is many times the slack of a softmax: the
    largest one's key is the result, wherever it lies."""
    rng = np.random.default_rng(36)
    cache = L.Cache(rng, cache_type, [(300, rows), (1, 1)], table_extra=32).fill(rng)
    keys = [cache.keys(0, 300), cache.keys(1, 1)]
    for sign in (1, -1):
        q = rng.standard_normal((cache.rows, 16, 576))
        got, v, scale = run_attend(rng, cache, dtype, 16, workspace, q=q, scale=sign * 2.0 ** power)
        for r, s, j in cache.each_row():
            k = keys[s][:j + 1]
            x = v[r] @ k.T * scale
            order = np.sort(x, 1)
            # a score is off by 2 * 1728 additions' half last places of the magnitudes added
            off = 2 * 1728 * U.HALF_F32 * (np.abs(v[r]) @ np.abs(k).T).max(1) * abs(scale)
            clear = order[:, -1] - order[:, -2] > 2 * off + 200 if j else np.ones(16, bool)
            want = k[x.argmax(1), :512]
            # p v / p: three f32 roundings, then the result's
            half = U.HALF_BF16 if dtype == MLK_BF16 else U.HALF_F32
            assert np.all(np.abs(got[r] - want)[clear] <= (np.abs(want) * (half + 4 * U.HALF_F32))[clear]), (r, s)
            assert np.all(np.abs(got[r]) <= np.abs(k[:, :512]).max(0) * (1 + 2 * half + 8 * U.HALF_F32))
            assert clear.any()


@pytest.mark.parametrize("dtype,length", [(MLK_F32, 1 << 20), (MLK_BF16, 1 << 24)])
def test_attend_leaves_rows_that_sequences_share(device, workspace, dtype, length):
    """Starts that go back and forth give the same rows to a hundred long sequences, more work than
    is counted in 32 bits: nothing is done, and nothing that an earlier call left in the workspace
    becomes a result."""
    rows, heads, seqs, page = 1024, 16, 200, 1 << 14
    size = L.item_size(dtype)
    row = native.latent_row_bytes(MLK_BF16, 512, 64)
    data = DeviceBuffer.from_array(np.zeros(page * row, np.uint8))
    tables = DeviceBuffer.from_array(np.zeros((seqs, length // page), np.int32))
    rng = np.random.default_rng(37)
    qb, qat = put(L.typed(dtype, rng.standard_normal((rows, heads, 576)))[0])
    lengths, starts = DeviceBuffer(4 * seqs), DeviceBuffer(4 * (seqs + 1))
    batch = native.LatentBatch(MLK_BF16, data, 512, 64, 1, page, seqs, tables, length // page, lengths, starts)
    for far, begins in ((3000, [0] + [rows - 24] * seqs), (length, [0, rows] * (seqs // 2) + [0])):
        lengths.upload(np.full(seqs, far, np.int32))
        starts.upload(np.array(begins, np.int32))
        out = Out(rows * heads * 512 * size)
        native.latent_attend(batch, dtype, qat, out.ptr, rows, heads, 0.1, workspace)
        got = out.get(np.uint8, (rows, heads * 512 * size))
        done = rows - 24 if far == 3000 else 0
        assert np.all(got[:done] == 0) and np.all(got[done:] == out.fill)


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
def test_many_pairs_past_32_bits(device, workspace, cache_type):
    """A prompt's chunk over pages more than 2^32 bytes into the cache."""
    rng = np.random.default_rng(38)
    rows, heads, length, page = 140, 16, 2600, 1024
    row = native.latent_row_bytes(cache_type, 512, 64)
    pages = (1 << 32) // (page * row) + 40
    cache = L.Cache(rng, cache_type, [(length, rows)], page_size=page, table_extra=0).fill(rng)
    data = DeviceBuffer(pages * page * row)
    places = np.array([[pages - 1, 3, pages - 20]], np.int32)
    for at, held in zip(places[0], cache.tables[0]):
        data.upload(cache.pool[held].reshape(-1), int(at) * page * row)
    tables = DeviceBuffer.from_array(places)
    lengths, starts = DeviceBuffer.from_array(cache.lengths), DeviceBuffer.from_array(cache.starts)
    batch = native.LatentBatch(cache_type, data, 512, 64, pages, page, 1, tables, 3, lengths, starts)
    raw, q = L.typed(MLK_BF16, rng.standard_normal((rows, heads, 576)))
    qb, qat = put(raw)
    out = Out(rows * heads * 512 * 2)
    native.latent_attend(batch, MLK_BF16, qat, out.ptr, rows, heads, 0.07, workspace)
    got = L.values(MLK_BF16, out.get(np.uint8, rows * heads * 512 * 2)).reshape(rows, heads, 512)
    want, mass, score = L.attend(cache, q, heads, F64(F32(0.07)))
    assert np.all(np.abs(got - want) <= L.attend_tolerance(cache, want, mass, score, MLK_BF16))


@pytest.mark.parametrize("cache_type", [MLK_BF16, MLK_FP4])
@pytest.mark.parametrize("starts", [True, False])
def test_many_pairs_of_more_sequences_than_threads(device, workspace, cache_type, starts):
    """Many heads of a few rows each, some sequences without rows or keys."""
    rng = np.random.default_rng(39)
    counts = rng.integers(0, 4, 300) if starts else np.ones(300, int)
    pairs = [(int(rng.integers(0, 40)), int(n)) for n in counts]
    pairs[7] = (1500, pairs[7][1])
    cache = L.Cache(rng, cache_type, pairs, starts=starts, table_extra=8).fill(rng)
    check_attend(rng, cache, MLK_BF16, 128, workspace)
