"""Paged latent caches in numpy: rows of bf16 or of e2m1 codes, and the formulas of the
latent entry points in 64 bits."""
import numpy as np

import fp8_util as U
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, MLK_FP4, DeviceBuffer

F32, F64 = np.float32, np.float64
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
GROUP, LEAST = 32, -100
GUARD = 256


def bf16_round(v):
    """f64 -> f32 -> bf16 bits, ties to even."""
    with np.errstate(over="ignore"):
        return U.to_bf16(np.where(np.isnan(v), np.nan, v).astype(F32))


def fp4_nearest(a):
    """Index of the magnitude nearest to a (0 .. 6), ties to the even one."""
    mid = (MAGNITUDES[:-1] + MAGNITUDES[1:]) / 2
    lo = np.searchsorted(mid, a, side="left")
    tie = (lo < 7) & (a == mid[np.minimum(lo, 6)])
    return np.where(tie & (lo % 2 == 1), lo + 1, lo)


def scale_place(b):
    return 4 * (b % 4) + b // 4


def encode_row(v, cache_type, latent):
    """Bytes of a cached row of values [latent + rope]."""
    if cache_type == MLK_BF16:
        return bf16_round(v).view(np.uint8)
    codes = np.zeros(latent, np.uint8)
    scales = np.zeros(16, np.uint8)
    for b in range(latent // GROUP):
        x = v[b * GROUP:(b + 1) * GROUP]
        amax = np.max(np.abs(x))
        if not amax < 2.0 ** 127:
            scales[scale_place(b)] = 255
            continue
        share, power = np.frexp(amax)  # amax = share * 2^power, share in [0.5, 1)
        e = max(LEAST, int(power) - (3 if share <= 0.75 else 2)) if amax > 0 else LEAST
        assert amax <= 6.0 * 2.0 ** e and (e == LEAST or amax > 3.0 * 2.0 ** e)
        scales[scale_place(b)] = e + 127
        codes[b * GROUP:(b + 1) * GROUP] = fp4_nearest(np.abs(x) / 2.0 ** e) + 8 * (x < 0)
    return np.concatenate([codes[0::2] | codes[1::2] << 4, scales, bf16_round(v[latent:]).view(np.uint8)])


def decode_row(raw, cache_type, latent):
    """f64 values of a cached row's bytes."""
    if cache_type == MLK_BF16:
        return U.from_bf16(raw.view(np.uint16)).astype(F64)
    byte = raw[:latent // 2]
    codes = np.stack([byte & 15, byte >> 4], -1).reshape(-1)
    v = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    for b in range(latent // GROUP):
        s = int(raw[latent // 2 + scale_place(b)])
        v[b * GROUP:(b + 1) * GROUP] *= np.nan if s == 255 else 2.0 ** (s - 127)
    rope = U.from_bf16(raw[latent // 2 + 16:].copy().view(np.uint16)).astype(F64)
    return np.concatenate([v, rope])


def same_rows(a, b, cache_type, latent):
    """Whether two rows' bytes stand for the same values (codes of a NaN block and the scale
    bytes that no block has aside)."""
    return np.array_equal(decode_row(a, cache_type, latent), decode_row(b, cache_type, latent), equal_nan=True)


class Cache:
    """Pages on the host, every byte of them 0xFF (NaN of either type) but for the rows that
    are put, and the tables of sequences of `pairs` (length, rows), in a random order."""

    def __init__(self, rng, cache_type, pairs, latent=512, rope=64, page_size=16, spare=2, starts=True,
                 rows_behind=0, table_extra=1):
        self.type, self.latent, self.rope, self.page = cache_type, latent, rope, page_size
        self.row = native.latent_row_bytes(cache_type, latent, rope)
        self.lengths = np.array([p[0] for p in pairs], np.int32)
        counts = [p[1] for p in pairs]
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + rows_behind
        need = [-(-max(n, 0) // page_size) for n in self.lengths]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.width = max(need + [0]) + table_extra
        self.tables = np.full((len(pairs), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = order[at:at + n]
            at += n
        self.pool = np.full((self.pages, page_size, self.row), 0xFF, np.uint8)
        self.use_starts = starts

    def place(self, s, j):
        return self.tables[s, j // self.page], j % self.page

    def put(self, s, j, v):
        self.pool[self.place(s, j)] = encode_row(v, self.type, self.latent)

    def get(self, s, j):
        return decode_row(self.pool[self.place(s, j)], self.type, self.latent)

    def fill(self, rng, loud=4.0):
        """Every key of every sequence."""
        columns = np.where(rng.random(self.latent + self.rope) < 0.03, loud, 1.0)
        for s, n in enumerate(self.lengths):
            for j in range(n):
                self.put(s, j, rng.standard_normal(self.latent + self.rope) * columns)
        return self

    def keys(self, s, n):
        return np.stack([self.get(s, j) for j in range(n)]) if n else np.zeros((0, self.latent + self.rope))

    def each_row(self):
        """(row, sequence, key position) of the batch's rows."""
        for s, n in enumerate(self.lengths):
            for r in range(self.starts[s], self.starts[s + 1]):
                yield r, s, int(n) - int(self.starts[s + 1]) + r

    def upload(self):
        """The batch on the device; `self.device_pool` keeps the pages."""
        raw = np.full(self.pool.size + GUARD, 0xFF, np.uint8)
        raw[:self.pool.size] = self.pool.reshape(-1)
        self.device_pool = DeviceBuffer.from_array(raw)
        self.held = [DeviceBuffer.from_array(a if a.size else np.zeros(1, np.int32))
                     for a in (self.tables, self.lengths, self.starts)]
        return native.LatentBatch(self.type, self.device_pool, self.latent, self.rope, self.pages, self.page,
                                  len(self.lengths), self.held[0], self.width, self.held[1],
                                  self.held[2] if self.use_starts else None)

    def download(self):
        raw = self.device_pool.download(np.uint8)
        assert np.all(raw[self.pool.size:] == 0xFF)
        return raw[:self.pool.size].reshape(self.pool.shape)


def rotate(v, position, freq):
    """Pairs (2i, 2i + 1) of [..., rope] turned by position * freq[i]."""
    a = position * np.asarray(freq, F32).astype(F64)
    c, s = np.cos(a), np.sin(a)
    x, y = v[..., 0::2], v[..., 1::2]
    return np.concatenate([x * c - y * s, y * c + x * s], -1)


def normed(c, w, eps):
    if w is None:
        return c
    return c / np.sqrt((c * c).mean() + F64(F32(eps))) * w.astype(F64)


def attend(cache, q, heads, scale):
    """(out, weight of the magnitudes, largest sum of score magnitudes) of q [rows, heads,
    latent + rope] in f64."""
    out = np.zeros((cache.rows, heads, cache.latent))
    mass, score = np.zeros_like(out), np.zeros((cache.rows, heads, 1))
    longest = [max(int(n), 0) for n in cache.lengths]
    keys = [cache.keys(s, n) for s, n in enumerate(longest)]
    for r, s, j in cache.each_row():
        if j < 0:
            continue
        k = keys[s][:j + 1]
        x = q[r] @ k.T * scale
        with np.errstate(invalid="ignore", over="ignore"):
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[r] = p @ k[:, :cache.latent]
            mass[r] = p @ np.abs(k[:, :cache.latent])
            score[r, :, 0] = (np.abs(q[r]) @ np.abs(k).T * abs(scale)).max(1)
    return out, mass, score


def attend_tolerance(cache, out, mass, score, dtype):
    """A score is a sum of latent + rope products, of three parts each for f32 queries, exact
    but for f32 additions off by at most a last place (2 * 2^-24) of the magnitudes
    added, then two factors and a difference rounded: p is off by a factor of 1 + that (in
    natural logarithms), and the sum of the p by as much.  Sums over n keys and the joins
    of at most 512 parts are f32 additions again; bf16: p rounded, and the result."""
    longest = max(int(cache.lengths.max()), 1)
    terms = (cache.latent + cache.rope) * (1 if dtype == MLK_BF16 else 3)
    p_off = (2 * terms * U.HALF_F32 + 8 * U.HALF_F32) * score + 8 * U.HALF_F32
    room = mass * (2 * p_off + 2 * U.HALF_F32 * (3 * longest + 520))
    if dtype == MLK_BF16:
        room = room + mass * 2 * U.HALF_BF16
        room = room + U.HALF_BF16 * (np.abs(out) + room)
    return room


def typed(dtype, v):
    """(what is uploaded, its values in f64)."""
    if dtype == MLK_BF16:
        bits = U.to_bf16(v.astype(F32))
        return bits, U.from_bf16(bits).astype(F64)
    return v.astype(F32), v.astype(F32).astype(F64)


def values(dtype, raw):
    return (U.from_bf16(raw.view(np.uint16)) if dtype == MLK_BF16 else raw.view(F32)).astype(F64)


def item_size(dtype):
    return 2 if dtype == MLK_BF16 else 4
