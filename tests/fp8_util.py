"""e4m3 codes and bf16 bits in numpy, and the formulas of the fp8 entry points in
64 bits.

Codes: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f / 0xff are NaN, there
is no infinity and the largest value is 448."""
import numpy as np

F32 = np.float32
HALF_F32 = 2.0 ** -24
HALF_BF16 = 2.0 ** -8
TOP, TINY, BLOCK = F32(448.0), F32(2.0 ** -126), 128


def _table():
    code = np.arange(256)
    exp, frac = (code >> 3) & 15, code & 7
    v = np.where(exp == 0, frac * 2.0 ** -9, (8 + frac) * 2.0 ** (exp - 10.0))
    v[(code & 0x7f) == 0x7f] = np.nan
    return np.where(code >> 7, -v, v)


VALUES = _table()
# midpoints between the 127 magnitudes: the code of a magnitude is the number of
# midpoints below it (ties settled apart)
_MID = (VALUES[:126] + VALUES[1:127]) / 2


def decode(codes):
    return VALUES[np.asarray(codes, np.uint8)]


def encode(v):
    """Nearest code, ties to the even one; magnitudes up to 464 only."""
    v = np.asarray(v, np.float64)
    a = np.abs(v)
    assert not np.any(a > 464.0)
    lo = np.searchsorted(_MID, a, side="left")  # a tie goes down
    tie = (lo < 126) & (a == _MID[np.minimum(lo, 125)])
    code = np.where(tie & (lo % 2 == 1), lo + 1, lo)
    code = np.where(np.signbit(v), code | 0x80, code)
    return np.where(np.isnan(v), 0x7f, code).astype(np.uint8)


def step(v):
    """Distance of neighbouring codes at magnitude v."""
    e = np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6)))
    return 2.0 ** (e - 3)


def to_bf16(v):
    """f32 -> bf16 bits, to nearest, ties to even."""
    u = np.ascontiguousarray(v, F32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(F32)


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def spread(scale, rows, cols, block_rows):
    """Scales as one number per value."""
    wide = np.repeat(scale, BLOCK, -1)[..., :cols]
    return np.repeat(wide, block_rows, -2)[..., :rows, :] if block_rows > 1 else wide


def amax_blocks(v, block_rows):
    rows, cols = v.shape
    a = np.abs(np.where(np.isnan(v), 0.0, v))
    a = np.pad(a, ((0, -rows % block_rows), (0, -cols % BLOCK)))
    return a.reshape(-1, block_rows, blocks(cols), BLOCK).max((1, 3))


def quantize(x, block_rows):
    """The codes and scales that the formula in f32 gives, bit for bit."""
    x = np.asarray(x, F32)
    with np.errstate(all="ignore"):
        scale = np.maximum(amax_blocks(x, block_rows).astype(F32) / TOP, TINY)
        inv = F32(1.0) / scale
        code = encode(x * spread(inv, *x.shape, block_rows))
    return code, scale


def dequantize(code, scale, block_rows):
    return decode(code) * spread(scale.astype(np.float64), *code.shape[-2:], block_rows)


def check_codes(code, scale, v, delta):
    """Codes and 1 x 128 scales of values that the kernel computed within `delta`
    (relative) of v: the scale is off by delta and its own quotient's rounding; a
    code is a nearest one of a value off by delta and the three roundings of
    x * (1 / s) and s."""
    want = np.maximum(amax_blocks(v, 1) / 448.0, 2.0 ** -126)
    np.testing.assert_allclose(scale, want, rtol=delta + 2 * HALF_F32, atol=0)
    q = np.abs(v) / spread(scale.astype(np.float64), *v.shape, 1)
    off = np.abs(decode(code) - v / spread(scale.astype(np.float64), *v.shape, 1))
    room = q * (delta + 4 * HALF_F32)
    assert np.all(off <= step(q + room) / 2 + room), np.max(off / (step(q + room) / 2 + room))


def product(x, xs, w, ws):
    """(y, mass, top): the product in 64 bits, the sum of the magnitudes added, and the
    sum of the largest magnitude of each 8 neighbouring columns."""
    a, b = dequantize(x, xs, 1), dequantize(w, ws, BLOCK)
    top = np.zeros((a.shape[0], b.shape[0]))
    for c in range(0, a.shape[1], 8):
        part = np.zeros_like(top)
        for i in range(c, min(c + 8, a.shape[1])):
            np.maximum(part, np.abs(a[:, i, None] * b[None, :, i]), out=part)
        top += part
    return a @ b.T, np.abs(a) @ np.abs(b).T, top


def product_tolerance(y, mass, top, inp, out_bf16, resid=None):
    """A sum of n f32 additions in any order, each off by at most a whole last
    place (2 * 2^-24: to nearest or cut off), is within n * 2^-23 of the magnitudes
    added; per output 128 in a block, then a rounded factor and an addition per
    block, and up to 8 more where waves join their shares or a residual is added.
    Products for bf16 outputs may come from fp8 matrix instructions, which add 8
    neighbouring products after cutting each below 2^-13 of the largest's power of
    two."""
    n = min(inp, BLOCK) + 2 * blocks(inp) + 8
    room = n * 2 * HALF_F32 * (mass if resid is None else mass + np.abs(resid))
    total = y if resid is None else y + resid
    if not out_bf16:
        return room
    room = room + 8 * 2.0 ** -13 * top
    return room + HALF_BF16 * (np.abs(total) + room)
