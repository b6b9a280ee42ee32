"""SwiGLU rows whose gates are so low that exp(-gate) nears and passes f32's range."""
import numpy as np
import pytest

import fp8_util as U
from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, DeviceBuffer

pytestmark = pytest.mark.gpu

F32 = np.float32


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("up", [1e37, -3.3e38, 2.0 ** 60])
def test_low_gates(device, dtype, up):
    """One value a row, so that each has its own scale.  The results are normal numbers
    above the smallest scale's, down to exp(-gate) = 2^224."""
    g = np.concatenate([np.linspace(-155.0, -70.0, 341), [-88.7228, -88.7229, -87.3365, -87.3366]])
    pair = np.stack([g, np.full_like(g, up)], 1).astype(F32)
    raw = U.to_bf16(pair) if dtype == MLK_BF16 else pair
    g, u = (U.from_bf16(raw) if dtype == MLK_BF16 else raw).astype(np.float64).T
    want = g * np.exp(g) / (1.0 + np.exp(g)) * u
    # above the range where a code or the scale is below its own type's normal range
    some = np.abs(want) > 448 * 2.0 ** -120
    assert some.sum() > 100
    x, q, s = DeviceBuffer.from_array(raw), DeviceBuffer(len(g)), DeviceBuffer(4 * len(g))
    native.swiglu_fp8(dtype, x.ptr, len(g), 1, q.ptr, s.ptr)
    # half places: 2^t 2, its rest's product and sum 2, the two products 2; where the
    # reciprocal is taken 1 + exp 1 and it 2 more
    U.check_codes(q.download(np.uint8)[some, None], s.download(F32)[some, None], want[some, None],
                  9 * U.HALF_F32)


def test_lowest_gates(device):
    """Infinite products of the gate give zeros, an infinite gate NaN as the formula
    does, a NaN gate NaN."""
    x = np.array([[-3e38, 1.0], [-1e6, 3e38], [-np.inf, 1.0], [np.nan, 1.0], [-100.0, 0.0]], F32)
    b, q, s = DeviceBuffer.from_array(x), DeviceBuffer(5), DeviceBuffer(20)
    native.swiglu_fp8(MLK_F32, b.ptr, 5, 1, q.ptr, s.ptr)
    v = U.decode(q.download(np.uint8)) * s.download(F32)
    assert np.all(v[[0, 1, 4]] == 0) and np.isnan(v[[2, 3]]).all()
