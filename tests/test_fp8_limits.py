"""Sizes and offsets at the ends of what the fp8 products' kernels address (fp8.h).
No GPU."""
import os
import shutil
import subprocess

import pytest

from floyd_amd import native
from floyd_amd.native import MLK_BF16, MLK_F32, NativeError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

needs_hipcc = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
P = 1 << 20  # stands for an address; the refusals below never look at it


def host_program(tmp_path, body):
    """The integers that a host program over fp8.h prints."""
    src, exe = tmp_path / "values.cpp", tmp_path / "values"
    src.write_text('#include <cstdio>\n#include "fp8.h"\n'
                   "using namespace mlh;\nint main() { %s }\n" % body)
    subprocess.run([HIPCC, "-std=c++17", "--cuda-host-only", "-x", "hip",
                    "-I" + os.path.join(ROOT, "floyd_amd", "csrc"),
                    "-I" + os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    return [int(v) for v in out.split()]


@needs_hipcc
def test_scalar_offsets_stay_inside_one_row(tmp_path):
    """The streams' rings and the tiles' next scale group run past the last block of
    columns (at most 8 waves of 4 stages ahead).  The scalar offset of such a copy is
    0; every other lies inside a buffer of one row of codes, and one of scales."""
    wrong = host_program(tmp_path, """
        for (int width = 1; width <= 5000; ++width) {
            const int blocks = fp8_blocks(width);
            for (int b = 0; b < blocks + 8 * 5; ++b) {
                const int codes = fp8_scalar_offset(b, blocks, kFp8Block);
                const int scales = fp8_scalar_offset(b, blocks, 4);
                const bool live = b < blocks;
                if (codes != (live ? b * 128 : 0) || codes >= width || scales != (live ? b * 4 : 0) ||
                    scales >= blocks * 4)
                    printf("%d %d ", width, b);
            }
        }""")
    assert wrong == []


@needs_hipcc
def test_scales_in_reach(tmp_path):
    """Scale offsets, f32 a block of 128 columns, of `rows` rows: all end at 0xF0000000
    bytes or below, in 64-bit arithmetic, at every width up to 2^30."""
    rows = (1, 8, 64, 119, 120, 128, 256, 1 << 22, (1 << 31) - 1)
    widths = (1, 128, 129, 2048, 11264, 1 << 22, (1 << 22) + 1, 1 << 29, (1 << 30) - 128, 1 << 30)
    got = host_program(tmp_path, "".join('printf("%%d ", (int)fp8_scales_in_reach(%dL, %d));' % (r, w)
                                         for r in rows for w in widths))
    assert got == [int(r * -(-w // 128) * 4 < 0xF0000000) for r in rows for w in widths]
    # the widest rows leave the smaller tiles and all streams
    assert [r for r in (8, 16, 32, 64, 128, 256) if r * 2 ** 23 * 4 < 0xF0000000] == [8, 16, 32, 64]


@pytest.mark.parametrize("dtype", [MLK_F32, MLK_BF16])
@pytest.mark.parametrize("x_rows,inp", [((1 << 31) - 1, 128), (0x3C000000, 1), (0x1E000000, 256),
                                        (120, 1 << 30)])
def test_gathered_scales_out_of_reach_are_refused(dtype, x_rows, inp):
    with pytest.raises(NativeError, match=r"-4.*x_rows"):
        native.matmul_fp8_grouped(dtype, P, P, P, P, P, 64, inp, 3, P, 4, row_ids=P, x_rows=x_rows)


@pytest.mark.parametrize("more", [dict(x_rows=0x3C000000 - 1, row_ids=P), dict(x_rows=0x3C000000)])
def test_scales_in_reach_are_taken(more):
    """One row less, or rows that are not gathered: refused for the addresses only."""
    with pytest.raises(NativeError, match="no HIP device|not device memory"):
        native.matmul_fp8_grouped(MLK_F32, P, P, P, P, P, 64, 128, 3, P, 4, **more)
