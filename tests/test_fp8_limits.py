"""Sizes and offsets at the ends of what the fp8 products' kernels address (fp8.h).
No GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")


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
