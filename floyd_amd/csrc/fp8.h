// fp8.h -- fp8 rows, matrices and their products (internal).
//
// A value is code * scale: e4m3 codes (the OCP format: largest value 448, one
// NaN per sign, no infinity) with one f32 scale per block of 128 columns of a
// row (activations) or of 128 x 128 (weights).  Blocks start at row and column
// 0; the last ones may be narrower.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlh {

constexpr int kFp8Block = 128;
constexpr float kFp8Top = 448.0f;
// the smallest scale: that of a block of zeros, and of one whose largest value
// is below 448 * 2^-126 (a subnormal scale would lose bits of its own)
constexpr float kFp8TinyScale = 0x1p-126f;

// Columns of a row are counted in 32 bits, with room for a step past the last.
constexpr int kFp8MaxWidth = 1 << 30;

inline int fp8_blocks(int n) { return (n - 1) / kFp8Block + 1; }  // n > 0

// Offsets from a buffer's first row stay below this; a load at it is out of the buffer.
constexpr long kFp8Outside = 0xF0000000L;
// Whether the scales of `rows` rows, a tile's or all that row_ids may name, are reached by
// such offsets.
inline bool fp8_scales_in_reach(long rows, int I) {
    return rows * fp8_blocks(I) * 4 < kFp8Outside;
}

// Scalar offset of a copy of column block b, `bytes` a block.  The range check takes it
// from the buffer's length before it looks at a lane's offset, so it has to stay inside
// the buffer: a copy past the last block, whose lanes are all out of range, takes 0.
__host__ __device__ constexpr int fp8_scalar_offset(int b, int blocks, int bytes) {
    return b < blocks ? b * bytes : 0;
}

// Rows to quantise.  bf16: x (and resid, sum) are bfloat16, else f32.
struct Fp8Rows {
    bool bf16 = false;
    const void *x = nullptr;
    int rows = 0, cols = 0;
    uint8_t *q = nullptr;
    float *scale = nullptr;
};

// block_rows 1 or 128
int fp8_quantize(const Fp8Rows &p, int block_rows, hipStream_t stream);
// h = x + resid (resid may be null), stored to sum when that is set (it may be
// x or resid); the RMSNorm of the stored h, quantised
int fp8_rmsnorm(const Fp8Rows &p, const void *resid, const float *norm_w, float eps, void *sum,
                hipStream_t stream);
// x: rows of cols gate values, then cols up values; silu(gate) * up, quantised
int fp8_swiglu(const Fp8Rows &p, hipStream_t stream);

// y[r, o] = sum over column blocks b of xs[r, b] ws[o / 128, b] (x_r . w_o over b)
struct Fp8Matmul {
    const uint8_t *w = nullptr;   // [groups, O, I]
    const float *ws = nullptr;    // [groups, ceil(O / 128), ceil(I / 128)]
    const uint8_t *x = nullptr;   // [x_rows, I]
    const float *xs = nullptr;    // [x_rows, ceil(I / 128)]
    void *y = nullptr;            // [rows, O], f32 or bf16
    const void *resid = nullptr;  // [rows, O] of y's type, optional
    bool bf16 = false;
    int O = 0, I = 0, rows = 0;
    // grouped: rows offsets[g] .. offsets[g + 1] of y belong to matrix g;
    // rows = the entries of y, x row of entry j = row_ids ? row_ids[j] : j
    int groups = 0;  // 0: one matrix for every row
    const int *offsets = nullptr;
    const int *row_ids = nullptr;
    int x_rows = 0;
};
int fp8_matmul(const Fp8Matmul &p, hipStream_t stream);

}  // namespace mlh
