// fp8_matmul.hip -- fp8 rows times fp8 matrices, one matrix or one per group of
// rows (gfx950, wave64).
//
//   y[r, o] = sum over blocks b of xs[r, b] ws[o / 128, b] (sum over i in b of x[r, i] w[o, i])
//
// Codes are widened to bf16, which holds every e4m3 value, and multiplied on
// v_mfma_f32_16x16x32_bf16: the products are exact in f32 and a block's 128 are
// added in f32.  Each block's sum is then scaled and added in f32.
//
// Weights are the A operand and rows the B operand: lane l supplies matrix row
// and token l % 16, and of a block of 128 columns the 16-byte chunks l / 16 and
// 4 + l / 16 (which of the lane's values meet in one instruction does not
// matter, as long as both operands agree).  Register r of lane l of a result
// is output column 4 (l / 16) + r of token l % 16, so that a lane scales with
// one factor and stores 4 neighbouring outputs.
#include "fp8.h"
#include "mlh_device.h"
#include "mlh_host.h"

namespace mlh {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ bf16x8 widen8(unsigned lo, unsigned hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ float bf16_float(uint16_t b) {
    return __uint_as_float((unsigned)b << 16);
}
// to the nearest bf16, ties to even; a NaN stays one
__device__ __forceinline__ unsigned float_bf16(float v) {
    const unsigned u = __float_as_uint(v);
    if (v != v) return (u >> 16) | 0x40u;
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// 16 bytes at any address
__device__ __forceinline__ u32x4 load16_any(const uint8_t *p) {
    u32x4 v;
    __builtin_memcpy(&v, p, 16);
    return v;
}

// columns c .. c + 15 of a row of `width` codes, zeros past its end
__device__ __forceinline__ u32x4 load16_tail(const uint8_t *row, int c, int width) {
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (c + i < width) v[i / 4] |= (unsigned)row[c + i] << (8 * (i % 4));
    return v;
}

// The rows of one workgroup's tile: `count` rows from `first` on (entries of y)
// of group `group`; count 0: none.
struct RowTile {
    int group, first, count;
};

// Row tile `slot` of a launch: the groups' tiles one after the other, a wave's
// lanes counting 64 groups at a time.  Offsets that decrease or leave
// [0, rows] are read as empty or shortened groups.
template <int BM> __device__ __forceinline__ RowTile row_tile(const Fp8Matmul &p, int slot) {
    if (p.groups == 0) {
        const int first = slot * BM;
        return RowTile{0, first, min(BM, p.rows - first)};
    }
    const int lane = threadIdx.x & (kWave - 1);
    int before = 0;
    for (int g0 = 0; g0 < p.groups; g0 += kWave) {
        const int g = g0 + lane;
        int start = 0, count = 0;
        if (g < p.groups) {
            start = min(max(p.offsets[g], 0), p.rows);
            count = max(min(p.offsets[g + 1], p.rows), start) - start;
        }
        const int tiles = (count + BM - 1) / BM;
        int incl = tiles;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int v = __shfl_up(incl, o, kWave);
            if (lane >= o) incl += v;
        }
        const int at = slot - before - (incl - tiles);
        const unsigned long long hit = __ballot(at >= 0 && at < tiles);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            const int t = __builtin_amdgcn_readlane(at, src);
            const int s = __builtin_amdgcn_readlane(start, src);
            const int c = __builtin_amdgcn_readlane(count, src);
            return RowTile{g0 + src, s + t * BM, min(BM, c - t * BM)};
        }
        before += __builtin_amdgcn_readlane(incl, kWave - 1);
    }
    return RowTile{0, 0, 0};
}

// Row tiles that `rows` entries in `groups` groups can need.
template <int BM> long row_tiles(const Fp8Matmul &p) {
    if (p.groups == 0) return ((long)p.rows + BM - 1) / BM;
    const long used = p.groups < p.rows ? p.groups : p.rows;  // groups that can hold a row
    return (p.rows + used * (BM - 1)) / BM;
}

// Four neighbouring outputs of a row; those from O on are left out.
template <bool BF16>
__device__ __forceinline__ void store4(const Fp8Matmul &p, long row, int o, f32x4 v) {
    const long at = row * p.O + o;
    if (o + 4 <= p.O && p.O % 4 == 0) {
        if constexpr (BF16) {
            uint16_t *y = static_cast<uint16_t *>(p.y) + at;
            if (p.resid) {
                const uint16_t *r = static_cast<const uint16_t *>(p.resid) + at;
                uint16_t h[4];
                __builtin_memcpy(h, r, 8);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] += bf16_float(h[i]);
            }
            const unsigned u[2] = {float_bf16(v[0]) | (float_bf16(v[1]) << 16),
                                   float_bf16(v[2]) | (float_bf16(v[3]) << 16)};
            __builtin_memcpy(y, u, 8);
        } else {
            float *y = static_cast<float *>(p.y) + at;
            if (p.resid) {
                f32x4 r;
                __builtin_memcpy(&r, static_cast<const float *>(p.resid) + at, 16);
                v += r;
            }
            __builtin_memcpy(y, &v, 16);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (o + i >= p.O) break;
        if constexpr (BF16) {
            float r = p.resid ? bf16_float(static_cast<const uint16_t *>(p.resid)[at + i]) : 0.0f;
            static_cast<uint16_t *>(p.y)[at + i] = (uint16_t)float_bf16(v[i] + r);
        } else {
            float r = p.resid ? static_cast<const float *>(p.resid)[at + i] : 0.0f;
            static_cast<float *>(p.y)[at + i] = v[i] + r;
        }
    }
}

// Both operands straight from memory into registers, any width and alignment.
// A wave holds NT x MT results of 16 x 16; WO waves share the tile's tokens, WM
// its matrix rows, and WK waves take every WK-th block of columns, added
// through LDS.
template <int NT_, int MT_, int WO_, int WM_, int WK_> struct DirectShape {
    static constexpr int NT = NT_, MT = MT_, WO = WO_, WM = WM_, WK = WK_;
    static constexpr int kWaves = WO * WM * WK;
    static constexpr int kThreads = kWaves * kWave;
    static constexpr int BO = 16 * NT * WO, BM = 16 * MT * WM;
};

template <class Sh, bool BF16>
__global__ __launch_bounds__(Sh::kThreads) void fp8_direct_kernel(Fp8Matmul p, int o_tiles) {
    constexpr int NT = Sh::NT, MT = Sh::MT, WO = Sh::WO, WM = Sh::WM, WK = Sh::WK;
    __shared__ f32x4 red[WK > 1 ? (WK - 1) * WO * WM * NT * MT * kWave : 1];
    const int slot = blockIdx.x / o_tiles;
    const RowTile rt = row_tile<Sh::BM>(p, slot);
    if (rt.count <= 0) return;  // the same for the whole workgroup
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int l16 = lane & 15, quad = lane >> 4;
    const int wk = wave % WK, wo = wave / WK % WO, wm = wave / (WK * WO);
    const int o0 = (blockIdx.x - slot * o_tiles) * Sh::BO + wo * 16 * NT;
    const int m0 = wm * 16 * MT;
    const int blocks = (p.I - 1) / kFp8Block + 1, whole = p.I / kFp8Block;
    const int o_blocks = (p.O - 1) / kFp8Block + 1;
    const uint8_t *wbase = p.w + (long)rt.group * p.O * p.I;
    const float *wsbase = p.ws + (long)rt.group * o_blocks * blocks;

    // rows past the tile's end are those of its last one, columns past O those
    // of the last: neither is stored
    const uint8_t *wrow[NT], *xrow[MT];
    const float *wsrow[NT], *xsrow[MT];
    bool bad[MT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int o = min(o0 + 16 * n, p.O - 1);
        wrow[n] = wbase + (long)min(o0 + 16 * n + l16, p.O - 1) * p.I;
        wsrow[n] = wsbase + (long)(o / kFp8Block) * blocks;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        int r = rt.first + min(m0 + 16 * m + l16, rt.count - 1);
        bad[m] = false;
        if (p.row_ids) {
            r = p.row_ids[r];
            bad[m] = r < 0 || r >= p.x_rows;
            if (bad[m]) r = 0;
        }
        xrow[m] = p.x + (long)r * p.I;
        xsrow[m] = p.xs + (long)r * blocks;
    }

    struct Step {
        u32x4 w[NT][2], x[MT][2];
        float ws[NT], xs[MT];
    };
    auto load = [&](Step &s, int b) {
        const int c = b * kFp8Block + 16 * quad;
        if (b < whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int n = 0; n < NT; ++n) s.w[n][h] = load16_any(wrow[n] + c + 64 * h);
#pragma unroll
                for (int m = 0; m < MT; ++m) s.x[m][h] = load16_any(xrow[m] + c + 64 * h);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int n = 0; n < NT; ++n) s.w[n][h] = load16_tail(wrow[n], c + 64 * h, p.I);
#pragma unroll
                for (int m = 0; m < MT; ++m) s.x[m][h] = load16_tail(xrow[m], c + 64 * h, p.I);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) s.ws[n] = wsrow[n][b];
#pragma unroll
        for (int m = 0; m < MT; ++m) s.xs[m] = xsrow[m][b];
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0, 0, 0, 0};
    auto multiply = [&](const Step &s) {
        f32x4 d[NT][MT];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int h = q / 2, e = 2 * (q % 2);
            bf16x8 x[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m] = widen8(s.x[m][h][e], s.x[m][h][e + 1]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bf16x8 w = widen8(s.w[n][h][e], s.w[n][h][e + 1]);
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    d[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        w, x[m], q == 0 ? f32x4{0, 0, 0, 0} : d[n][m], 0, 0, 0);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const float f = s.ws[n] * s.xs[m];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(d[n][m][i], f, acc[n][m][i]);
            }
    };
    Step s0, s1;
    if (wk < blocks) load(s0, wk);
    for (int b = wk; b < blocks; b += 2 * WK) {
        if (b + WK < blocks) load(s1, b + WK);
        multiply(s0);
        if (b + WK >= blocks) break;
        if (b + 2 * WK < blocks) load(s0, b + 2 * WK);
        multiply(s1);
    }

    if constexpr (WK > 1) {
        f32x4 *mine = red + ((long)(wk - 1) * WO * WM + wm * WO + wo) * NT * MT * kWave + lane;
        if (wk > 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) mine[(n * MT + m) * kWave] = acc[n][m];
        }
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int k = 1; k < WK; ++k) {
            const f32x4 *other = red + ((long)(k - 1) * WO * WM + wm * WO + wo) * NT * MT * kWave + lane;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[n][m] += other[(n * MT + m) * kWave];
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = m0 + 16 * m + l16;
        if (r >= rt.count) continue;
        const float nan = __int_as_float(0x7fc00000);
#pragma unroll
        for (int n = 0; n < NT; ++n)
            store4<BF16>(p, rt.first + r, o0 + 16 * n + 4 * quad,
                         bad[m] ? f32x4{nan, nan, nan, nan} : acc[n][m]);
    }
}

constexpr long kMaxGrid = 0xFFFFFF;  // workgroups of 256 threads in a launch

template <class Sh> int launch_direct(const Fp8Matmul &p, hipStream_t stream) {
    const long o_tiles = ((long)p.O + Sh::BO - 1) / Sh::BO;
    const long tiles = row_tiles<Sh::BM>(p) * o_tiles;
    if (tiles > kMaxGrid) return kErrSize;
    if (tiles == 0) return kOk;
    if (p.bf16)
        hipLaunchKernelGGL((fp8_direct_kernel<Sh, true>), dim3((unsigned)tiles), dim3(Sh::kThreads),
                           0, stream, p, (int)o_tiles);
    else
        hipLaunchKernelGGL((fp8_direct_kernel<Sh, false>), dim3((unsigned)tiles),
                           dim3(Sh::kThreads), 0, stream, p, (int)o_tiles);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace

int fp8_matmul(const Fp8Matmul &p, hipStream_t stream) {
    if (p.rows == 0) return kOk;
    const long per_group = p.groups ? (p.rows + p.groups - 1) / p.groups : p.rows;
    if (per_group <= 16) return launch_direct<DirectShape<1, 1, 1, 1, 4>>(p, stream);
    return launch_direct<DirectShape<2, 2, 2, 2, 1>>(p, stream);
}

}  // namespace mlh
