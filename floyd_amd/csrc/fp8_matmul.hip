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
#include <stdlib.h>

namespace mlh {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

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

// EACH neighbouring outputs of a row, 16 bytes, from LDS; those from O on are left out.
template <bool BF16, int EACH>
__device__ __forceinline__ void store_row(const Fp8Matmul &p, long row, int o, const float *v) {
    const long at = row * p.O + o;
    float f[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i += 4) {
        const f32x4 x = load_f4(v + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) f[i + k] = x[k];
    }
    constexpr int kSize = BF16 ? 2 : 4;
    if (o + EACH <= p.O && (long)p.O * kSize % 16 == 0) {
        const long byte = at * kSize;
        if (p.resid) {
            const u32x4 r = load16_any(static_cast<const uint8_t *>(p.resid) + byte);
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                if constexpr (BF16) f[i] += bf16_float((uint16_t)(r[i / 2] >> (16 * (i % 2))));
                else f[i] += __uint_as_float(r[i]);
            }
        }
        u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF16) u[i] = float_bf16(f[2 * i]) | (float_bf16(f[2 * i + 1]) << 16);
            else u[i] = __float_as_uint(f[i]);
        }
        __builtin_memcpy(static_cast<uint8_t *>(p.y) + byte, &u, 16);
        return;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (o + i >= p.O) break;
        if constexpr (BF16) {
            if (p.resid) f[i] += bf16_float(static_cast<const uint16_t *>(p.resid)[at + i]);
            static_cast<uint16_t *>(p.y)[at + i] = (uint16_t)float_bf16(f[i]);
        } else {
            if (p.resid) f[i] += static_cast<const float *>(p.resid)[at + i];
            static_cast<float *>(p.y)[at + i] = f[i];
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

// ---------------------------------------------------------------------------
// Tiles through LDS, for many rows
// ---------------------------------------------------------------------------
//
// A workgroup of WO x WM waves makes BO matrix rows x BM tokens; a wave NT x MT
// results of 16 x 16.  Each step of 128 columns is copied by DMA into one of
// `STAGES` LDS stages while the ones before it are multiplied: rows of 128 bytes as
// they lie in memory, 16-byte chunk c of row r at chunk c ^ (r / 2 & 7), so
// that the rows an operand read touches lie on different banks; the row and
// matrix scales behind them, copied in pieces of kSpan steps: a scale a
// token and step is 4 bytes of its own cache line, and copying each step's alone
// asked the L2 for as many lines as the operands.
constexpr int kSpan = 8;
template <int BO_, int BM_, int WO_, int WM_, int STAGES_> struct TileShape {
    static constexpr int BO = BO_, BM = BM_, WO = WO_, WM = WM_, kStages = STAGES_;
    static constexpr int kWaves = WO * WM, kThreads = kWaves * kWave;
    static constexpr int NT = BO / 16 / WO, MT = BM / 16 / WM;
    static constexpr int kStage = (BO + BM) * kFp8Block;
    // scales: two groups of kSpan steps, each BM / 8 pieces of 8 tokens by kSpan steps and
    // one of matrix blocks; behind them the place of copies that stand for none
    static constexpr int kPieces = BM / 8 + 1;
    static constexpr int kScales = kStages * kStage, kScaleGroup = kPieces * 256;
    static constexpr int kIdle = kScales + 2 * kScaleGroup;
    // offsets of the rows' scales: BM tokens, 8 matrix blocks, 8 that stand for none
    static constexpr int kRowOffsets = kIdle + 256;
    static constexpr int kLds = kRowOffsets + (BM + 16) * 4;
    static constexpr int kWPer = BO / 8 / kWaves, kXPer = BM / 8 / kWaves;  // DMA blocks of a wave
    static constexpr int kDma = kWPer + kXPer;
    static_assert(BO % (8 * kWaves) == 0 && BM % (8 * kWaves) == 0, "whole DMA blocks");
    static_assert((kPieces + kWaves - 1) / kWaves <= kSpan - (kStages - 2) && BO / kFp8Block <= 8,
                  "a group's scales land before its first step");
    static_assert(BO / 16 % WO == 0 && BM / 16 % WM == 0 && kFp8Block % (16 * NT) == 0,
                  "a wave's matrix rows lie in one block");
    static_assert(kLds <= 160 * 1024 && (kStages - 1) * (kDma + 1) < 64, "LDS, vmcnt");
};

template <int N> __device__ __forceinline__ void wait_vmcnt() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// Offsets from a tile's first row stay below this; a load at it is out of the buffer.
constexpr long kOutside = 0xF0000000L;

// Buffer of `bytes` from base: loads at offsets of that and more read zero.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void *base, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (unsigned)min(bytes, kOutside),
                                             0x00027000);
}

typedef __attribute__((address_space(3))) uint8_t LdsByte;

// 16 or 4 bytes a lane from voffset + soffset to consecutive LDS bytes.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t buf, unsigned voffset, int soffset, LdsByte *dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, dst, 16, voffset, soffset, 0, 0);
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t buf, unsigned voffset, int soffset, LdsByte *dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, dst, 4, voffset, soffset, 0, 0);
}

// Group tiles of a launch, all groups together (the same in every lane).
template <int BM> __device__ __forceinline__ int used_tiles(const Fp8Matmul &p) {
    if (p.groups == 0) return (p.rows - 1) / BM + 1;
    const int lane = threadIdx.x & (kWave - 1);
    int n = 0;
    for (int g = lane; g < p.groups; g += kWave) {
        const int start = min(max(p.offsets[g], 0), p.rows);
        n += (max(min(p.offsets[g + 1], p.rows), start) - start + BM - 1) / BM;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o, kWave);
    return __builtin_amdgcn_readfirstlane(n);
}

constexpr int kTileGroup = 4;  // row tiles that share matrix rows, one after the other

template <class Sh, bool FAST, bool BF16>
__global__ __launch_bounds__(Sh::kThreads, 2) void fp8_tile_kernel(Fp8Matmul p, int o_tiles, int slots) {
    constexpr int NT = Sh::NT, MT = Sh::MT, BO = Sh::BO, BM = Sh::BM, S = Sh::kStages;
    constexpr int kWaves = Sh::kWaves;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // Workgroups go to the 8 XCDs in turn: each XCD gets a run of neighbouring
    // tiles, kTileGroup row tiles by all matrix rows, whose operands its L2 holds.
    int slot, o_tile;
    {
        const int used = min(used_tiles<BM>(p), slots);
        const int total = used * o_tiles, per = (total + 7) / 8;
        const int tile = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
        if ((int)(blockIdx.x >> 3) >= per || tile >= total) return;
        const int grp = tile / (kTileGroup * o_tiles), rem = tile - grp * kTileGroup * o_tiles;
        const int size = min(kTileGroup, used - grp * kTileGroup);
        slot = grp * kTileGroup + rem % size;
        o_tile = rem / size;
    }
    RowTile rt = row_tile<BM>(p, slot);
    if (rt.count <= 0) return;
    rt.group = __builtin_amdgcn_readfirstlane(rt.group);  // (known to be one value, for the buffers)
    rt.first = __builtin_amdgcn_readfirstlane(rt.first);
    rt.count = __builtin_amdgcn_readfirstlane(rt.count);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, quad = lane >> 4;
    const int wo = wave % Sh::WO, wm = wave / Sh::WO;
    const int o0 = o_tile * BO;
    const int blocks = (p.I - 1) / kFp8Block + 1;
    const int o_blocks = (p.O - 1) / kFp8Block + 1;

    // ---- copies: a DMA block is 8 rows of 128 bytes, wave w takes blocks w, w +
    // kWaves, ...; lane l fills chunk l % 8 of row l / 8
    const int dma_row = lane >> 3;
    const uint8_t *const w_base = p.w + ((long)rt.group * p.O + o0) * p.I;
    const float *const ws_base = p.ws + ((long)rt.group * o_blocks + o0 / kFp8Block) * blocks;
    const long x_first = p.row_ids ? 0 : rt.first, x_count = p.row_ids ? p.x_rows : rt.count;
    const uint8_t *const x_base = p.x + x_first * p.I;
    const float *const xs_base = p.xs + x_first * blocks;
    const long w_bytes = (long)(p.O - o0) * p.I, x_bytes = x_count * p.I;
    auto x_row = [&](int m) -> int {  // buffer row of token m; -1: none, or an id out of range
        if (m >= rt.count) return -1;
        if (!p.row_ids) return m;
        const int r = p.row_ids[rt.first + m];
        return r >= 0 && r < p.x_rows ? r : -1;
    };
    unsigned x_off[Sh::kXPer];
#pragma unroll
    for (int q = 0; q < Sh::kXPer; ++q) {
        const int r = x_row((wave + kWaves * q) * 8 + dma_row);
        x_off[q] = r < 0 ? (unsigned)kOutside : (unsigned)r * (unsigned)p.I;
    }
    const unsigned w_off = (unsigned)(wave * 8 + dma_row) * (unsigned)p.I;
    // A piece of scales: lane l takes step l / 8 of the group and token (or matrix
    // block) l % 8; piece j of a group is copied by wave j % kWaves.
    const long xs_bytes = x_count * blocks * 4, ws_bytes = (long)(o_blocks - o0 / kFp8Block) * blocks * 4;
    const int sc_lane = lane & 7, sc_step = lane >> 3;
    unsigned *const row_off = reinterpret_cast<unsigned *>(lds + Sh::kRowOffsets);
    for (int i = threadIdx.x; i < BM + 16; i += Sh::kThreads) {
        const int r = i < BM ? x_row(i) : i - BM < BO / kFp8Block ? i - BM : -1;
        row_off[i] = r < 0 ? (unsigned)kOutside : (unsigned)r * (unsigned)blocks * 4u;
    }
    __syncthreads();
    auto scale_row = [&](int q) {  // for this wave's piece q of a group
        return row_off[min(q * kWaves + wave, BM / 8 + 1) * 8 + sc_lane];
    };
    auto copy_scales = [&](int g, int q, unsigned row) {
        const int piece = q * kWaves + wave;
        const bool rows = piece < BM / 8;
        const bool in = g * kSpan + sc_step < blocks && row != (unsigned)kOutside;
        dma4(buffer_of(rows ? xs_base : ws_base, rows ? xs_bytes : ws_bytes),
             in ? row + sc_step * 4u : (unsigned)kOutside, g * kSpan * 4,
             (LdsByte *)(lds + (piece <= BM / 8 ? Sh::kScales + (g & 1) * Sh::kScaleGroup + piece * 256
                                                : Sh::kIdle)));
    };
    // the operands of step b
    auto copy_tiles = [&](int b, int st) {
        LdsByte *stage = (LdsByte *)(lds + st * Sh::kStage);
        const int k0 = b * kFp8Block;
#pragma unroll
        for (int i = 0; i < Sh::kDma; ++i) {
            const int q = i < Sh::kWPer ? i : i - Sh::kWPer;
            const int blk = wave + kWaves * q;
            const int chunk = (lane & 7) ^ ((blk & 1) * 4 + dma_row / 2);
            // a row that ends inside the step, or before it: zeros past its end
            const bool past = k0 + kFp8Block > p.I && k0 + chunk * 16 >= p.I;
            if (i < Sh::kWPer)
                dma16(buffer_of(w_base, w_bytes),
                      past ? (unsigned)kOutside
                           : w_off + (unsigned)(q * kWaves * 8) * (unsigned)p.I + (unsigned)(chunk * 16),
                      k0, stage + blk * 1024);
            else
                dma16(buffer_of(x_base, x_bytes),
                      past || x_off[q] == (unsigned)kOutside ? (unsigned)kOutside
                                                             : x_off[q] + (unsigned)(chunk * 16),
                      k0, stage + BO * kFp8Block + blk * 1024);
        }
    };

    f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0, 0, 0, 0};

    // Operand of 16 rows from LDS row r0 on: this lane's chunks quad and quad + 4.
    const int frag0 = l16 * kFp8Block + ((quad ^ (l16 >> 1)) << 4);
    const int frag1 = l16 * kFp8Block + (((quad + 4) ^ (l16 >> 1)) << 4);
    auto read_frag = [&](const uint8_t *tile, int r0, u32x4 (&f)[2]) {
        f[0] = *reinterpret_cast<const u32x4 *>(tile + r0 * kFp8Block + frag0);
        f[1] = *reinterpret_cast<const u32x4 *>(tile + r0 * kFp8Block + frag1);
    };
    const bool live = wm * 16 * MT < rt.count;  // a wave without tokens copies only
    auto multiply = [&](int step, int st) {
        const uint8_t *stage = lds + st * Sh::kStage;
        const uint8_t *wt = stage, *xt = stage + BO * kFp8Block;
        const float *sc = reinterpret_cast<const float *>(lds + Sh::kScales + step / kSpan % 2 * Sh::kScaleGroup) +
                          step % kSpan * 8;
        const float ws = sc[BM / 8 * 64 + wo * 16 * NT / kFp8Block];
        float f[MT];
        u32x4 xf[MT][2], wf[2][2];
        f32x4 d[2][MT];
        read_frag(wt, wo * 16 * NT, wf[0]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            read_frag(xt, wm * 16 * MT + 16 * m, xf[m]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) f[m] = ws * sc[(wm * 2 * MT + 2 * m + l16 / 8) * 64 + l16 % 8];
        if constexpr (FAST) {
#pragma unroll
            for (int n = 0; n <= NT; ++n) {
                if (n + 1 < NT) read_frag(wt, wo * 16 * NT + 16 * (n + 1), wf[(n + 1) & 1]);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    if (n < NT) {
                        const u32x4 *a = wf[n & 1], *x = xf[m];
                        const i32x8 wa = {(int)a[0][0], (int)a[0][1], (int)a[0][2], (int)a[0][3],
                                          (int)a[1][0], (int)a[1][1], (int)a[1][2], (int)a[1][3]};
                        const i32x8 xa = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3],
                                          (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
                        d[n & 1][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                            wa, xa, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
                    }
                    if (n > 0) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[n - 1][m][i] = fmaf(d[(n - 1) & 1][m][i], f[m], acc[n - 1][m][i]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        } else {
            bf16x8 xb[MT][4];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    xb[m][q] = widen8(xf[m][q / 2][2 * (q % 2)], xf[m][q / 2][2 * (q % 2) + 1]);
#pragma unroll
            for (int n = 0; n <= NT; ++n) {
                if (n + 1 < NT) read_frag(wt, wo * 16 * NT + 16 * (n + 1), wf[(n + 1) & 1]);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    bf16x8 a;
                    if (n < NT) a = widen8(wf[n & 1][q / 2][2 * (q % 2)], wf[n & 1][q / 2][2 * (q % 2) + 1]);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        if (n < NT)
                            d[n & 1][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                a, xb[m][q], q == 0 ? f32x4{0, 0, 0, 0} : d[n & 1][m], 0, 0, 0);
                        if (n > 0 && q == 0) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                acc[n - 1][m][i] = fmaf(d[(n - 1) & 1][m][i], f[m], acc[n - 1][m][i]);
                        }
                    }
                }
            }
        }
    };
    // A wave's DMA completes in order: a step has landed when at most the copies of
    // the later steps in flight remain.  The barrier after the wait makes every
    // wave's part visible and frees the stage read last.  (A bare barrier:
    // __syncthreads() would wait for the DMA in flight as well.)
#pragma unroll
    for (int q = 0; q < (Sh::kPieces + kWaves - 1) / kWaves; ++q) copy_scales(0, q, scale_row(q));
#pragma unroll
    for (int b = 0; b < S - 1; ++b)
        copy_tiles(b, b);
    int st = 0, fill = S - 1;
    for (int b = 0; b < blocks; ++b) {
        if (S == 2) wait_vmcnt<0>();
        else if (b > 0) wait_vmcnt<(S - 2) * (Sh::kDma + 1)>();
        else wait_vmcnt<(S - 2) * Sh::kDma>();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        copy_tiles(b + S - 1, fill);
        copy_scales(b / kSpan + 1, b % kSpan, scale_row(b % kSpan));  // a part of the next group's
        if (live) multiply(b, st);
        st = st + 1 == S ? 0 : st + 1;
        fill = fill + 1 == S ? 0 : fill + 1;
    }
    wait_vmcnt<0>();  // no copy is in flight when the LDS is given back

    // Results go to memory through LDS, 16 tokens of a wave at a time: the lanes of a
    // result hold 16 different rows, whose pieces the memory pipe takes one by one,
    // while 16 neighbouring bytes a lane and a row's pieces on neighbouring lanes are
    // taken 4 lanes at a time.
    __syncthreads();  // every wave has read its operands
    if (!live) return;
    constexpr int kPitch = 16 * NT + 4;  // floats
    static_assert(kWaves * 16 * kPitch * 4 <= Sh::kRowOffsets, "results of 16 tokens a wave");
    float *const out = reinterpret_cast<float *>(lds) + wave * 16 * kPitch;
    const int o_wave = o0 + wo * 16 * NT;
    const float nan = __int_as_float(0x7fc00000);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r0 = wm * 16 * MT + 16 * m;
        if (r0 >= rt.count) break;  // (the same for the wave)
        const bool bad = p.row_ids && row_off[r0 + l16] == (unsigned)kOutside;
#pragma unroll
        for (int n = 0; n < NT; ++n)
            *reinterpret_cast<f32x4 *>(out + l16 * kPitch + 16 * n + 4 * quad) =
                bad ? f32x4{nan, nan, nan, nan} : acc[n][m];
        constexpr int kEach = BF16 ? 8 : 4, kLanes = 16 * NT / kEach;  // outputs of a lane, lanes of a row
#pragma unroll
        for (int i = lane; i < 16 * kLanes; i += kWave) {
            const int r = i / kLanes, c = i % kLanes * kEach;
            if (r0 + r < rt.count) store_row<BF16, kEach>(p, rt.first + r0 + r, o_wave + c, out + r * kPitch + c);
        }
    }
}

constexpr long kMaxGrid = 0x7FFFFF;  // workgroups of at most 512 threads in a launch

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

template <class Sh, bool FAST, bool BF16>
int launch_tile(const Fp8Matmul &p, hipStream_t stream) {
    static const bool attr = [] {
        return hipFuncSetAttribute(reinterpret_cast<const void *>(&fp8_tile_kernel<Sh, FAST, BF16>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, Sh::kLds) == hipSuccess;
    }();
    (void)attr;
    const long o_tiles = ((long)p.O + Sh::BO - 1) / Sh::BO, slots = row_tiles<Sh::BM>(p);
    const long tiles = o_tiles * slots;
    if (tiles > kMaxGrid - 8) return kErrSize;
    if (tiles == 0) return kOk;
    hipLaunchKernelGGL((fp8_tile_kernel<Sh, FAST, BF16>), dim3((unsigned)((tiles + 7) / 8 * 8)),
                       dim3(Sh::kThreads), Sh::kLds, stream, p, (int)o_tiles, (int)slots);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

// The tiles copy 16-byte chunks and reach a tile's rows, and gathered rows from
// the first one, by 32-bit offsets.
bool tiles_take(const Fp8Matmul &p) {
    const long blocks = fp8_blocks(p.I);
    return p.I % 16 == 0 && ((uintptr_t)p.w & 15) == 0 && ((uintptr_t)p.x & 15) == 0 && p.I <= (1 << 22) &&
           (!p.row_ids || ((long)p.x_rows * p.I < kOutside && (long)p.x_rows * blocks * 4 < kOutside));
}

}  // namespace

int fp8_matmul(const Fp8Matmul &p, hipStream_t stream) {
    if (p.rows == 0) return kOk;
    const long per_group = p.groups ? (p.rows + p.groups - 1) / p.groups : p.rows;
    if (tiles_take(p) && per_group > 32) {
        static const int force = getenv("FP8_SHAPE") ? atoi(getenv("FP8_SHAPE")) : 0;
        if (p.bf16) {
            if (force == 1) return launch_tile<TileShape<256, 256, 2, 4, 2>, true, true>(p, stream);
            if (force == 2) return launch_tile<TileShape<256, 128, 4, 2, 3>, true, true>(p, stream);
            if (force == 3) return launch_tile<TileShape<128, 128, 2, 2, 2>, true, true>(p, stream);
            if (force == 4) return launch_tile<TileShape<128, 64, 4, 1, 3>, true, true>(p, stream);
        } else {
            if (force == 1) return launch_tile<TileShape<256, 128, 4, 2, 3>, false, false>(p, stream);
            if (force == 2) return launch_tile<TileShape<128, 256, 2, 4, 2>, false, false>(p, stream);
            if (force == 3) return launch_tile<TileShape<128, 128, 2, 2, 2>, false, false>(p, stream);
            if (force == 4) return launch_tile<TileShape<128, 64, 4, 1, 3>, false, false>(p, stream);
        }
    }
    if (per_group <= 16) return launch_direct<DirectShape<1, 1, 1, 1, 4>>(p, stream);
    return launch_direct<DirectShape<2, 2, 2, 2, 1>>(p, stream);
}

}  // namespace mlh
