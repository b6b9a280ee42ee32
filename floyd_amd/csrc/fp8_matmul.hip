// fp8_matmul.hip -- fp8 rows times fp8 matrices, one matrix or one per group of
// rows (gfx950, wave64).
//
//   y[r, o] = sum over blocks b of xs[r, b] ws[o / 128, b] (sum over i in b of x[r, i] w[o, i])
//
// Codes are widened to bf16, which holds every e4m3 value, and multiplied on
// v_mfma_f32_16x16x32_bf16: the products are exact in f32 and a block's 128 are
// added in f32.  Tiles of many rows with bf16 outputs multiply the codes as they are,
// with sums of fewer bits (multiply_fp8).  Each block's sum is then scaled and added in f32.
//
// Weights are the A operand and rows the B operand: lane l supplies matrix row
// and token l % 16, and of a block of 128 columns the 16-byte chunks l / 16 and
// 4 + l / 16 (which of the lane's values meet in one instruction does not
// matter, as long as both operands agree).  Register r of lane l of a result
// is output column 4 (l / 16) + r of token l % 16, so that a lane scales with
// one factor and holds 4 neighbouring outputs.
//
// Operands pass through LDS: the lanes of an operand read hold 16 different rows,
// whose 16-byte pieces the memory pipe takes one a clock (a 1 KB load in 64 clocks),
// while 8 neighbouring lanes on a row's 128 bytes are taken 64 bytes a clock.
#include "fp8.h"
#include "mlh_device.h"
#include "mlh_host.h"

#include <math.h>

namespace mlh {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x4_word __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bf16x8 widen8(unsigned lo, unsigned hi) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The 128 products of a block for 16 x 16 outputs, added, on codes as they are.
// The instruction cuts 8 neighbouring columns' products below 2^-13 of the largest's
// power of two, adds them, and these sums in f32: off by at most 2^-10 of the sum of the
// eights' largest products.  So it makes bf16 outputs of tiles only, at twice the rate of
// widened codes: 4096 x 22528 x 2048 203 us, widened 352.  On rows with 0.4 % loud columns
// (x 31) an output is off by up to 3.5e-4 of the outputs' root mean square (f32 sums:
// 1.2e-6), a sixth of its half place at that size; 1.4 % of the outputs, small ones left
// where loud products cancel, are off by more than their own rounding, the worst by all
// their bits.
__device__ __forceinline__ f32x4 multiply_fp8(const u32x4 (&w)[2], const u32x4 (&x)[2]) {
    const i32x8 a = {(int)w[0][0], (int)w[0][1], (int)w[0][2], (int)w[0][3],
                     (int)w[1][0], (int)w[1][1], (int)w[1][2], (int)w[1][3]};
    const i32x8 b = {(int)x[0][0], (int)x[0][1], (int)x[0][2], (int)x[0][3],
                     (int)x[1][0], (int)x[1][1], (int)x[1][2], (int)x[1][3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
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

// Rows at any byte, read by words (333 x 1001 x 1999 f32 11.2 us, by loads of 16 bytes at
// any byte 12.6): 8 neighbouring lanes hold 128 bytes of a row from its first word on, 16
// each; a lane's last bytes are in the next lane's first word, and the 8th loads them.  No
// word is read that holds none of the row's bytes.
__device__ __forceinline__ const uint8_t *word_of(const uint8_t *p) {
    return reinterpret_cast<const uint8_t *>((uintptr_t)p & ~(uintptr_t)3);
}
// 16 bytes of a lane that start `start` < 4 bytes into the words v
__device__ __forceinline__ u32x4 shift_in(const u32x4 &v, unsigned end, unsigned start, bool last) {
    // lane + 1's first word (row_shl:1)
    const unsigned next = (unsigned)__builtin_amdgcn_update_dpp((int)end, (int)v[0], 0x101, 0xF, 0xF, false);
    const unsigned e = last ? end : next;
    return u32x4{__builtin_amdgcn_alignbyte(v[1], v[0], start), __builtin_amdgcn_alignbyte(v[2], v[1], start),
                 __builtin_amdgcn_alignbyte(v[3], v[2], start), __builtin_amdgcn_alignbyte(e, v[3], start)};
}

// columns c .. c + 15 of a row of `width` codes, zeros past its end; nothing
// outside the row is read
__device__ __forceinline__ u32x4 load16_tail(const uint8_t *row, int c, int width) {
    u32x4 v = {0, 0, 0, 0};
    if (c + 16 <= width) return load16_any(row + c);
    if (c >= width) return v;
    if (width >= 16) {  // the row's last 16, moved down
        const u32x4 u = load16_any(row + width - 16);
        const unsigned long long lo = u[0] | (unsigned long long)u[1] << 32;
        const unsigned long long hi = u[2] | (unsigned long long)u[3] << 32;
        const int bits = 8 * (c + 16 - width);  // 8 .. 120
        const unsigned long long l =
            bits >= 64 ? hi >> (bits - 64) : lo >> bits | hi << (64 - bits);
        const unsigned long long h = bits >= 64 ? 0 : hi >> bits;
        v[0] = (unsigned)l;
        v[1] = (unsigned)(l >> 32);
        v[2] = (unsigned)h;
        v[3] = (unsigned)(h >> 32);
        return v;
    }
    unsigned long long l = 0, h = 0;
#pragma unroll 1
    for (int i = 0; c + i < width; ++i) {
        if (i < 8) l |= (unsigned long long)row[c + i] << (8 * i);
        else h |= (unsigned long long)row[c + i] << (8 * (i - 8));
    }
    v[0] = (unsigned)l;
    v[1] = (unsigned)(l >> 32);
    v[2] = (unsigned)h;
    v[3] = (unsigned)(h >> 32);
    return v;
}

// The rows of one workgroup's tile: `count` rows from `first` on (entries of y)
// of group `group`; count 0: none.
struct RowTile {
    int group, first, count;
};

// Rows of the groups g0 + 64 j + lane, j < N (a group past the last one is empty), all
// loads in flight together: 4096 tokens on 160 experts, 2048 x 1408, 203 us one after the
// other, 197 by fours; the streams, 64 experts or fewer as often, take two.  Offsets that
// decrease or leave [0, rows] are read as empty or shortened groups.
constexpr int kTileLoads = 4, kStreamLoads = 2;
template <int N>
__device__ __forceinline__ void group_rows(const Fp8Matmul &p, int g0, int (&start)[N], int (&count)[N]) {
    int from[N], to[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int g = min(g0 + j * kWave + (int)(threadIdx.x & (kWave - 1)), p.groups - 1);
        from[j] = p.offsets[g];
        to[j] = p.offsets[g + 1];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const bool in = g0 + j * kWave + (int)(threadIdx.x & (kWave - 1)) < p.groups;
        start[j] = min(max(from[j], 0), p.rows);
        count[j] = in ? max(min(to[j], p.rows), start[j]) - start[j] : 0;
    }
}

// Row tile `slot` of a launch: the groups' tiles one after the other, a wave's
// lanes counting 64 groups at a time.
template <int BM, int N> __device__ __forceinline__ RowTile row_tile(const Fp8Matmul &p, int slot) {
    if (p.groups == 0) {
        const int first = slot * BM;
        return RowTile{0, first, min(BM, p.rows - first)};
    }
    const int lane = threadIdx.x & (kWave - 1);
    int before = 0;
    for (int g0 = 0; g0 < p.groups; g0 += N * kWave) {
        int start[N], count[N];
        group_rows(p, g0, start, count);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (g0 + j * kWave >= p.groups) break;
            const int tiles = (count[j] + BM - 1) / BM;
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
                const int s = __builtin_amdgcn_readlane(start[j], src);
                const int c = __builtin_amdgcn_readlane(count[j], src);
                return RowTile{g0 + j * kWave + src, s + t * BM, min(BM, c - t * BM)};
            }
            before += __builtin_amdgcn_readlane(incl, kWave - 1);
        }
    }
    return RowTile{0, 0, 0};
}

// Row tiles that `rows` entries in `groups` groups can need.
long row_tiles(const Fp8Matmul &p, int bm) {
    if (p.groups == 0) return ((long)p.rows + bm - 1) / bm;
    const long used = p.groups < p.rows ? p.groups : p.rows;  // groups that can hold a row
    return (p.rows + used * (bm - 1)) / bm;
}

// Four neighbouring outputs of a row; those from O on are left out.
template <bool BF16>
__device__ __forceinline__ void store4(const Fp8Matmul &p, long row, int o, f32x4 v) {
    const long at = row * p.O + o;
    if (o + 4 <= p.O) {  // (at any address)
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
    if (o + EACH <= p.O) {  // (at any address)
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
        // past the L2: results of many rows would push the operands out of it (4096 x
        // 22528 x 2048 bf16 197 us, stored through it 219)
        __builtin_nontemporal_store(u, reinterpret_cast<u32x4_any *>(static_cast<uint8_t *>(p.y) + byte));
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

// ---------------------------------------------------------------------------
// Tiles through LDS, for many rows
// ---------------------------------------------------------------------------
//
// A workgroup of WO x WM waves makes BO matrix rows x BM tokens; a wave NT x MT
// results of 16 x 16.  Each step of 128 columns is copied by DMA into one of two LDS
// stages while the step before it is multiplied: rows of 128 bytes as they lie in
// memory, 16-byte chunk c of row r at chunk c ^ (r / 2 & 7), so that the rows an
// operand read touches lie on different banks; the row and matrix scales behind
// them, copied in pieces of kSpan steps: a scale a token and step is 4 bytes of its
// own cache line, and copying each step's alone asked the L2 for as many lines as
// the operands.
//
// 256 x 256 (bf16 outputs, 146 KB of LDS) asks the L2 for least: 4096 x 22528 x 2048
// 199 us, 1900 TFLOP/s, on 128 x 128 237.  A tile there takes 2 us to its first copies,
// 3 to the first step, 1.7 a step (1.1 of it matrix instructions), and 5 for its
// results, which all CUs store at once.  f32 outputs, 128 x 128: 366 us, 1030 TFLOP/s,
// bound by the widening beside the matrix instructions.
constexpr int kSpan = 8;
template <int BO_, int BM_, int WO_, int WM_> struct TileShape {
    static constexpr int BO = BO_, BM = BM_, WO = WO_, WM = WM_;
    static constexpr int kWaves = WO * WM, kThreads = kWaves * kWave;
    static constexpr int NT = BO / 16 / WO, MT = BM / 16 / WM;
    static constexpr int kStage = (BO + BM) * kFp8Block;
    // scales: two groups of kSpan steps, each BM / 8 pieces of 8 tokens by kSpan steps and
    // one of matrix blocks
    static constexpr int kPieces = BM / 8 + 1, kMatrixBlocks = (BO + kFp8Block - 1) / kFp8Block;
    static constexpr int kScales = 2 * kStage, kScaleGroup = kPieces * 256;
    // offsets of the rows' scales: BM tokens, 8 matrix blocks
    static constexpr int kRowOffsets = kScales + 2 * kScaleGroup;
    static constexpr int kLds = kRowOffsets + (BM + 8) * 4;
    // the waves that copy: with two on a SIMD one of them
    static constexpr int kCopiers = kWaves == 8 ? 4 : kWaves;
    static constexpr int kWPer = BO / 8 / kCopiers, kXPer = BM / 8 / kCopiers;  // DMA blocks of one
    static constexpr int kDma = kWPer + kXPer;
    static_assert(BO % (8 * kCopiers) == 0 && BM % (8 * kCopiers) == 0, "whole DMA blocks");
    static_assert((kPieces - 1 + kCopiers - 1) / kCopiers <= kSpan && kMatrixBlocks <= 8 &&
                      (BO % kFp8Block == 0 || kFp8Block % BO == 0),
                  "a group's scales land before its first step");
    static_assert(BO / 16 % WO == 0 && BM / 16 % WM == 0 && kFp8Block % (16 * NT) == 0,
                  "a wave's matrix rows lie in one block");
    static_assert(kLds <= 160 * 1024, "LDS");
};

template <int N> __device__ __forceinline__ void wait_vmcnt() {
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

constexpr long kOutside = kFp8Outside;

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
    int n = 0;
    for (int g0 = 0; g0 < p.groups; g0 += kTileLoads * kWave) {
        int start[kTileLoads], count[kTileLoads];
        group_rows(p, g0, start, count);
#pragma unroll
        for (int j = 0; j < kTileLoads; ++j) n += (count[j] + BM - 1) / BM;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o, kWave);
    return __builtin_amdgcn_readfirstlane(n);
}

constexpr int kTileGroup = 4;  // row tiles that share matrix rows, one after the other

template <class Sh, bool FAST, bool BF16, bool DMA>
__global__ __launch_bounds__(Sh::kThreads, 2) void fp8_tile_kernel(Fp8Matmul p, int o_tiles, int slots) {
    constexpr int NT = Sh::NT, MT = Sh::MT, BO = Sh::BO, BM = Sh::BM;
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
    RowTile rt = row_tile<BM, kTileLoads>(p, slot);
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
    unsigned x_off[Sh::kXPer];  // byte offsets; without DMA the rows (0 where there is none)
#pragma unroll
    for (int q = 0; q < Sh::kXPer; ++q) {
        const int r = x_row((wave % Sh::kCopiers + Sh::kCopiers * q) * 8 + dma_row);
        if constexpr (DMA) x_off[q] = r < 0 ? (unsigned)kOutside : (unsigned)r * (unsigned)p.I;
        else x_off[q] = max(r, 0);
    }
    const unsigned w_off = (unsigned)(wave * 8 + dma_row) * (unsigned)p.I;
    // A piece of scales: lane l takes step l / 8 of the group and token (or matrix
    // block) l % 8; piece j of a group is copied by wave j % kWaves.
    const long xs_bytes = x_count * blocks * 4, ws_bytes = (long)(o_blocks - o0 / kFp8Block) * blocks * 4;
    const int sc_lane = lane & 7, sc_step = lane >> 3;
    unsigned *const row_off = reinterpret_cast<unsigned *>(lds + Sh::kRowOffsets);
    for (int i = threadIdx.x; i < BM + 8; i += Sh::kThreads) {
        const int r = i < BM ? x_row(i) : i - BM < Sh::kMatrixBlocks ? i - BM : -1;
        row_off[i] = r < 0 ? (unsigned)kOutside : (unsigned)r * (unsigned)blocks * 4u;
    }
    __syncthreads();
    auto copy_scales = [&](int g, int piece) {
        const unsigned row = row_off[piece * 8 + sc_lane];
        const bool rows = piece < BM / 8;
        const bool in = g * kSpan + sc_step < blocks && row != (unsigned)kOutside;
        dma4(buffer_of(rows ? xs_base : ws_base, rows ? xs_bytes : ws_bytes),
             in ? row + sc_step * 4u : (unsigned)kOutside, fp8_scalar_offset(g * kSpan, blocks, 4),
             (LdsByte *)(lds + Sh::kScales + (g & 1) * Sh::kScaleGroup + piece * 256));
    };
    // a step's part of the next group's scales
    auto copy_next_scales = [&](int b) {
        const int g = b / kSpan + 1, piece = b % kSpan * Sh::kCopiers + wave;
        if (piece < Sh::kPieces) copy_scales(g, piece);
        // (one piece more than the steps have copies)
        if (Sh::kPieces > kSpan * Sh::kCopiers && b % kSpan == 0 && wave == 0) copy_scales(g, Sh::kPieces - 1);
    };
    // the operands of step b
    auto copy_tiles = [&](int b, int st) {
        LdsByte *stage = (LdsByte *)(lds + st * Sh::kStage);
        const int k0 = b * kFp8Block;
#pragma unroll
        for (int i = 0; i < Sh::kDma; ++i) {
            const int q = i < Sh::kWPer ? i : i - Sh::kWPer;
            const int blk = wave + Sh::kCopiers * q;
            const int chunk = (lane & 7) ^ ((blk & 1) * 4 + dma_row / 2);
            // a row that ends inside the step: zeros past its end
            const bool past = k0 + kFp8Block > p.I && k0 + chunk * 16 >= p.I;
            if (i < Sh::kWPer)
                dma16(buffer_of(w_base, w_bytes),
                      past ? (unsigned)kOutside
                           : w_off + (unsigned)(q * Sh::kCopiers * 8) * (unsigned)p.I + (unsigned)(chunk * 16),
                      k0, stage + blk * 1024);
            else
                dma16(buffer_of(x_base, x_bytes),
                      past || x_off[q] == (unsigned)kOutside ? (unsigned)kOutside
                                                             : x_off[q] + (unsigned)(chunk * 16),
                      k0, stage + BO * kFp8Block + blk * 1024);
        }
    };
    // The same through registers, for rows at any address: loaded before a step's
    // products, stored after them.
    u32x4 held[DMA ? 1 : Sh::kDma];
    auto load_tiles = [&](int b) {
        const int k0 = b * kFp8Block;
#pragma unroll
        for (int i = 0; i < Sh::kDma; ++i) {
            const int q = i < Sh::kWPer ? i : i - Sh::kWPer;
            const int blk = wave + Sh::kCopiers * q;
            const int c = k0 + ((lane & 7) ^ ((blk & 1) * 4 + dma_row / 2)) * 16;
            const uint8_t *row = i < Sh::kWPer ? w_base + (long)min(blk * 8 + dma_row, p.O - 1 - o0) * p.I
                                               : x_base + (long)x_off[q] * p.I;
            if (k0 + kFp8Block <= p.I) held[i] = load16_any(row + c);
            else held[i] = load16_tail(row, c, p.I);
        }
    };
    auto store_tiles = [&](int st) {
#pragma unroll
        for (int i = 0; i < Sh::kDma; ++i) {
            const int q = i < Sh::kWPer ? i : i - Sh::kWPer;
            *reinterpret_cast<u32x4 *>(lds + st * Sh::kStage + (i < Sh::kWPer ? 0 : BO * kFp8Block) +
                                       (wave + Sh::kCopiers * q) * 1024 + lane * 16) = held[i];
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
                        d[n & 1][m] = multiply_fp8(wf[n & 1], xf[m]);
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
    for (int piece = wave; piece < Sh::kPieces; piece += kWaves) copy_scales(0, piece);
    // Eight waves: the first four, one on each SIMD, hand the copies to the memory pipe,
    // which holds them up until it has taken them, while the other four multiply.
    const bool copier = wave < Sh::kCopiers;
    if (copier) {
        if constexpr (DMA) {
            copy_tiles(0, 0);
        } else {
            load_tiles(0);
            store_tiles(0);
        }
    }
    for (int b = 0; b < blocks; ++b) {
        const int st = b & 1;
        // The wait lands this wave's part of the step; the barrier makes every wave's
        // visible and frees the stage read last.
        if constexpr (DMA) wait_vmcnt<0>();
        else __builtin_amdgcn_s_waitcnt(0);  // (the stores to LDS)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const bool more = copier && b + 1 < blocks;
        if (more) {
            if constexpr (DMA) copy_tiles(b + 1, st ^ 1);
            else load_tiles(b + 1);
            copy_next_scales(b);
        }
        if (live) multiply(b, st);
        if constexpr (!DMA) {
            if (more) store_tiles(st ^ 1);
        }
    }

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

// ---------------------------------------------------------------------------
// Few rows: the matrix as a stream
// ---------------------------------------------------------------------------
//
// A workgroup's WK waves share 16 NT matrix rows and up to 8 XB tokens; wave k
// takes the blocks of columns k, k + WK, ... and copies both operands by DMA into a
// ring of its own, STAGES blocks ahead, so that no wave waits for another until the
// shares are added through LDS.  Rows of 128 bytes with the tiles' swizzle.
// Without DMA, for rows at any address: through registers, as far ahead, into one
// stage a wave.  BYTES: some row does not start at a word; then the pieces are read by
// words and moved into place, as a load of 16 bytes at any byte takes longer.
//
// Bound by the matrix where it is read once: 22528 x 2048, 1 row, 9.4 us, 4.9 TB/s; the
// 27 of 64 experts that 8 tokens reach, 2816 x 2048, 34 us, 4.6 TB/s.  With more rows
// each strip of 8 or 16 reads it from the L2 again, two steps a wave in flight: 2048 x
// 11264, 61 rows, 11.4 us.
template <int NT_, int XB_, int WK_, int STAGES_, bool DMA_ = true> struct StreamShape {
    static constexpr int NT = NT_, XB = XB_, MT = (XB + 1) / 2, WK = WK_, kStages = STAGES_;
    static constexpr bool DMA = DMA_;
    static constexpr int kThreads = WK * kWave, BO = 16 * NT, BM = 8 * XB;
    static constexpr int kStage = 2 * NT * 1024 + 2 * MT * 1024;
    static constexpr int kLoads = 2 * NT + XB + MT + 1;  // a step's, scales among them
    static constexpr int kRing = (DMA ? kStages : 1) * kStage;
    static constexpr int kRed = (WK - 1) * NT * MT * 1024;
    static constexpr int kLds = WK * kRing > kRed ? WK * kRing : kRed;
    static_assert(kLds <= 160 * 1024 && kStages * kLoads < 64, "LDS, vmcnt");
    static_assert(kFp8Block % (16 * NT) == 0, "the matrix rows lie in one block");
};

template <class Sh, bool BF16, bool BYTES>
__global__ __launch_bounds__(Sh::kThreads) void fp8_stream_kernel(Fp8Matmul p, int o_tiles) {
    constexpr int NT = Sh::NT, MT = Sh::MT, XB = Sh::XB, WK = Sh::WK, S = Sh::kStages;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int slot = blockIdx.x / o_tiles;
    RowTile rt = row_tile<Sh::BM, kStreamLoads>(p, slot);
    if (rt.count <= 0) return;
    rt.group = __builtin_amdgcn_readfirstlane(rt.group);
    rt.first = __builtin_amdgcn_readfirstlane(rt.first);
    rt.count = __builtin_amdgcn_readfirstlane(rt.count);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l16 = lane & 15, quad = lane >> 4, dma_row = lane >> 3;
    const int o0 = (blockIdx.x - slot * o_tiles) * Sh::BO;
    const int blocks = (p.I - 1) / kFp8Block + 1;
    const int o_blocks = (p.O - 1) / kFp8Block + 1;
    const uint8_t *const w_base = p.w + ((long)rt.group * p.O + o0) * p.I;
    const float *const ws_base = p.ws + ((long)rt.group * o_blocks + o0 / kFp8Block) * blocks;
    const long x_first = p.row_ids ? 0 : rt.first, x_count = p.row_ids ? p.x_rows : rt.count;
    const uint8_t *const x_base = p.x + x_first * p.I;
    const float *const xs_base = p.xs + x_first * blocks;
    const long w_bytes = (long)(p.O - o0) * p.I, x_bytes = x_count * p.I;
    const long xs_bytes = x_count * blocks * 4, ws_bytes = (long)blocks * 4;
    // buffer row of token m (the last one's for those past the end, row 0 for an id
    // out of range: neither is stored as it is)
    auto x_row = [&](int m, bool *bad = nullptr) -> unsigned {
        m = min(m, rt.count - 1);
        if (!p.row_ids) return m;
        const int r = p.row_ids[rt.first + m];
        const bool out = r < 0 || r >= p.x_rows;
        if (bad) *bad = out;
        return out ? 0 : r;
    };
    unsigned x_off[XB], xs_off[MT];  // bytes; x_off without DMA: rows
    bool bad[MT];
#pragma unroll
    for (int q = 0; q < XB; ++q) x_off[q] = x_row(q * 8 + dma_row) * (Sh::DMA ? (unsigned)p.I : 1u);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        bad[m] = false;
        xs_off[m] = x_row(16 * m + l16, &bad[m]) * (unsigned)blocks * 4u;
    }
    const unsigned w_off = (unsigned)dma_row * (unsigned)p.I;
    uint8_t *const ring = lds + wave * Sh::kRing;
    float xs[S][MT], ws[S];
    constexpr int kPer = 2 * NT + XB;
    u32x4 held[Sh::DMA ? 1 : S][kPer];
    unsigned end[BYTES ? S : 1][kPer];
    auto row_of = [&](int q) -> const uint8_t * {
        return q < 2 * NT ? w_base + (long)min(q * 8 + dma_row, p.O - 1 - o0) * p.I
                          : x_base + (long)x_off[q - 2 * NT] * p.I;
    };
    // chunk of row q where this lane's 16 bytes lie in LDS, or come from
    auto chunk_of = [&](int q) {
        return (lane & 7) ^ (((q < 2 * NT ? q : q - 2 * NT) & 1) * 4 + dma_row / 2);
    };
    unsigned starts = 0;  // of the rows in their words, 2 bits a piece
    if constexpr (BYTES) {
        static_assert(kPer <= 16, "starts");
#pragma unroll
        for (int q = 0; q < kPer; ++q) starts |= ((unsigned)(uintptr_t)row_of(q) & 3) << (2 * q);
    }
    auto copy_scales = [&](int b, int st) {
        const int at = fp8_scalar_offset(b, blocks, 4);
#pragma unroll
        for (int m = 0; m < MT; ++m)
            xs[st][m] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
                buffer_of(xs_base, xs_bytes), b < blocks ? xs_off[m] : (unsigned)kOutside, at, 0));
        ws[st] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            buffer_of(ws_base, ws_bytes), b < blocks ? 0u : (unsigned)kOutside, at, 0));
    };
    auto load = [&](int b, int st) {
        if (b >= blocks) return;
        const int k0 = b * kFp8Block;
        if (k0 + kFp8Block <= p.I) {
#pragma unroll
            for (int q = 0; q < kPer; ++q) {
                const uint8_t *from = row_of(q) + k0 + (BYTES ? lane & 7 : chunk_of(q)) * 16;
                if constexpr (BYTES) held[st][q] = *reinterpret_cast<const u32x4_word *>(word_of(from));
                else held[st][q] = load16_any(from);
            }
            if constexpr (BYTES) {
                if ((lane & 7) == 7) {
#pragma unroll
                    for (int q = 0; q < kPer; ++q)
                        end[st][q] = *reinterpret_cast<const unsigned *>(word_of(row_of(q) + k0 + kFp8Block - 1));
                }
            }
        } else {
#pragma unroll
            for (int q = 0; q < kPer; ++q)
                held[st][q] = load16_tail(row_of(q), k0 + (BYTES ? lane & 7 : chunk_of(q)) * 16, p.I);
        }
        copy_scales(b, st);
    };
    auto store = [&](int b, int st) {
        const bool shift = BYTES && b * kFp8Block + kFp8Block <= p.I;
#pragma unroll
        for (int q = 0; q < kPer; ++q)
            *reinterpret_cast<u32x4 *>(ring + q * 1024 + dma_row * kFp8Block + (BYTES ? chunk_of(q) : lane & 7) * 16) =
                shift ? shift_in(held[st][q], end[st][q], starts >> (2 * q) & 3, (lane & 7) == 7) : held[st][q];
    };
    auto copy = [&](int b, int st) {
        LdsByte *stage = (LdsByte *)(ring + st * Sh::kStage);
        const int k0 = b * kFp8Block, at = fp8_scalar_offset(b, blocks, kFp8Block);
#pragma unroll
        for (int q = 0; q < 2 * NT; ++q) {
            const int chunk = (lane & 7) ^ ((q & 1) * 4 + dma_row / 2);
            const bool past = k0 + chunk * 16 >= p.I;  // (of a block past the last, all)
            dma16(buffer_of(w_base, w_bytes),
                  past ? (unsigned)kOutside : w_off + (unsigned)(q * 8) * (unsigned)p.I + (unsigned)(chunk * 16),
                  at, stage + q * 1024);
        }
#pragma unroll
        for (int q = 0; q < XB; ++q) {
            const int chunk = (lane & 7) ^ ((q & 1) * 4 + dma_row / 2);
            const bool past = k0 + chunk * 16 >= p.I;
            dma16(buffer_of(x_base, x_bytes), past ? (unsigned)kOutside : x_off[q] + (unsigned)(chunk * 16), at,
                  stage + (2 * NT + q) * 1024);
        }
        copy_scales(b, st);
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[n][m] = f32x4{0, 0, 0, 0};
    const int frag0 = l16 * kFp8Block + ((quad ^ (l16 >> 1)) << 4);
    const int frag1 = l16 * kFp8Block + (((quad + 4) ^ (l16 >> 1)) << 4);
    u32x4 wf[NT][2], xf[MT][2];
    auto read = [&](int st) {
        const uint8_t *stage = ring + st * Sh::kStage;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            wf[n][0] = *reinterpret_cast<const u32x4 *>(stage + n * 2048 + frag0);
            wf[n][1] = *reinterpret_cast<const u32x4 *>(stage + n * 2048 + frag1);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            xf[m][0] = *reinterpret_cast<const u32x4 *>(stage + (NT + m) * 2048 + frag0);
            xf[m][1] = *reinterpret_cast<const u32x4 *>(stage + (NT + m) * 2048 + frag1);
        }
    };
    auto multiply = [&](int st) {
        f32x4 d[NT][MT];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int h = q / 2, e = 2 * (q % 2);
            bf16x8 x[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) x[m] = widen8(xf[m][h][e], xf[m][h][e + 1]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const bf16x8 w = widen8(wf[n][h][e], wf[n][h][e + 1]);
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
                const float f = ws[st] * xs[st][m];
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(d[n][m][i], f, acc[n][m][i]);
            }
    };
    const int steps = (blocks - wave + WK - 1) / WK;  // (0 or less: none)
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if constexpr (Sh::DMA) copy(wave + s * WK, s);
        else load(wave + s * WK, s);
    }
    for (int t = 0; t < steps; t += S) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (t + s >= steps) break;
            if constexpr (!Sh::DMA) {  // a wave's LDS accesses are done in their order
                store(wave + (t + s) * WK, s);
                read(0);
                multiply(s);
                load(wave + (t + s + S) * WK, s);
                continue;
            }
            wait_vmcnt<(S - 1) * Sh::kLoads>();
            asm volatile("" ::: "memory");
            read(s);
            // (the reads are done before the stage is filled again)
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt 0
            asm volatile("" ::: "memory");
            multiply(s);
            copy(wave + (t + s + S) * WK, s);
        }
    }
    if constexpr (Sh::DMA) wait_vmcnt<0>();
    if constexpr (WK > 1) {
        __syncthreads();  // the rings become the place of the shares
        f32x4 *red = reinterpret_cast<f32x4 *>(lds);
        if (wave > 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) red[(((wave - 1) * NT + n) * MT + m) * kWave + lane] = acc[n][m];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int k = 0; k < WK - 1; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[n][m] += red[((k * NT + n) * MT + m) * kWave + lane];
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = 16 * m + l16;
        if (r >= rt.count) continue;
        const float nan = __int_as_float(0x7fc00000);
#pragma unroll
        for (int n = 0; n < NT; ++n)
            store4<BF16>(p, rt.first + r, o0 + 16 * n + 4 * quad, bad[m] ? f32x4{nan, nan, nan, nan} : acc[n][m]);
    }
}

template <class Sh, bool FAST, bool BF16, bool DMA = true>
int launch_tile(const Fp8Matmul &p, hipStream_t stream) {
    static const bool attr = [] {
        return hipFuncSetAttribute(reinterpret_cast<const void *>(&fp8_tile_kernel<Sh, FAST, BF16, DMA>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, Sh::kLds) == hipSuccess;
    }();
    (void)attr;
    const long o_tiles = ((long)p.O + Sh::BO - 1) / Sh::BO, slots = row_tiles(p, Sh::BM);
    const long tiles = o_tiles * slots;
    hipLaunchKernelGGL((fp8_tile_kernel<Sh, FAST, BF16, DMA>), dim3((unsigned)((tiles + 7) / 8 * 8)),
                       dim3(Sh::kThreads), Sh::kLds, stream, p, (int)o_tiles, (int)slots);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

template <class Sh, bool BF16, bool BYTES> int launch_stream_of(const Fp8Matmul &p, hipStream_t stream) {
    static const bool attr = [] {
        return hipFuncSetAttribute(reinterpret_cast<const void *>(&fp8_stream_kernel<Sh, BF16, BYTES>),
                                   hipFuncAttributeMaxDynamicSharedMemorySize, Sh::kLds) == hipSuccess;
    }();
    (void)attr;
    const long o_tiles = ((long)p.O + Sh::BO - 1) / Sh::BO;
    const long tiles = row_tiles(p, Sh::BM) * o_tiles;
    hipLaunchKernelGGL((fp8_stream_kernel<Sh, BF16, BYTES>), dim3((unsigned)tiles), dim3(Sh::kThreads), Sh::kLds,
                       stream, p, (int)o_tiles);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

template <class Sh, bool BF16> int launch_stream(const Fp8Matmul &p, hipStream_t stream) {
    if constexpr (!Sh::DMA)
        if (((uintptr_t)p.w | (uintptr_t)p.x | (unsigned)p.I) & 3) return launch_stream_of<Sh, BF16, true>(p, stream);
    return launch_stream_of<Sh, BF16, false>(p, stream);
}

// DMA takes 16-byte chunks, and a tile's rows by 32-bit offsets.
bool dma_takes(const Fp8Matmul &p) {
    return p.I <= (1 << 22) && p.I % 16 == 0 && ((uintptr_t)p.w & 15) == 0 && ((uintptr_t)p.x & 15) == 0 &&
           (!p.row_ids || (long)p.x_rows * p.I < kOutside);
}

// ---- which kernel: the one that a model of its time says is the fastest.
//
// A workgroup takes `start` us and `step` us for each of its waves' blocks of
// columns where every CU has at most one, `full` us a block where each CU holds
// per_cu of them, and in between for numbers in between; workgroups that follow
// others on their CU start in half the time.  The three numbers of each shape are
// fitted to its times on MI355X over 210 products (out_width 333 .. 22528, in_width
// 777 .. 11264, 1 .. 4096 rows, one matrix, 8 or 64), so that the choice costs
// little: 0.6 % more than the best shape's time on them, and 1.4 % (25 % at worst)
// on 110 others of sizes drawn by chance.  Some of those times (bf16, us; streams by
// matrix rows x tokens, "regs" without DMA):
//   22528 x 2048, 16 rows:   stream 16 x 16 regs 10.5, tile 64 x 64 11.3, stream 32 x 16 14.5
//                 100 rows:  tile 64 x 64 14.5, 128 x 128 18.4
//                 2048 rows: tile 256 x 256 102, 128 x 128 121
//   2048 x 11264, 1 row:     stream 16 x 8 7.1, 32 x 16 8.8
//                 40 rows:   stream 32 x 16 10.8, 16 x 16 regs 16.0, 32 x 32 16.4
//                 100 rows:  stream 32 x 32 16.6, 32 x 16 20.0, 32 x 32 regs 24.7
//                 230 rows:  stream 32 x 32 regs 27.2, 32 x 32 31.9, 64 x 64 33.4
//                 400 rows:  stream 64 x 64 33.5, tile 64 x 64 44.3
//                 1500 rows: tile 64 x 64 59.2, 128 x 128 66.4
struct Variant {
    int bo, bm, waves, per_cu;  // waves: those that share a reduction
    float start, step, full;
    bool dma;
    int (*launch)(const Fp8Matmul &, hipStream_t);
};

template <bool BF16, int BO, int BM, int WO, int WM, bool DMA>
constexpr Variant tile(int per_cu, float start, float step, float full) {
    return Variant{BO, BM, 1, per_cu, start, step, full, DMA,
                   &launch_tile<TileShape<BO, BM, WO, WM>, BF16, BF16, DMA>};
}
template <bool BF16, int NT, int XB, int WK, int STAGES, bool DMA>
constexpr Variant flow(int per_cu, float start, float step, float full) {
    using Sh = StreamShape<NT, XB, WK, STAGES, DMA>;
    return Variant{Sh::BO, Sh::BM, WK, per_cu, start, step, full, DMA, &launch_stream<Sh, BF16>};
}

constexpr Variant kBf16Variants[] = {
    flow<true, 1, 1, 4, 2, false>(4, 4.0f, 0.35f, 0.75f),
    flow<true, 1, 2, 4, 2, false>(4, 4.5f, 0.43f, 0.84f),
    flow<true, 2, 4, 4, 1, false>(2, 5.0f, 0.77f, 1.10f),
    tile<true, 64, 64, 2, 2, false>(4, 5.6f, 0.48f, 1.14f),
    tile<true, 128, 128, 2, 2, false>(2, 10.9f, 0.84f, 1.38f),
    flow<true, 1, 1, 8, 4, true>(1, 3.4f, 0.34f, 0.60f),
    flow<true, 2, 2, 8, 2, true>(1, 4.3f, 0.59f, 0.68f),
    flow<true, 2, 4, 4, 4, true>(1, 4.8f, 0.53f, 0.67f),
    flow<true, 4, 8, 4, 2, true>(1, 7.4f, 1.19f, 1.42f),
    tile<true, 64, 64, 2, 2, true>(4, 3.4f, 0.46f, 0.99f),
    tile<true, 128, 128, 2, 2, true>(2, 4.6f, 0.80f, 1.18f),
    tile<true, 256, 256, 2, 4, true>(1, 10.4f, 1.28f, 2.04f),
};
constexpr Variant kF32Variants[] = {
    flow<false, 1, 1, 4, 2, false>(4, 4.1f, 0.33f, 0.87f),
    flow<false, 1, 2, 4, 2, false>(4, 4.5f, 0.43f, 0.86f),
    flow<false, 2, 4, 4, 1, false>(2, 4.7f, 0.80f, 1.08f),
    tile<false, 64, 64, 2, 2, false>(4, 5.4f, 0.53f, 1.48f),
    tile<false, 128, 128, 2, 2, false>(2, 13.1f, 1.33f, 1.99f),
    flow<false, 1, 1, 8, 4, true>(1, 3.1f, 0.36f, 0.62f),
    flow<false, 2, 2, 8, 2, true>(1, 4.3f, 0.59f, 0.68f),
    flow<false, 2, 4, 4, 4, true>(1, 4.8f, 0.52f, 0.60f),
    flow<false, 4, 8, 4, 2, true>(1, 7.4f, 1.05f, 1.32f),
    tile<false, 64, 64, 2, 2, true>(4, 4.0f, 0.54f, 1.19f),
    tile<false, 128, 128, 2, 2, true>(2, 6.3f, 1.04f, 1.80f),
};

constexpr long kMaxGrid = 0x7FFFF0;  // workgroups of at most 512 threads in a launch

template <int N> int launch_best(const Variant (&variants)[N], const Fp8Matmul &p, hipStream_t stream) {
    constexpr float kCus = 256.0f;
    const bool dma = dma_takes(p);
    const int blocks = fp8_blocks(p.I);
    // the groups that rows spread by chance are expected to reach
    const float used =
        p.groups ? p.groups * (1.0f - powf(1.0f - 1.0f / p.groups, (float)p.rows)) : 0.0f;
    const Variant *best = nullptr;
    float least = 0.0f;
    for (const Variant &v : variants) {
        if (v.dma && !dma) continue;
        if (!fp8_scales_in_reach(v.bm, p.I)) continue;
        if (row_tiles(p, v.bm) * ((p.O - 1) / v.bo + 1) > kMaxGrid) continue;
        float row_tiles = (float)((p.rows - 1) / v.bm + 1);
        if (p.groups) {  // tiles of a group: half of one is spare, but for less than one
            const float each = (float)p.rows / (used * v.bm);
            row_tiles = used * fmaxf(1.0f, each > 1.0f ? each + 0.5f : 2.0f * each - 0.5f);
        }
        const float share = row_tiles * (float)((p.O - 1) / v.bo + 1) / kCus, fill = share / v.per_cu;
        const float rounds = 0.5f * (fill + ceilf(fill));
        const float step = share <= 1.0f  ? v.step
                           : fill <= 1.0f ? v.step + (v.full - v.step) * (share - 1.0f) / (v.per_cu - 1)
                                          : v.full * rounds;
        const float cost = v.start * (0.5f + 0.5f * fmaxf(1.0f, rounds)) +
                           (float)((blocks - 1) / v.waves + 1) * step;
        if (!best || cost < least) {
            best = &v;
            least = cost;
        }
    }
    return best ? best->launch(p, stream) : kErrSize;
}

}  // namespace

int fp8_matmul(const Fp8Matmul &p, hipStream_t stream) {
    if (p.rows == 0) return kOk;
    if (p.row_ids && !fp8_scales_in_reach(p.x_rows, p.I)) return kErrSize;
    return p.bf16 ? launch_best(kBf16Variants, p, stream) : launch_best(kF32Variants, p, stream);
}

}  // namespace mlh
