// latent_wide.hip -- attention over the latent cache for sequences with many (row, head)
// pairs, such as prompts in chunks (gfx950, wave64; bf16 queries, full rows).
//
// A tile is 64 pairs (columns) and a step 64 keys, which the four waves bring into LDS as bf16
// rows, once for all columns, while they work on the step before.
//   S[key][column]: wave (x, y) has columns 32 x .. and keys 32 y .., 36 products
//     v_mfma_f32_32x32x16_bf16 on queries that stay in registers.
//   P = exp2(scale S - top) goes through LDS, 8 KB, to all waves.  `top` is the columns' common
//     reference, which moves only when a score passes it by 2^kSlack; then all waves meet again.
//   O[latent][column] += V^T P: wave w has latent values 128 w .. of all columns.  Rows come out
//     of LDS transposed, 4 keys by 16 values at once.  The registers of S hold 4 keys in a row,
//     every 8, of a column, and so the operands of this product have them.
// (With sums split by columns and keys, as the scores are, every wave holds all 512 of 32 columns,
// 256 registers, reads V^T twice as often and moves all of it where the reference moves: 99 us
// where this split took 84.)  P is rounded to bf16, as one operand of the second product: a second
// part would double its matrix instructions and P's way through LDS; the results are 0.00177 of their
// norm off those in 64 bits, of which their own rounding is 0.00166.
//
// Measured, calls over 3000 .. 4096 keys with the join, which is 11 us of the first: four sequences of
// 32, 64, 96 and 128 rows of 16 heads (41 GFLOP, 18.5 steps a workgroup) bf16 keys 79 us, 4-bit ones
// 75; four of 128 rows (62 GFLOP, 28 steps) 103 and 99; one of 256 rows over 8192 keys (72 GFLOP, 32
// steps) 107 and 101.  (A large library product reaches 1150-1190 TFLOP/s, and products on random
// values in registers alone 1675 once they run long: the clock falls.)  The matrix unit is busy 22 %
// of the first one's time.  By cycle stamps, with which the call takes a tenth more, a wave of it lives
// 129 000 cycles at 2.2 GHz, the longest 17 % more.  Its steps are 99 000, 5400 each, of which 2200 are
// products: S 2400 with the bf16 rows' copies among them (4-bit keys 2000), edges and the search for
// the largest 290, exponentials 570, the moved reference 370 on average, two meetings 410, O 1350
// (2000 with the 4-bit keys' conversion).  What is not steps: the run and tiles found 6000, queries and
// first keys 13 000, results 10 500.
// Copies in the second product's time and more operands ahead made nothing of it faster; steps of
// 32 keys in three places, with the softmax beside the second product's instructions and one
// meeting a step, took 80 us where this took 74: what a step waits for at its beginning then comes
// twice as often.
#include "latent_attend.h"

namespace mlh {

namespace latent_attention {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kCols = Wide::kCols, kStepKeys = Wide::kStepKeys;
constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kWaveCols = 32, kWaveKeys = 32;  // of a wave's scores
constexpr int kWaveDims = kLatentMax / kWaves;  // of its sums
constexpr int kStageKeys = kStepKeys / kWaves;  // keys that a wave brings in
constexpr int kRowSteps = kLatentMax / 16, kQuerySteps = (kLatentMax + kLatentRopeMax) / 16;
constexpr int kGroup = 4;  // of products whose operands are read at once
constexpr int kTiles = kWaveDims / 32, kColTiles = kCols / 32;

// LDS: two steps' keys.  Piece q (16 bytes) of latent row k is at q ^ turn(k): 16 rows' pieces
// of one place lie in different banks, and the four neighbouring pieces of four rows do.
// Rope pieces: [16 keys][piece][key].
constexpr int kLatentBytes = kStepKeys * kLatentMax * 2;
constexpr int kStepBytes = kLatentBytes + kStepKeys * kLatentRopeMax * 2;
__device__ __forceinline__ int turn(int key) { return (key & 3) << 2 | (key >> 2 & 3); }

constexpr int kRopeRows = kStageKeys * kLatentRopeMax * 2;  // bytes of 16 keys
// Then, of each column, P of a step's keys: piece 2 k + h has those of product k that lane half h
// holds.
constexpr int kProbStride = kStepKeys * 2 + 16;
constexpr int kLdsBytes = 2 * kStepBytes + kCols * kProbStride;
// Over the keys, at the end of a tile, each wave's results, piece q of column c at q ^ c % 16.
static_assert(2 * kStepBytes >= kCols * kLatentMax * 4, "LDS");

__device__ __forceinline__ f32x16 mfma(const u32x4 &a, const u32x4 &b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                   c, 0, 0, 0);
}

// The sums stay in accumulation registers.
__device__ __forceinline__ void keep(f32x16 &v) { asm volatile("" : "+a"(v)); }

// Over the two halves of a wave.
__device__ __forceinline__ float halves_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

typedef __attribute__((address_space(3))) uint8_t LdsByte;
typedef __attribute__((address_space(3))) u32x4 LdsPiece;
typedef const __attribute__((address_space(1))) void *GlobalPtr;

// All of this wave's LDS accesses are done (and, meet, its loads have arrived); then all waves'.
__device__ __forceinline__ void meet_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <bool FP4> __global__ __launch_bounds__(kThreads, 1) void latent_wide_kernel(Params p) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float highs[2][kCols], sums[2][kCols];
    __shared__ __attribute__((aligned(16))) unsigned bads[2][kWaves];  // of a step's keys: those without a place
    __shared__ int flags[2];
    __shared__ LatentSeq held[kThreads];
    const int t = threadIdx.x, wave = uniform(t / kWave), lane = t % kWave;
    const int col0 = wave % 2 * kWaveCols, half = wave / 2;  // half: which keys of a step
    const int c = lane % 32, h = lane / 32;
    constexpr int kWidth = kLatentMax + kLatentRopeMax;
    constexpr int row_bytes = latent_row_bytes(FP4, kLatentMax, kLatentRopeMax);
    LdsByte *const base_lds = (LdsByte *)lds;

    // Workgroups go to the 8 XCDs in turn: each gets a run of neighbouring tiles, whose keys
    // its L2 holds.
    const int xcd = blockIdx.x % 8, longer = p.groups % 8;
    const int group = xcd * (p.groups / 8) + (xcd < longer ? xcd : longer) + blockIdx.x / 8;
    const Run run = find_run<Wide, kWaves>(p, group, held);
    begin_records(p, run, group);

    // Where a lane reads: of keys (queries) their row c, and of 4 keys' 64 bytes its 8; a place in a
    // row is reached by changing bits of these.
    const int row_turn = c * (kLatentMax * 2) + (h ^ turn(c)) * 16;
    const int rope_turn = kLatentBytes + c / 16 * kRopeRows + c % 16 * 16 + h * 256;
    const int v_key = lane % 16 / 4;
    const int v_at = (4 * h + v_key) * (kLatentMax * 2) + lane % 2 * 8 + wave * (kWaveDims * 2) +
                     16 * ((2 * (c / 16) + lane % 4 / 2) ^ (v_key << 2 | h));
    const int prob_at = 2 * kStepBytes + c * kProbStride + 16 * h;
    // and where it brings keys to: key c16 of its wave's, lane group g
    const int c16 = lane % 16, g = lane / 16;
    const int own_key = kStageKeys * wave + c16;

    int left = run.length, offset = run.offset;
    for (int s = run.seq; left > 0 && s < p.b.seqs; ++s, offset = 0) {
        const LatentSeq seq = p.b.seqs <= kThreads ? held[s] : latent_seq(p.b, s, p.rows);
        const Work w = work_of<Wide>(p, {uniform(seq.begin), uniform(seq.count), uniform(seq.length)});
        while (left > 0 && offset < w.per * w.tiles) {
            const int tile = (int)((unsigned)offset / (unsigned)w.per), first = offset - tile * w.per;
            const int last = left < w.per - first ? first + left : w.per;
            left -= last - first;
            offset += last - first;

            // the tile's columns, and the keys that they see, as far as the table goes
            const int pair0 = tile * kCols, pairs = w.seq.count * p.heads;
            const int used = pairs - pair0 < kCols ? pairs - pair0 : kCols;
            const long base = (long)w.seq.begin * p.heads + pair0;  // among all (row, head) pairs
            const auto sees_of = [&](int col) {
                return (long)w.seq.length - w.seq.count + 1 + (int)p.head.quotient((unsigned)(pair0 + col));
            };
            const auto within_of = [&](long sees) { return sees < 0 ? 0 : sees < w.keys ? (int)sees : w.keys; };
            const bool mine = col0 + c < used;
            const long sees = sees_of(mine ? col0 + c : 0);
            const int limit = mine ? within_of(sees) : 0;
            const int least = uniform(within_of(sees_of(0))), most = uniform(within_of(sees_of(used - 1)));
            // in steps
            const int from = first << p.shift, seen_steps = (most + kStepKeys - 1) >> Wide::kStepShift;
            const int upto = (last << p.shift) < seen_steps ? last << p.shift : seen_steps;

            // The keys that a wave brings in: their pages, asked for two steps before those, and then
            // their addresses and whether they have one.  Keys that nothing sees are taken from page 0.
            const int *table = p.b.tables + (long)s * p.b.table_width;
            unsigned in_page;
            bool any_page;
            int page;
            const auto ask = [&](int step) {
                const unsigned j = (unsigned)step * kStepKeys + own_key, at = p.page.quotient(j);
                in_page = j - at * (unsigned)p.b.page_size;
                any_page = step >= upto || j >= (unsigned)most;
                page = table[any_page ? 0 : at];
            };
            const uint8_t *row = nullptr;
            const auto find = [&](int step) {
                const int place = any_page ? 0 : page;
                const bool there = (unsigned)place < (unsigned)p.b.pages;
                bads[step & 1][wave] = (unsigned)__ballot(!there) & 0xFFFFu;
                const unsigned long slot = (unsigned long)(there ? (unsigned)place : 0u) * (unsigned)p.b.page_size +
                                           (there ? in_page : 0u);
                row = static_cast<const uint8_t *>(p.b.data) + slot * row_bytes;
            };
            ask(from);
            // 4-bit keys go through registers, to be written as bf16 ones, 16 bytes of a lane at a time.
            Raw<true> codes;
            const auto load_codes = [&] {
                if constexpr (FP4) {
#pragma unroll
                    for (int j = 0; j < kSteps / 4; ++j) codes.codes[j] = load_global16(row + 64 * j + 16 * g);
                    codes.scales = *(const __attribute__((address_space(1))) unsigned *)(row + kLatentMax / 2 + 4 * g);
                }
            };
            // row k of a wave's, from the lane that has its address
            const auto bring_row = [&](LdsByte *to, const uint8_t *row, int k) {
                const unsigned lo = (unsigned)(unsigned long long)row, hi = (unsigned)((unsigned long long)row >> 32);
                void *from = (void *)((unsigned long long)__builtin_amdgcn_readlane(hi, k) << 32 |
                                      (unsigned)__builtin_amdgcn_readlane(lo, k));
                unsigned at = 16 * lane;
                asm volatile("" : "+v"(at));
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    __builtin_amdgcn_make_buffer_rsrc(from, 0, kLatentMax * 2, 0x00027000),
                    to + (kStageKeys * wave + k) * (kLatentMax * 2), 16, at ^ 16 * turn(k), 0, 0, 0);
            };
            const auto bring_rope = [&](LdsByte *to, const uint8_t *rope, int k) {
                __builtin_amdgcn_global_load_lds((GlobalPtr)(rope + 16 * g + 64 * k),
                                                 to + kLatentBytes + wave * kRopeRows + 1024 * k, 16, 0, 0);
            };
            constexpr int kPieces = (FP4 ? 0 : kStageKeys) + 2;
            const auto bring = [&](int step, int k) {
                LdsByte *to = base_lds + (step & 1) * kStepBytes;
                if (k < kPieces - 2) bring_row(to, row, k);
                else bring_rope(to, row + latent_part_bytes(FP4, kLatentMax), k - (kPieces - 2));
            };
            const auto put = [&](int step, int j) {
                if constexpr (FP4) {
                    int at = own_key * (kLatentMax * 2) + 16 * (4 * g ^ turn(c16)) + (step & 1) * kStepBytes;
                    asm volatile("" : "+v"(at));
                    at &= 0x3FFFF;
                    *(LdsPiece *)(base_lds + (at ^ 16 * (j % 4)) + 256 * (j / 4)) =
                        operand<true, true>(codes, j, g, kLatentMax);
                }
            };

            // The columns' reference, of columns c and 32 + c; a wave's share of its columns' sums; a row
            // that sees keys behind its table is NaN.
            float top[2] = {-INFINITY, -INFINITY};
            float sum = mine && sees > w.keys ? NAN : 0.0f;
            u32x4 query[kQuerySteps];
            f32x16 out[kTiles][kColTiles];
            __syncthreads();  // (the tile before is done with the LDS)
            if (t == 0) flags[from & 1] = 0;
            if (from < upto) {
                // The queries come as keys do, in the place of the second step's.  (Columns without a pair
                // take the last one's; nobody asks for their results.)
                LdsByte *to = base_lds + (~from & 1) * kStepBytes;
                const int col = own_key < used ? own_key : used - 1;
                const uint8_t *at = static_cast<const uint8_t *>(p.q) + (base + col) * (kWidth * 2);
#pragma unroll
                for (int k = 0; k < kStageKeys; ++k) bring_row(to, at, k);
#pragma unroll
                for (int k = 0; k < 2; ++k) bring_rope(to, at + kLatentMax * 2, k);
                find(from);
                ask(from + 1);
                load_codes();
#pragma unroll
                for (int k = 0; k < kPieces; ++k) bring(from, k);
#pragma unroll
                for (int j = 0; j < kSteps; ++j) put(from, j);
                find(from + 1);
                ask(from + 2);
                meet();
                int straight = row_turn + col0 * (kLatentMax * 2) + (~from & 1) * kStepBytes;
                asm volatile("" : "+v"(straight));
                straight &= 0x3FFFF;
#pragma unroll
                for (int j = 0; j < kQuerySteps; ++j)
                    query[j] = *(const LdsPiece *)(base_lds +
                                                   (j < kRowSteps ? (straight ^ 2 * j % 16 * 16) + 256 * (j / 8)
                                                                  : rope_turn + col0 / 16 * kRopeRows +
                                                                        (~from & 1) * kStepBytes + 512 * (j - kRowSteps)));
            }
#pragma unroll
            for (int j = 0; j < kTiles; ++j)
#pragma unroll
                for (int x = 0; x < kColTiles; ++x) {
                    out[j][x] = f32x16{0.f};
                    keep(out[j][x]);
                }

            for (int step = from; step < upto; ++step) {
                const int buf = step & 1, key0 = step * kStepKeys;
                meet();
                const u32x4 bad4 = *(const LdsPiece *)bads[buf];
                // (addresses are computed anew, which leaves registers for the products)
                int straight = row_turn + half * (kWaveKeys * kLatentMax * 2) + buf * kStepBytes, turned = v_at + buf * kStepBytes;
                asm volatile("" : "+v"(straight), "+v"(turned));
                straight &= 0x3FFFF, turned &= 0x3FFFF;

                // S; reads are two groups ahead of their products
                u32x4 part[3][kGroup];
                const auto read = [&](int n) {
#pragma unroll
                    for (int x = 0; x < kGroup; ++x) {
                        const int j = n * kGroup + x;
                        part[n % 3][x] = *(const LdsPiece *)(base_lds +
                                                             (j < kRowSteps ? (straight ^ 2 * j % 16 * 16) + 256 * (j / 8)
                                                                            : rope_turn + 2 * half * kRopeRows +
                                                                                  buf * kStepBytes + 512 * (j - kRowSteps)));
                    }
                };
                read(0);
                read(1);
                load_codes();  // (behind the last step: keys from page 0, that nothing uses)
                f32x16 score = {0.f};
                asm volatile("" : "+v"(score));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < kQuerySteps / kGroup; ++n) {
                    if (n + 2 < kQuerySteps / kGroup) read(n + 2);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int x = 0; x < kGroup; ++x) {
                        score = mfma(part[n % 3][x], query[n * kGroup + x], score);
                        const int k = 2 * n + x / 2 - (2 * kQuerySteps / kGroup - kPieces);
                        if (x % 2 && k >= 0) bring(step + 1, k);
                        if (x % 2) __builtin_amdgcn_sched_barrier(0);
                    }
                }

                float scale = p.scale;
                float high = score[0], low = score[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) high = fmaxf(high, score[i]), low = fminf(low, score[i]);
                if (__any(fmaxf(fabsf(high), fabsf(low)) * fabsf(scale) >= kLarge)) {
                    // (the product that `top` is of is the one that is subtracted from)
#pragma unroll
                    for (int i = 0; i < 16; ++i) score[i] = large_score(score[i] * scale);
                    high = scale >= 0 ? high * scale : low * scale;
                    scale = 1.0f;
                } else {
                    high = scale >= 0 ? high * scale : low * scale;
                }
                const unsigned bad = (unsigned)uniform((int)(bad4[0] | bad4[1] | bad4[2] | bad4[3]));
                if (bad || key0 + kStepKeys > least) {
                    // Keys that not every column sees, or that have no place: those that a column
                    // does not see must not reach it by 0 * NaN either, so rows that are not finite
                    // (or not there) become zeros and make NaN of the scores of the columns that
                    // see them.
                    // (Each wave those that it brought; a row that others may still be reading for S
                    // counts for nothing there.)
                    int own_at = buf * kStepBytes + own_key * (kLatentMax * 2);
                    asm volatile("" : "+v"(own_at));
                    u16x2 largest = {0, 0};
#pragma unroll 8
                    for (int j = 0; j < kLatentMax / 32; ++j) {  // (in an order that has lanes on all banks)
                        const u32x4 v = *(const LdsPiece *)(base_lds + own_at + 16 * ((4 * j + g) ^ c16));
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            largest = __builtin_elementwise_max(largest, __builtin_bit_cast(u16x2, v[i] & 0x7FFF7FFFu));
                    }
                    const bool seen = key0 + own_key < most;
                    const unsigned long long which = __ballot(seen && (largest[0] >= 0x7F80u || largest[1] >= 0x7F80u));
                    const unsigned wrong = bads[buf][wave] |
                                           ((unsigned)(which | which >> 16 | which >> 32 | which >> 48) & 0xFFFFu);
                    if (!seen || (wrong >> c16 & 1u)) {
#pragma unroll 8
                        for (int j = 0; j < kLatentMax / 32; ++j)
                            *(LdsPiece *)(base_lds + own_at + 16 * ((4 * j + g) ^ c16)) = u32x4{0, 0, 0, 0};
                    }
                    bads[buf][wave] = wrong;
                    meet_lds();
                    const unsigned bits = (bads[buf][2 * half] | bads[buf][2 * half + 1] << 16) >> 4 * h;
                    const int end = limit - (key0 + kWaveKeys * half + 4 * h);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int k = 8 * (i / 4) + i % 4;
                        score[i] = bits >> k & 1u ? NAN : score[i] * scale;
                        if (k >= end) score[i] = -INFINITY;
                    }
                    scale = 1.0f;
                    high = score[0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) high = fmaxf(high, score[i]);
                }
                high = halves_max(high);
                highs[half][col0 + c] = high;
                flags[~step & 1] = 0;
                const float own_top = col0 ? top[1] : top[0];
                if (__any(high > own_top + kSlack)) flags[step & 1] = 1;
                float added;
                const auto exponentials = [&](float to) {
                    added = 0.0f;
                    u32x4 probs[2];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float a = __builtin_amdgcn_exp2f(fmaf(score[2 * i], scale, -to));
                        const float b = __builtin_amdgcn_exp2f(fmaf(score[2 * i + 1], scale, -to));
                        const bf16x2 r = {(__bf16)a, (__bf16)b};
                        added = __builtin_amdgcn_fdot2_f32_bf16(r, bf16x2{(__bf16)1.0f, (__bf16)1.0f}, added, false);
                        probs[i / 4][i % 4] = __builtin_bit_cast(unsigned, r);
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m)
                        *(LdsPiece *)(base_lds + prob_at + col0 * kProbStride + 32 * (2 * half + m)) = probs[m];
                };
                exponentials(own_top == -INFINITY ? 0.0f : own_top);

                // O; reads are a group ahead, the first values before all waves' P are there
                u32x4 values[2][kTiles], probs[2][kColTiles];
                const auto read_values = [&](int k) {
#pragma unroll
                    for (int j = 0; j < kTiles; ++j)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            LdsByte *at = base_lds + (turned ^ (j * 64 | u * 32)) + (16 * k + 8 * u) * (kLatentMax * 2);
                            const auto y = __builtin_bit_cast(unsigned long long, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                                                      (__attribute__((address_space(3))) s16x4 *)at));
                            values[k % 2][j][2 * u] = (unsigned)y;
                            values[k % 2][j][2 * u + 1] = (unsigned)(y >> 32);
                        }
                };
                const auto read_probs = [&](int k) {
#pragma unroll
                    for (int x = 0; x < kColTiles; ++x)
                        probs[k % 2][x] = *(const LdsPiece *)(base_lds + prob_at + 32 * x * kProbStride + 32 * k);
                };
                read_values(0);
                meet_lds();
                const int flag = flags[step & 1];
                read_probs(0);
                asm volatile("" : "+v"(probs[0][0]), "+v"(probs[0][1]));  // (read with the flag, not after it)
                if (uniform(flag)) {
                    const bool begun = __any(top[0] != -INFINITY || top[1] != -INFINITY);  // (else there is nothing yet, or NaN)
                    float by[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float next = fmaxf(top[x], fmaxf(highs[0][32 * x + c], highs[1][32 * x + c]));
                        by[x] = top[x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top[x] - next);
                        top[x] = next;
                    }
                    sum *= col0 ? by[1] : by[0];
                    if (begun) {
#pragma unroll
                        for (int j = 0; j < kTiles; ++j)
#pragma unroll
                            for (int x = 0; x < kColTiles; ++x) {
                                keep(out[j][x]);
                                out[j][x] *= by[x];
                                keep(out[j][x]);
                            }
                    }
                    const float to = col0 ? top[1] : top[0];
                    exponentials(to == -INFINITY ? 0.0f : to);
                    meet_lds();
                    read_probs(0);
                }
                sum += added;

#pragma unroll
                for (int k = 0; k < kStepKeys / 16; ++k) {
                    if (k + 1 < kStepKeys / 16) {
                        read_probs(k + 1);
                        read_values(k + 1);
                    }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) {
                        if (k == 0 && j == 2) find(step + 2);
                        if (k == 1 && j == 0) ask(step + 3);
#pragma unroll
                        for (int x = 0; x < kColTiles; ++x)
                            out[j][x] = mfma(values[k % 2][j], probs[k % 2][x], out[j][x]);
                        put(step + 1, 4 * k + j);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }

            // Columns' sums, then results by way of LDS, each wave its own values: as they lie in
            // registers, a store would take 16 bytes of each of 64 rows.
            const bool whole = first == 0 && last == w.per;
            const int part = 2 * group + (first == 0 ? 1 : 0);
            sum += __shfl_xor(sum, 32, kWave);
            if (h == 0) sums[half][col0 + c] = sum;
            meet();
            // (what follows from this is not worth registers from one tile to the next)
            int id = lane;
            asm volatile("" : "+v"(id));
            float col_sum[kColTiles];
#pragma unroll
            for (int x = 0; x < kColTiles; ++x) col_sum[x] = sums[0][32 * x + id % 32] + sums[1][32 * x + id % 32];
            if (!whole && wave == 0) {
                p.parts.stats[part * 2 * kCols + id] = h ? top[1] : top[0];
                p.parts.stats[(part * 2 + 1) * kCols + id] = h ? col_sum[1] : col_sum[0];
            }
            float *results = reinterpret_cast<float *>(lds) + wave * (kCols * kWaveDims);
#pragma unroll
            for (int x = 0; x < kColTiles; ++x) {
                const float over = !whole ? 1.0f : col_sum[x] == 0.0f ? 0.0f : 1.0f / col_sum[x];
#pragma unroll
                for (int j = 0; j < kTiles; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x16 &o = out[j][x];
                        *reinterpret_cast<f32x4 *>(results + (32 * x + id % 32) * kWaveDims +
                                                   4 * ((8 * j + 2 * i + id / 32) ^ id % 16)) =
                            f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]} * over;
                    }
            }
#pragma unroll 8
            for (int pass = 0; pass < kCols / 2; ++pass) {
                const int col = 2 * pass + id / 32, d = wave * kWaveDims + 4 * (id % 32);
                const f32x4 v = load_f4(results + col * kWaveDims + 4 * (id % 32 ^ col % 16));
                if (!whole) *reinterpret_cast<f32x4 *>(p.parts.sums + ((long)part * kCols + col) * kLatentMax + d) = v;
                else if (col < used) store4<true>(p.out, (base + col) * kLatentMax + d, v);
            }
            if (t == 0 && last == w.per && (first > 0 || p.parts.tiles)) {
                // (owner: of the tile's first unit)
                const Record record = {s, tile, first > 0 ? run.owner(run.begin - first) : -1, group};
                p.parts.records[p.parts.tiles ? (int)(base / kCols) + s : group] = record;
            }
        }
    }
}

template <bool FP4> int launch(const Params &p, hipStream_t stream) {
    const auto kernel = latent_wide_kernel<FP4>;
    static const bool ok = allow_lds(kernel, kLdsBytes);
    if (!ok) return kErrLaunch;
    kernel<<<p.groups, kThreads, kLdsBytes, stream>>>(p);
    if (hipGetLastError() != hipSuccess) return kErrLaunch;
    return launch_join<Wide, true>(p, stream);
}

}  // namespace

int launch_wide(bool fp4, const Params &p, hipStream_t stream) {
    return fp4 ? launch<true>(p, stream) : launch<false>(p, stream);
}

}  // namespace latent_attention

}  // namespace mlh
