// latent_attend.hip -- attention of a batch's token rows over a paged latent cache
// (gfx950, wave64).
//
//   s_j = scale * q . [latent_j | rope_j],  out = sum_j exp(s_j - m) latent_j / sum_j exp(s_j - m)
//
// for each (token row, head); a sequence's (row, head) pairs are taken 16 at a time (a tile:
// the 16 columns of a matrix instruction), and a tile's keys 16 at a time (a step, and a unit
// of work where those can be counted in 32 bits).  The units of all tiles, in order, are
// dealt out in equal runs to as many workgroups as the chip holds, so ragged lengths leave
// none of them idle; a tile whose units fell to several is joined by latent_join_kernel from
// their partial sums.
//
// The waves of a workgroup take its steps in turn, with a running maximum and sum of their
// own, and meet at the end of a tile.  The keys are read straight into the matrix operand
// (lane (k, g): 8 values of key k at a product step), so the scores S[key][column] come from
// v_mfma_f32_16x16x32_bf16; their registers hold 4 keys of a column, which is the operand
// layout of the second product O[latent][column] += V^T P on v_mfma_f32_16x16x16_bf16.
// V^T, the same keys with the latent index across lanes, is a product too: with the
// identity, whose result registers hold 4 keys of a latent value, exact and to be packed.
// (Through LDS, written in rows and read transposed, it is 16 KB of writes and as much of
// reads a step: 4-bit keys took the same, bf16 ones 3 % less, and f32 queries, for which the
// LDS then has room for four waves only, 13 % more.)  f32 queries and probabilities go in as
// three bf16 parts each, which add up to them.
//
// The next keys are on their way from when the first product has taken the present ones, and
// the page numbers of those after them.
//
// What runs once costs its instructions' way from memory, about 4 cycles a byte: loops are
// entered a step early rather than with a copy of their loads before them, and unrolled
// only where registers are counted.
//
// With bf16 queries a key's p is rounded to bf16, as one operand of the second product: in two bf16
// parts, which add up to 16 bits of it, 64 rows over 4-bit keys take 58 us instead of 53 and 16 long
// rows over bf16 keys 72 instead of 71, and the results come as near to those in 64 bits as their own
// rounding lets them, 0.00159 and 0.00166 of their norm; with the one part it is 0.00172 and 0.00176.
//
// Measured with 16 heads (calls without the join, and what it adds): 16 rows over 16000 .. 16384
// bf16 keys each, 299 MB, 66 and 5 us, 4.5 TB/s; a kernel that only reads the same rows, a key's 64
// bytes by four lanes, takes 54, one that reads 1 KB runs 47-49 and a plain read 43: what bounds it is
// the reads, by the order that the operand asks for, and the start.  64 rows over 4-bit keys, 159 MB,
// 48 and 5; reading alone takes 31, a plain read 23: two waves a SIMD whose products, codes'
// conversion (twice a step, once for each product) and softmax follow each other keep the matrix
// unit busy 26 % of the time and the vector units 34 %.  The scores of a step beside the softmax of
// the one before are not tried: the kernel has 243 of 256 registers, 128 of them sums.  One row over
// 4096 bf16 keys 10 and 6, 17 rows of f32 queries over 4-bit keys 21 and 6: some seven trips to
// memory that depend on each other, a microsecond each, with lengths and tables among them.
// f32 queries and probabilities take 182 products of 16 columns by 16 keys: chunks of 32, 64, 96 and
// 128 rows over 3000 .. 4096 keys 190 us over 4-bit keys and 290 over bf16 ones, whose registers leave
// one wave a SIMD instead of two: the matrix unit is busy 54 and 33 % of the time.
#include "latent_attend.h"

namespace mlh {

using namespace latent_attention;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kCols = Narrow::kCols, kStepKeys = Narrow::kStepKeys;
constexpr int kAllSteps = kSteps + kRopeSteps;
constexpr int kDims = kLatentMax / 16;  // 16-value tiles of a latent row

// Waves of a workgroup, one workgroup a CU.  4-bit keys leave a wave in 256 registers, for two
// waves on a SIMD; of bf16 keys, 72 registers a step, two steps are held by one.
template <bool FP4> constexpr int kWavesOf = FP4 ? 8 : 4;

// LDS: the queries (three bf16 parts of f32 ones); then, over them, the waves' results,
// kJoinDims latent values of each column at a time, piece q (16 bytes) of column c at q ^ c:
// the 16 lanes that write a piece of each column find them in different banks.
constexpr int kQueryStride = kLatentMax + kLatentRopeMax + 8;
template <bool BF16> constexpr int kQueryBytes = (BF16 ? 1 : 3) * kCols * kQueryStride * 2;
constexpr int kJoinDims = 256;
constexpr int kJoinBytes = kCols * kJoinDims * 4;  // of a wave
template <bool FP4, bool BF16> constexpr int kLdsBytes =
    kQueryBytes<BF16> > kWavesOf<FP4> * kJoinBytes ? kQueryBytes<BF16> : kWavesOf<FP4> * kJoinBytes;

// x as three bf16 parts that add up to it, cut off one after the other.
__device__ __forceinline__ void split3(float x, unsigned (&part)[3]) {
    const unsigned a = __float_as_uint(x) & 0xFFFF0000u;
    const float r = x - __uint_as_float(a);
    const unsigned b = __float_as_uint(r) & 0xFFFF0000u;
    const float l = r - __uint_as_float(b);
    part[0] = a >> 16;
    part[1] = b >> 16;
    part[2] = __float_as_uint(l) >> 16;
}

__device__ __forceinline__ f32x4 mfma32(const u32x4 &a, const u32x4 &b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The largest of a value over the four lane groups.
__device__ __forceinline__ float groups_max(float v) {
    const unsigned u = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const unsigned w = __float_as_uint(m);
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A sum that is in an accumulation register here.  With 512 registers, where sums begin and
// where they are scaled, on both sides: else the compiler has all 128 moved out and back at
// every step.  (Of 256 all are alike.)
__device__ __forceinline__ void keep(f32x4 &v) { asm volatile("" : "+a"(v)); }

template <bool FP4, bool BF16, bool FULL>
__global__ __launch_bounds__((kWavesOf<FP4> * kWave), 1) void latent_attend_kernel(Params p) {
    constexpr int kWaves = kWavesOf<FP4>, kThreads = kWaves * kWave;
    constexpr int kParts = BF16 ? 1 : 3;  // bf16 parts of a query value and of a probability
    constexpr int kGroup = 4;  // product steps that may be mixed: more of them takes more registers
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ __attribute__((aligned(16))) float tops[kCols][kWaves], sums[kCols][kWaves];
    __shared__ LatentSeq held[kThreads];
    const int t = threadIdx.x, wave = uniform(t / kWave), lane = t % kWave;
    const int g = lane / 16, c = lane % 16;
    const int latent = FULL ? kLatentMax : p.b.latent, rope = FULL ? kLatentRopeMax : p.b.rope;
    const int width = latent + rope;
    const int row_bytes = latent_row_bytes(FP4, latent, rope);
    uint16_t *query_lds = reinterpret_cast<uint16_t *>(lds);

    // Column c of the identity's two halves: with 32 values of each key as the other operand,
    // out comes value c, or 16 + c, of every key.
    u32x4 identity[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            identity[h][i] = g == 2 * h + c / 8 && i == c % 8 / 2 ? c % 2 ? 0x3F800000u : 0x3F80u : 0u;

    const int group = blockIdx.x;
    const Run run = find_run<Narrow, kWaves>(p, group, held);
    begin_records(p, run, group);
    int left = run.length, offset = run.offset;
    for (int s = run.seq; left > 0 && s < p.b.seqs; ++s, offset = 0) {
        const LatentSeq seq = p.b.seqs <= kThreads ? held[s] : latent_seq(p.b, s, p.rows);
        const Work w = work_of<Narrow>(p, {uniform(seq.begin), uniform(seq.count), uniform(seq.length)});
        while (left > 0 && offset < w.per * w.tiles) {
            // (what follows from it is not worth a register from one tile to the next)
            int tid = t;
            asm volatile("" : "+v"(tid));
            const int tile = (int)((unsigned)offset / (unsigned)w.per), first = offset - tile * w.per;
            const int last = left < w.per - first ? first + left : w.per;
            left -= last - first;
            offset += last - first;

            // the tile's columns, and the keys that they see, as far as the table goes
            const int pair0 = tile * kCols, pairs = w.seq.count * p.heads;
            const int used = pairs - pair0 < kCols ? pairs - pair0 : kCols;
            const long base = (long)w.seq.begin * p.heads + pair0;  // among all (row, head) pairs
            // (the row's own key, and those before it; 32 bits: both are below 2^31)
            const long sees = (long)w.seq.length - w.seq.count + 1 +
                              (int)p.head.quotient((unsigned)(pair0 + (c < used ? c : 0)));
            const int within = sees < 0 ? 0 : sees < w.keys ? (int)sees : w.keys;
            const int limit = c < used ? within : 0;
            const int least = __builtin_amdgcn_readlane(within, 0);
            const int most = __builtin_amdgcn_readlane(within, used - 1);
            // in steps
            const int from = first << p.shift, seen_steps = (most + kStepKeys - 1) / kStepKeys;
            const int upto = (last << p.shift) < seen_steps ? last << p.shift : seen_steps;

            // A key's page, asked for a step before the key; keys that nothing sees are taken from
            // page 0 (and out of the products).
            const int *table = p.b.tables + (long)s * p.b.table_width;
            const auto page_of = [&](int step, unsigned *in_page) {
                const unsigned j = (unsigned)step * kStepKeys + c, at = p.page.quotient(j);
                *in_page = j - at * (unsigned)p.b.page_size;
                int page = 0;
                if (step < upto && j < (unsigned)most) page = table[at];
                return page;
            };
            unsigned in_page;
            int page = page_of(from + wave, &in_page);

            // the queries, 8 values a thread and pass
            constexpr int kPieces = (kLatentMax + kLatentRopeMax) / 8;
            constexpr int kLoads = (kCols * kPieces + kThreads - 1) / kThreads;
            u32x4 pieces[kLoads][BF16 ? 1 : 2];
#pragma unroll
            for (int y = 0; y < kLoads; ++y) {
                const int i = tid + y * kThreads, col = i / kPieces, d = 8 * (i % kPieces);
                const bool in = col < used && (FULL || (d < kLatentMax ? d < latent : d - kLatentMax < rope));
                const long at = (base + col) * width + (FULL || d < kLatentMax ? d : latent + d - kLatentMax);
#pragma unroll
                for (int h = 0; h < (BF16 ? 1 : 2); ++h) {
                    pieces[y][h] = u32x4{0, 0, 0, 0};
                    if (!in) continue;
                    if constexpr (BF16) pieces[y][h] = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(p.q) + at);
                    else __builtin_memcpy(&pieces[y][h], static_cast<const float *>(p.q) + at + 4 * h, 16);
                }
            }
            // Running softmax: lane (c, g) holds column c, its sum over keys 4 g .. 4 g + 3 of
            // every step; a row that sees keys behind its table is NaN.
            float top = -INFINITY, sum = c < used && sees > w.keys ? NAN : 0.0f;
            f32x4 out[kDims];

            Raw<FP4> raw, next;
            unsigned bad_pages, next_bad;  // keys without a place
            // the keys of the step whose pages are there, and the pages of the step after it
            const auto go_on = [&](int step) {
                const bool there = (unsigned)page < (unsigned)p.b.pages;
                const long slot = there ? (long)page * p.b.page_size + in_page : 0;
                next_bad = (unsigned)__ballot(!there) & 0xFFFFu;
                page = page_of(step + kWaves, &in_page);
                load_key<FP4, FULL>(next, static_cast<const uint8_t *>(p.b.data) + slot * row_bytes, g, latent, rope);
            };
            go_on(from + wave);
            __syncthreads();  // (the tile before is done with them)
#pragma unroll
            for (int y = 0; y < kLoads; ++y) {
                const int i = tid + y * kThreads, col = i / kPieces, d = 8 * (i % kPieces);
                if (kCols * kPieces % kThreads && i >= kCols * kPieces) break;
                uint16_t *to = query_lds + col * kQueryStride + d;
                if constexpr (BF16) {
                    *reinterpret_cast<u32x4 *>(to) = pieces[y][0];
                } else {
                    u32x4 v[3];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        unsigned lo[3], hi[3];
                        split3(__uint_as_float(pieces[y][k / 2][2 * (k % 2)]), lo);
                        split3(__uint_as_float(pieces[y][k / 2][2 * (k % 2) + 1]), hi);
#pragma unroll
                        for (int x = 0; x < 3; ++x) v[x][k] = lo[x] | hi[x] << 16;
                    }
#pragma unroll
                    for (int x = 0; x < 3; ++x) *reinterpret_cast<u32x4 *>(to + x * kCols * kQueryStride) = v[x];
                }
            }
            __syncthreads();
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                out[d] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (kWaves == 4) keep(out[d]);
            }

            for (int step = from + wave; step < upto; step += kWaves) {
                const int key0 = step * kStepKeys;
                raw = next;
                bad_pages = next_bad;
                f32x4 score[kParts];
#pragma unroll
                for (int k = 0; k < kParts; ++k) score[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < kAllSteps; ++j) {
                    const u32x4 v = operand<FP4, FULL>(raw, j, g, latent);
                    const int at = j < kSteps ? dim_of<FP4>(j, g) : kLatentMax + 32 * (j - kSteps) + 8 * g;
#pragma unroll
                    for (int k = 0; k < kParts; ++k)
                        score[k] = mfma32(v, *reinterpret_cast<const u32x4 *>(query_lds + (k * kCols + c) * kQueryStride + at),
                                          score[k]);
                    if (j % kGroup == kGroup - 1) __builtin_amdgcn_sched_barrier(0);
                }
                if (step + kWaves < upto) go_on(step + kWaves);
                f32x4 sc = score[0];
                if constexpr (!BF16) sc += score[1] + score[2];
                bool hidden[4] = {false, false, false, false};
                if (bad_pages || key0 + kStepKeys > least) {
                    // Keys that not every column sees, or that have no place: those that a
                    // column does not see must not reach it by 0 * NaN either, so rows that
                    // are not finite (or not there) are taken out of the second product and
                    // make NaN of the scores of the columns that see them.
                    const bool mine = key0 + c < most;
                    const unsigned long long which = __ballot(mine && not_finite(raw, g, latent));
                    const unsigned bad = bad_pages | ((unsigned)(which | which >> 16 | which >> 32 | which >> 48) & 0xFFFFu);
                    if (!mine || (bad >> c & 1u)) drop(raw);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (bad >> (4 * g + i) & 1u) sc[i] = NAN;
                        hidden[i] = key0 + 4 * g + i >= limit;
                    }
                }
                float scale = p.scale, high = -INFINITY;
                const auto set_high = [&] {
                    high = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; ++i) high = fmaxf(high, hidden[i] ? -INFINITY : sc[i] * scale);
                };
                set_high();
                const float largest = fabsf(scale) * fmaxf(fmaxf(fabsf(sc[0]), fabsf(sc[1])), fmaxf(fabsf(sc[2]), fabsf(sc[3])));
                if (__any(high > top + kSlack || largest >= kLarge)) {
                    if (__any(largest >= kLarge)) {
                        // (the product that `top` is of is the one that is subtracted from)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[i] = large_score(sc[i] * scale);
                        scale = 1.0f;
                        set_high();
                    }
                    const float next = fmaxf(top, groups_max(high));
                    const float by = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next);
                    const bool begun = __any(top != -INFINITY);  // (else there is nothing yet, or NaN)
                    sum *= by;
                    top = next;
                    if (begun) {
#pragma unroll
                        for (int d = 0; d < kDims; ++d) {
                            if constexpr (kWaves == 4) keep(out[d]);
                            out[d] *= by;
                            if constexpr (kWaves == 4) keep(out[d]);
                        }
                    }
                }
                const float to = top == -INFINITY ? 0.0f : top;
                s16x4 probs[kParts];
                float prob[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    prob[i] = hidden[i] ? 0.0f : __builtin_amdgcn_exp2f(fmaf(sc[i], scale, -to));
                if constexpr (BF16) {
                    bf16x4 r;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        r[i] = (__bf16)prob[i];
                        sum += (float)r[i];
                    }
                    probs[0] = __builtin_bit_cast(s16x4, r);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        unsigned part[3];
                        split3(prob[i], part);
#pragma unroll
                        for (int k = 0; k < kParts; ++k) probs[k][i] = (short)part[k];
                        sum += prob[i];
                    }
                }
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    if (!FULL && !FP4 && 32 * j >= latent) continue;
                    const u32x4 v = operand<FP4, FULL>(raw, j, g, latent);
                    s16x4 turned[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const u32x4 x = __builtin_bit_cast(u32x4, mfma32(v, identity[h], f32x4{0.f, 0.f, 0.f, 0.f}));
                        // (the upper halves: bf16 values are exact)
                        const unsigned lo = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
                        const unsigned hi = __builtin_amdgcn_perm(x[3], x[2], 0x07060302u);
                        turned[h] = __builtin_bit_cast(s16x4, (unsigned long)hi << 32 | lo);
                    }
#pragma unroll
                    for (int k = 0; k < kParts; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            out[2 * j + h] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(turned[h], probs[k], out[2 * j + h], 0, 0, 0);
                    if (j % kGroup == kGroup - 1) __builtin_amdgcn_sched_barrier(0);
                }
            }

            // the waves' sums: each to the largest of their maxima, then added
            top = groups_max(top);
            sum += __shfl_xor(sum, 16, kWave);
            sum += __shfl_xor(sum, 32, kWave);
            if (g == 0) {
                tops[c][wave] = top;
                sums[c][wave] = sum;
            }
            const int busy = upto - from < kWaves ? upto - from : kWaves;  // waves that had a step
            const bool whole = first == 0 && last == w.per;
            const int part = 2 * group + (first == 0 ? 1 : 0);
            // a thread's column of the results, 4 values at a time
            constexpr int kColThreads = kThreads / kCols, kPasses = kJoinDims / (4 * kColThreads);
            const int col = tid / kColThreads, at = 4 * (tid % kColThreads);
            float col_top = -INFINITY, col_sum = 0.0f, by[kWaves], over = 0.0f;
            float *results = reinterpret_cast<float *>(lds);
#pragma unroll
            for (int round = 0; round < kLatentMax / kJoinDims; ++round) {
                if (!FULL && round * kJoinDims >= latent) break;
                __syncthreads();  // (the queries, or the last round's results, are read)
                if (wave < busy) {
#pragma unroll
                    for (int d = 0; d < kJoinDims / 16; ++d) {
                        // rows 4 g .. 4 g + 3 of out[2 j + h] are 4 latent values of lane group
                        // 2 h + g / 2 at step j
                        const int at = dim_of<FP4>(d / 2, 2 * (d % 2) + g / 2) + 4 * (g % 2);
                        *reinterpret_cast<f32x4 *>(results + wave * (kJoinBytes / 4) + c * kJoinDims + 4 * ((at / 4) ^ c)) =
                            out[round * (kJoinDims / 16) + d];
                    }
                }
                __syncthreads();
                if (round == 0) {
#pragma unroll
                    for (int x = 0; x < kWaves; ++x) col_top = fmaxf(col_top, tops[col][x]);
#pragma unroll
                    for (int x = 0; x < kWaves; ++x) {
                        by[x] = __builtin_amdgcn_exp2f(tops[col][x] - (col_top == -INFINITY ? 0.0f : col_top));
                        col_sum += by[x] * sums[col][x];
                    }
                    over = whole ? col_sum == 0.0f ? 0.0f : 1.0f / col_sum : 1.0f;
                }
                f32x4 v[kPasses];
#pragma unroll
                for (int k = 0; k < kPasses; ++k) v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < kWaves; ++x) {
                    if (x >= busy) break;
#pragma unroll
                    for (int k = 0; k < kPasses; ++k)
                        v[k] += by[x] * load_f4(results + x * (kJoinBytes / 4) + col * kJoinDims +
                                                4 * ((at / 4 + kColThreads * k) ^ col));
                }
#pragma unroll
                for (int k = 0; k < kPasses; ++k) {
                    const int d = round * kJoinDims + at + 4 * kColThreads * k;
                    if (!FULL && d >= latent) break;
                    if (!whole)
                        *reinterpret_cast<f32x4 *>(p.parts.sums + (part * kCols + col) * kLatentMax + d) = v[k];
                    else if (col < used)
                        store4<BF16>(p.out, (base + col) * latent + d, v[k] * over);
                }
            }
            if (!whole && at == 0) {
                p.parts.stats[part * 2 * kCols + col] = col_top;
                p.parts.stats[(part * 2 + 1) * kCols + col] = col_sum;
            }
            if (t == 0 && last == w.per && (first > 0 || p.parts.tiles)) {
                // (owner: of the tile's first unit)
                const Record record = {s, tile, first > 0 ? run.owner(run.begin - first) : -1, group};
                p.parts.records[p.parts.tiles ? (int)(base / kCols) + s : group] = record;
            }
        }
    }
}

template <bool FP4, bool BF16, bool FULL> int launch(const Params &p, hipStream_t stream) {
    constexpr int kThreads = kWavesOf<FP4> * kWave;
    constexpr int bytes = kLdsBytes<FP4, BF16>;
    const auto kernel = latent_attend_kernel<FP4, BF16, FULL>;
    static const bool ok = allow_lds(kernel, bytes);
    if (!ok) return kErrLaunch;
    kernel<<<p.groups, kThreads, bytes, stream>>>(p);
    if (hipGetLastError() != hipSuccess) return kErrLaunch;
    return launch_join<Narrow, BF16>(p, stream);
}

}  // namespace

// Whether the wide kernel is taken, for bf16 queries of full rows: it reads keys once for 64 columns
// and not for 16, but begins and ends a tile more slowly.  The host knows the pairs, the sequences
// and the keys that a table holds.  Calls in us, wide and narrow, by the pairs of each sequence (16 to
// a row), 3000 .. 4096 keys:
//   bf16 keys   4 sequences of 128 41 and 39, of 256 42 and 53, of 512 49 and 82, of 2048 103 and
//               284; 16 of 48 46 and 50, of 64 49 and 56; 32 of 32 63 and 61, of 64 65 and 98; 64 of
//               64 97 and 177
//   4-bit keys  4 of 128 39 and 29, of 256 40 and 37, of 512 48 and 54, of 2048 99 and 152; 16 of 64
//               44 and 38; 32 of 32 49 and 38, of 64 53 and 54, of 128 69 and 93; 64 of 64 75 and 95
// One sequence of 4096 pairs over 256 keys: bf16 27 and 21, 4 bits 27 and 16; of 8192 pairs over
// 512 keys 37 and 53, 37 and 36.  One of 2048 pairs over 4096 keys beside 63 of 16: bf16 110 and 122,
// 4 bits 88 and 77; one of 8192 beside them 184 and 325, 150 and 189.  So the rule errs by a tenth to a
// fifth near its borders, where one sequence's pairs are far from the average, and by more for prompts
// of few keys whose table is wide: the host does not know lengths.  Queries at 16-byte addresses,
// which it copies so.
static bool wide_pays(const MlkLatentBatch &b, const LatentAttend &p) {
    const long pairs = (long)p.rows * p.heads, few = b.type == MLK_FP4 ? 2 : 1;
    return p.bf16 && b.latent == kLatentMax && b.rope == kLatentRopeMax && (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 &&
           pairs >= 64 * few * b.seqs && pairs >= 1024 * few && (long)b.table_width * b.page_size >= 512;
}

constexpr int kMostKeys = 0x7FFFFF80;  // (a step may begin behind the last one)

size_t latent_attend_workspace() { return kSumsBytes + kStatsBytes + kRecordBytes; }

int latent_attend(const MlkLatentBatch &b, const LatentAttend &p, int cu_count, hipStream_t stream) {
    Params a;
    a.b = b;
    a.q = p.q;
    a.out = p.out;
    a.rows = p.rows;
    a.heads = p.heads;
    a.scale = p.scale * 1.44269504f;
    const bool wide = wide_pays(b, p);
    const int most_groups = wide ? Wide::kGroups : Narrow::kGroups;
    a.groups = cu_count < most_groups ? cu_count : most_groups;
    const long room = (long)b.table_width * b.page_size;
    a.keys = room < kMostKeys ? (int)room : kMostKeys;
    // units of more keys where there could be 2^31 of them (a tile has at least a column; tiles are at
    // most 2^27 + kLatentMaxSeqs)
    const long tiles = (long)p.rows * p.heads / (wide ? Wide::kCols : Narrow::kCols) + b.seqs;
    const int step_shift = wide ? Wide::kStepShift : Narrow::kStepShift;
    a.parts.tiles = tiles <= kMaxTileRecords ? (int)tiles : 0;
    for (a.shift = 0; tiles * (((a.keys - 1) >> (step_shift + a.shift)) + 1) >= 0x7FFFFFFF; ++a.shift) {}
    a.page = Divisor::of((unsigned)b.page_size);
    a.head = Divisor::of((unsigned)p.heads);
    uint8_t *at = static_cast<uint8_t *>(p.workspace);
    a.parts.sums = reinterpret_cast<float *>(at);
    a.parts.stats = reinterpret_cast<float *>(at + kSumsBytes);
    a.parts.records = reinterpret_cast<Record *>(at + kSumsBytes + kStatsBytes);
    if (wide) return launch_wide(b.type == MLK_FP4, a, stream);
    const bool full = b.latent == kLatentMax && b.rope == kLatentRopeMax;
    if (b.type == MLK_FP4)
        return p.bf16 ? (full ? launch<true, true, true>(a, stream) : launch<true, true, false>(a, stream))
                      : (full ? launch<true, false, true>(a, stream) : launch<true, false, false>(a, stream));
    return p.bf16 ? (full ? launch<false, true, true>(a, stream) : launch<false, true, false>(a, stream))
                  : (full ? launch<false, false, true>(a, stream) : launch<false, false, false>(a, stream));
}

}  // namespace mlh
