// latent_attend.hip -- attention of a batch's token rows over a paged latent cache
// (gfx950, wave64).
//
//   s_j = scale * q . [latent_j | rope_j],  out = sum_j exp(s_j - m) latent_j / sum_j exp(s_j - m)
//
// for each (token row, head); a sequence's (row, head) pairs are taken 16 at a time
// (a tile: the 16 columns of a matrix instruction), and a tile's keys a unit at a time,
// 16 for each wave of a workgroup.  The units of all tiles, in order, are dealt out in
// equal runs to as many workgroups as the chip holds, so ragged lengths leave none of them
// idle; a tile whose units fell to several is joined by latent_join_kernel from their
// partial sums.
//
// Each wave takes 16 of a unit's keys, with a running maximum and sum of its own, and the
// waves meet at the end of a tile.  The keys are read straight into the matrix operand
// (lane (k, g): 8 values of key k at a step), so the scores S[key][column] come from
// v_mfma_f32_16x16x32_bf16; their registers hold 4 keys of a column, which is the operand
// layout of the second product O[latent][column] += V^T P on v_mfma_f32_16x16x16_bf16.
// V^T, the same keys with the latent index across lanes, goes through a piece of LDS of
// the wave's own, written in rows and read transposed (ds_read_b64_tr_b16).  The next
// keys are on their way from when the first product has taken the present ones, and the
// page numbers of those after them.
#include "bf16.h"
#include "latent.h"
#include "mlh_device.h"
#include "mlh_host.h"

namespace mlh {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

constexpr int kCols = 16;       // (row, head) pairs of a tile
constexpr int kTileKeys = 16;   // keys of a wave's step
constexpr int kSteps = kLatentMax / 32;          // product steps over a latent row
constexpr int kRopeSteps = kLatentRopeMax / 32;  // and over a rope row
constexpr int kAllSteps = kSteps + kRopeSteps;
constexpr int kDims = kLatentMax / 16;           // 16-value tiles of a latent row
constexpr int kMaxGroups = 512;                  // workgroups of a launch

// Waves of a workgroup, one workgroup a CU: with bf16 queries in LDS (18 KB) beside 17 KB of
// keys for each wave there is room for two waves on a SIMD, one's loads under the other's
// products; f32 queries take three bf16 parts (55 KB).
template <bool BF16> constexpr int kWavesOf = BF16 ? 8 : 4;
template <bool BF16> constexpr int kAheadOf = BF16 ? 2 : 3;  // steps that queries are read ahead

// A wave's keys in LDS: rows 32 bytes apart from a multiple of the banks, so that neither
// the rows of a transposed read nor those of a write share them.
constexpr int kKeyStride = 2 * kLatentMax + 32;
constexpr int kKeyBytes = kTileKeys * kKeyStride;
// The waves' results in LDS, kJoinDims latent values of each column at a time.
constexpr int kJoinDims = 256;
constexpr int kJoinStride = kJoinDims + 4;
static_assert(kCols * kJoinStride * 4 <= kKeyBytes, "the results fit where the keys were");
constexpr int kQueryStride = kLatentMax + kLatentRopeMax + 8;
template <bool BF16> constexpr int kQueryBytes = (BF16 ? 1 : 3) * kCols * kQueryStride * 2;

// Partial sums of tiles: slot 2w holds the tile that workgroup w found begun, slot 2w + 1
// the one that it left unfinished.
struct Parts {
    float *sums;    // [2 groups][kCols][kLatentMax]
    float *stats;   // [2 groups][2][kCols] maxima, then sums
    int *records;   // [groups][kRecord]
};
// Of a workgroup's first tile, if it was begun by another one and ends here: sequence,
// tile, first workgroup; else -1.
constexpr int kRecord = 4;

constexpr size_t kSumsBytes = 2L * kMaxGroups * kCols * kLatentMax * 4;
constexpr size_t kStatsBytes = 2L * kMaxGroups * 2 * kCols * 4;
constexpr size_t kRecordBytes = (size_t)kMaxGroups * kRecord * 4;

struct Params {
    MlkLatentBatch b;
    const void *q;
    void *out;
    int rows, heads;
    float scale;  // times log2(e)
    int groups;
    Parts parts;
};

// A sequence's work.
struct Work {
    LatentSeq seq;
    int keys;    // that its table can hold
    int per;     // units of a tile
    int tiles;
    __device__ __forceinline__ long units() const { return (long)per * tiles; }
};

template <int UNIT> __device__ __forceinline__ Work work_of(const Params &p, int s) {
    Work w;
    w.seq = latent_seq(p.b, s, p.rows);
    const long room = (long)p.b.table_width * p.b.page_size;
    const int length = w.seq.length < 0 ? 0 : w.seq.length;
    w.keys = length < room ? length : (int)room;
    w.per = w.keys > UNIT ? (w.keys - 1) / UNIT + 1 : 1;
    // (rows * heads is below 2^31 - 15)
    w.tiles = (int)(((unsigned)w.seq.count * (unsigned)p.heads + (kCols - 1)) / kCols);
    return w;
}

// a / b, in 32 bits where both fit: a quarter of the instructions.
__device__ __forceinline__ long quotient(long a, long b) {
    if (((unsigned long)a | (unsigned long)b) >> 32) return a / b;
    return (unsigned)a / (unsigned)b;
}

__device__ __forceinline__ long wave_sum_long(long v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// A workgroup's run of units: `length` of them from the one that is `offset` after the first
// of sequence `seq`; `begin` is that one's place among all.
struct Run {
    int seq;
    long offset, begin, length, total;
    int groups;   // workgroups that have one: of `share` units, the first `rest` of one more
    long share;
    int rest;
    __device__ __forceinline__ int owner(long unit) const {
        const long longer = (share + 1) * rest;
        return (int)(unit < longer ? quotient(unit, share + 1) : rest + quotient(unit - longer, share));
    }
};

template <int WAVES> __device__ __forceinline__ Run find_run(const Params &p, int group) {
    constexpr int kThreads = WAVES * kWave, kUnit = WAVES * kTileKeys;
    __shared__ long sums[WAVES];
    __shared__ long at[2];
    const int t = threadIdx.x, wave = t / kWave, lane = t % kWave;
    const auto units_of = [&](int s) { return s < p.b.seqs ? work_of<kUnit>(p, s).units() : 0L; };
    const long first_units = units_of(t);
    long mine = first_units;
    for (int s = t + kThreads; s < p.b.seqs; s += kThreads) mine += units_of(s);
    mine = wave_sum_long(mine);
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    Run r;
    r.total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) r.total += sums[w];
    // (no workgroup's run is empty between those of a tile)
    r.groups = r.total < p.groups ? (int)r.total : p.groups;
    r.seq = 0;
    r.offset = r.begin = r.length = r.share = 0;
    r.rest = 0;
    if (group >= r.groups) return r;
    r.share = quotient(r.total, r.groups);
    r.rest = (int)(r.total - r.share * r.groups);
    r.begin = r.share * group + (group < r.rest ? group : r.rest);
    r.length = r.share + (group < r.rest ? 1 : 0);
    long before = 0;
    for (int s0 = 0; s0 < p.b.seqs; s0 += kThreads) {
        const long units = s0 == 0 ? first_units : units_of(s0 + t);
        long upto = units;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const long below = __shfl_up(upto, o, kWave);
            if (lane >= o) upto += below;
        }
        __syncthreads();
        if (lane == kWave - 1) sums[wave] = upto;
        __syncthreads();
        long first = before + upto - units;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w < wave) first += sums[w];
            before += sums[w];
        }
        if (r.begin >= first && r.begin < first + units) {
            at[0] = s0 + t;
            at[1] = r.begin - first;
        }
        if (r.begin < before) break;
    }
    __syncthreads();
    r.seq = (int)at[0];
    r.offset = at[1];
    return r;
}

// Product step st, lane group g: the first of the 8 values that a lane holds.  Codes are
// taken 32 at a time, one scale, so four steps go over 128 values.
template <bool FP4> __device__ __forceinline__ int dim_of(int st, int g) {
    if (FP4 && st < kSteps) return 128 * (st / 4) + 32 * g + 8 * (st % 4);
    return 32 * st + 8 * g;
}

// A lane's share of a key as it is read.
template <bool FP4> struct Raw;
template <> struct Raw<false> {
    u32x4 v[kAllSteps];
};
template <> struct Raw<true> {
    u32x4 codes[kSteps / 4];
    unsigned scales;
    u32x4 rope[kRopeSteps];
};

template <bool FP4, bool FULL>
__device__ __forceinline__ void load_key(Raw<FP4> &raw, const uint8_t *row, int g, int latent, int rope) {
    const u32x4 none = {0, 0, 0, 0};
    if constexpr (FP4) {
#pragma unroll
        for (int j = 0; j < kSteps / 4; ++j) {
            const bool in = FULL || 128 * j + 32 * g < latent;
            raw.codes[j] = in ? load_global16(row + 64 * j + 16 * g) : none;
        }
        raw.scales = *(const __attribute__((address_space(1))) unsigned *)(row + latent / 2 + 4 * g);
        const uint8_t *tail = row + latent_part_bytes(true, latent);
#pragma unroll
        for (int j = 0; j < kRopeSteps; ++j) {
            const bool in = FULL || 32 * j + 8 * g < rope;
            raw.rope[j] = in ? load_global16(tail + 64 * j + 16 * g) : none;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kAllSteps; ++j) {
            // (steps past the latent row are the rope's)
            const int at = j < kSteps ? 32 * j + 8 * g : 32 * (j - kSteps) + 8 * g;
            const bool in = FULL || at < (j < kSteps ? latent : rope);
            raw.v[j] = in ? load_global16(row + 2 * (j < kSteps ? at : latent + at)) : none;
        }
    }
}

// Its 8 values at step j.
template <bool FP4, bool FULL>
__device__ __forceinline__ u32x4 operand(const Raw<FP4> &raw, int j, int g, int latent) {
    if constexpr (FP4) {
        if (j >= kSteps) return raw.rope[j - kSteps];
        const bool in = FULL || 128 * (j / 4) + 32 * g < latent;
        const float scale = __uint_as_float(in ? (raw.scales >> (8 * (j / 4)) & 0xFFu) << 23 : 0x3F800000u);
        const unsigned codes = raw.codes[j / 4][j % 4];
        u32x4 v;
        v[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
        v[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
        v[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
        v[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
        return v;
    } else {
        return raw.v[j];
    }
}

__device__ __forceinline__ bool not_finite(const u32x4 &v) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        bad |= (v[i] & 0x7F80u) == 0x7F80u || (v[i] & 0x7F800000u) == 0x7F800000u;
    return bad;
}

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

// Results of one column, 4 values of it.
template <bool BF16> __device__ __forceinline__ void store4(void *out, long at, f32x4 v) {
    typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
    typedef f32x4 f32x4_any __attribute__((aligned(4)));
    if constexpr (BF16)
        *reinterpret_cast<u32x2_any *>(static_cast<uint16_t *>(out) + at) =
            u32x2_any{bf16_bits(v[0]) | bf16_bits(v[1]) << 16, bf16_bits(v[2]) | bf16_bits(v[3]) << 16};
    else *reinterpret_cast<f32x4_any *>(static_cast<float *>(out) + at) = v;
}

// The reference that exponents are taken to moves up only when a score is this far above
// it (in powers of 2): p stays below 2^8 and sums lose nothing by that, and most steps need
// neither the maximum over the lane groups nor to scale what is summed.
constexpr float kSlack = 8.0f;

template <bool FP4, bool BF16, bool FULL>
__global__ __launch_bounds__(kWavesOf<BF16> *kWave, 1) void latent_attend_kernel(Params p) {
    constexpr int kWaves = kWavesOf<BF16>, kThreads = kWaves * kWave, kUnit = kWaves * kTileKeys;
    constexpr int kParts = BF16 ? 1 : 3;  // bf16 parts of a query value and of a probability
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float tops[kWaves][kCols], sums[kWaves][kCols];
    const int t = threadIdx.x, wave = t / kWave, lane = t % kWave;
    const int g = lane / 16, c = lane % 16;
    const int latent = FULL ? kLatentMax : p.b.latent, rope = FULL ? kLatentRopeMax : p.b.rope;
    const int width = latent + rope, dims = latent / 16;
    const int row_bytes = latent_row_bytes(FP4, latent, rope);
    const uint8_t *data = static_cast<const uint8_t *>(p.b.data);
    uint8_t *keys_lds = lds + wave * kKeyBytes;
    uint16_t *query_lds = reinterpret_cast<uint16_t *>(lds + kWaves * kKeyBytes);

    const int group = blockIdx.x;
    const Run run = find_run<kWaves>(p, group);
    int *record = p.parts.records + kRecord * group;
    if (t == 0) record[0] = -1;
    long left = run.length, offset = run.offset;
    for (int s = run.seq; left > 0 && s < p.b.seqs; ++s, offset = 0) {
        const Work w = work_of<kUnit>(p, s);
        while (left > 0 && offset < w.units()) {
            const int tile = (int)quotient(offset, w.per), from = (int)(offset - (long)tile * w.per);
            const int upto = left < w.per - from ? from + (int)left : w.per;
            left -= upto - from;
            offset += upto - from;

            // the tile's columns, and the keys that they see, as far as the table goes
            const unsigned pair0 = (unsigned)tile * kCols, pairs = (unsigned)w.seq.count * (unsigned)p.heads;
            const int used = pairs - pair0 < kCols ? (int)(pairs - pair0) : kCols;
            const long base = (long)w.seq.begin * p.heads + pair0;  // among all (row, head) pairs
            const long sees = (long)w.seq.length - w.seq.count + 1 + (pair0 + (c < used ? c : 0)) / (unsigned)p.heads;
            const int within = sees < 0 ? 0 : sees < w.keys ? (int)sees : w.keys;
            const int limit = c < used ? within : 0;
            const int least = __builtin_amdgcn_readlane(within, 0);
            const int most = __builtin_amdgcn_readlane(within, used - 1);

            // the wave's first keys, and the pages of its second ones
            const auto key_of = [&](int unit) { return unit * kUnit + wave * kTileKeys + c; };
            const auto slot_of = [&](int unit) {
                const int j = key_of(unit);
                return unit < upto && j < most ? latent_slot(p.b, s, (unsigned)j) : 0L;
            };
            long slot = slot_of(from);
            Raw<FP4> raw;
            load_key<FP4, FULL>(raw, data + (slot < 0 ? 0 : slot) * row_bytes, g, latent, rope);
            long next_slot = slot_of(from + 1);

            // the queries, 8 values a thread and pass, into LDS
            __syncthreads();  // (the tile before is done with it)
#pragma unroll 1
            for (int i = t; i < kCols * (kLatentMax + kLatentRopeMax) / 8; i += kThreads) {
                constexpr int kPieces = (kLatentMax + kLatentRopeMax) / 8;
                const int col = i / kPieces, d = 8 * (i % kPieces);
                const bool in = col < used && (FULL || (d < kLatentMax ? d < latent : d - kLatentMax < rope));
                const long at = (base + (in ? col : 0)) * width + (!in ? 0 : d < kLatentMax ? d : latent + d - kLatentMax);
                if constexpr (BF16) {
                    u32x4 v = *reinterpret_cast<const u32x4_any *>(static_cast<const uint16_t *>(p.q) + at);
                    if (!in) v = u32x4{0, 0, 0, 0};
                    *reinterpret_cast<u32x4 *>(query_lds + col * kQueryStride + d) = v;
                } else {
                    float x[8];
                    __builtin_memcpy(x, static_cast<const float *>(p.q) + at, sizeof(x));
                    u32x4 v[3];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        unsigned lo[3], hi[3];
                        split3(in ? x[2 * k] : 0.0f, lo);
                        split3(in ? x[2 * k + 1] : 0.0f, hi);
#pragma unroll
                        for (int y = 0; y < 3; ++y) v[y][k] = lo[y] | hi[y] << 16;
                    }
#pragma unroll
                    for (int y = 0; y < 3; ++y)
                        *reinterpret_cast<u32x4 *>(query_lds + (y * kCols + col) * kQueryStride + d) = v[y];
                }
            }
            __syncthreads();

            // Running softmax: lane (c, g) holds column c, its sum over keys 4 g .. 4 g + 3 of
            // every step; a row that sees keys behind its table is NaN.
            float top = -INFINITY, sum = c < used && sees > w.keys ? NAN : 0.0f;
            f32x4 out[kDims];
#pragma unroll
            for (int d = 0; d < kDims; ++d) out[d] = f32x4{0.f, 0.f, 0.f, 0.f};

            for (int unit = from; unit < upto; ++unit) {
                const int key0 = unit * kUnit + wave * kTileKeys;
                if (key0 >= most) break;
                unsigned bad = (unsigned)__ballot(slot < 0) & 0xFFFFu;  // keys without a place
                f32x4 score[kParts];
#pragma unroll
                for (int k = 0; k < kParts; ++k) score[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                // (queries come from LDS a few steps ahead of their product, and no more:
                // registers are what limits a wave here)
                constexpr int kAhead = kAheadOf<BF16>;
                u32x4 ahead[2][kAhead][kParts];
                const auto fetch = [&](int j0) {
#pragma unroll
                    for (int x = 0; x < kAhead; ++x) {
                        const int j = j0 + x;
                        const int at = j < kSteps ? dim_of<FP4>(j, g) : kLatentMax + 32 * (j - kSteps) + 8 * g;
#pragma unroll
                        for (int k = 0; k < kParts; ++k)
                            ahead[j0 / kAhead % 2][x][k] =
                                *reinterpret_cast<const u32x4 *>(query_lds + (k * kCols + c) * kQueryStride + at);
                    }
                };
                fetch(0);
#pragma unroll
                for (int j0 = 0; j0 < kAllSteps; j0 += kAhead) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (j0 + kAhead < kAllSteps) fetch(j0 + kAhead);
#pragma unroll
                    for (int x = 0; x < kAhead; ++x) {
                        const int j = j0 + x;
                        const u32x4 v = operand<FP4, FULL>(raw, j, g, latent);
                        if (j < kSteps)
                            *reinterpret_cast<u32x4 *>(keys_lds + c * kKeyStride + 2 * dim_of<FP4>(j, g)) = v;
#pragma unroll
                        for (int k = 0; k < kParts; ++k) score[k] = mfma32(v, ahead[j0 / kAhead % 2][x][k], score[k]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                slot = next_slot;
                if (unit + 1 < upto)
                    load_key<FP4, FULL>(raw, data + (slot < 0 ? 0 : slot) * row_bytes, g, latent, rope);
                next_slot = slot_of(unit + 2);
                f32x4 sc = score[0];
                if constexpr (!BF16) sc += score[1] + score[2];

                const bool edge = bad || key0 + kTileKeys > least;
                bool hidden[4] = {false, false, false, false};
                if (edge) {
                    // Keys that not every column sees, or that have no place: those that a
                    // column does not see must not reach it by 0 * NaN either, so rows that
                    // are not finite (or not there) are taken out of the second product and
                    // make NaN of the scores of the columns that see them.
                    const bool there = key0 + c < most;
                    bool odd = false;
#pragma unroll 1
                    for (int j = 0; j < kSteps; ++j)
                        odd |= not_finite(*reinterpret_cast<const u32x4 *>(keys_lds + c * kKeyStride + 2 * dim_of<FP4>(j, g)));
                    const unsigned long long which = __ballot(odd && there);
                    bad |= (unsigned)(which | which >> 16 | which >> 32 | which >> 48) & 0xFFFFu;
                    if (!there || (bad >> c & 1u)) {
#pragma unroll 1
                        for (int j = 0; j < kSteps; ++j)
                            *reinterpret_cast<u32x4 *>(keys_lds + c * kKeyStride + 2 * dim_of<FP4>(j, g)) = u32x4{0, 0, 0, 0};
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (bad >> (4 * g + i) & 1u) sc[i] = NAN;
                        hidden[i] = key0 + 4 * g + i >= limit;
                    }
                }
                float high = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = hidden[i] ? -INFINITY : sc[i] * p.scale;
                    high = fmaxf(high, x);
                }
                if (__any(high > top + kSlack)) {
                    const float next = fmaxf(top, groups_max(high));
                    const float by = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next);
                    sum *= by;
                    top = next;
#pragma unroll
                    for (int d = 0; d < kDims; ++d) out[d] *= by;
                }
                const float to = top == -INFINITY ? 0.0f : top;
                s16x4 probs[kParts];
                float prob[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    prob[i] = hidden[i] ? 0.0f : __builtin_amdgcn_exp2f(fmaf(sc[i], p.scale, -to));
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
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                const uint8_t *from_lds = keys_lds + (4 * g + c / 4) * kKeyStride + 8 * (c % 4);
                constexpr int kRead = BF16 ? 4 : 8;
                s16x4 turned[2][kRead];
                const auto read = [&](int d0) {
#pragma unroll
                    for (int x = 0; x < kRead; ++x)
                        turned[d0 / kRead % 2][x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4 *)(from_lds + 32 * (d0 + x)));
                };
                read(0);
#pragma unroll
                for (int d0 = 0; d0 < kDims; d0 += kRead) {
                    if (!FULL && d0 >= dims) break;
                    __builtin_amdgcn_sched_barrier(0);
                    if (d0 + kRead < kDims) read(d0 + kRead);
#pragma unroll
                    for (int x = 0; x < kRead; ++x)
#pragma unroll
                        for (int k = 0; k < kParts; ++k)
                            out[d0 + x] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(turned[d0 / kRead % 2][x], probs[k],
                                                                                   out[d0 + x], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }

            // the waves' sums: each to the largest of their maxima, then added
            top = groups_max(top);
            sum += __shfl_xor(sum, 16, kWave);
            sum += __shfl_xor(sum, 32, kWave);
            if (g == 0) {
                tops[wave][c] = top;
                sums[wave][c] = sum;
            }
            __syncthreads();
            float all = tops[0][c];
#pragma unroll
            for (int k = 1; k < kWaves; ++k) all = fmaxf(all, tops[k][c]);
            const float by = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - all);
            const bool whole = from == 0 && upto == w.per;
            const int part = 2 * group + (from == 0 ? 1 : 0);
            // a thread's column of the results, 4 values at a time
            constexpr int kColThreads = kThreads / kCols;
            const int col = t / kColThreads;
            float col_top = tops[0][col], col_sum = 0.0f;
#pragma unroll
            for (int k = 1; k < kWaves; ++k) col_top = fmaxf(col_top, tops[k][col]);
#pragma unroll
            for (int k = 0; k < kWaves; ++k)
                col_sum += sums[k][col] * (tops[k][col] == -INFINITY
                                               ? 0.0f  // (times 0, or NaN where a column is)
                                               : __builtin_amdgcn_exp2f(tops[k][col] - col_top));
            const float over = col_top == -INFINITY && !(col_sum != col_sum) ? 0.0f : 1.0f / col_sum;
            float *results = reinterpret_cast<float *>(lds);
#pragma unroll
            for (int round = 0; round < kLatentMax / kJoinDims; ++round) {
                if (!FULL && round * kJoinDims >= latent) break;
                if (round) __syncthreads();
#pragma unroll
                for (int d = 0; d < kJoinDims / 16; ++d)
                    *reinterpret_cast<f32x4 *>(results + (wave * kCols + c) * kJoinStride + 16 * d + 4 * g) =
                        out[round * (kJoinDims / 16) + d] * by;
                __syncthreads();
#pragma unroll
                for (int k = 0; k < kJoinDims / (4 * kColThreads); ++k) {
                    const int at = 4 * (t % kColThreads) + 4 * kColThreads * k, d = round * kJoinDims + at;
                    if (!FULL && d >= latent) break;
                    f32x4 v = load_f4(results + col * kJoinStride + at);
#pragma unroll
                    for (int x = 1; x < kWaves; ++x) v += load_f4(results + (x * kCols + col) * kJoinStride + at);
                    if (!whole)
                        *reinterpret_cast<f32x4 *>(p.parts.sums + ((long)part * kCols + col) * kLatentMax + d) = v;
                    else if (col < used)
                        store4<BF16>(p.out, (base + col) * latent + d, v * over);
                }
            }
            if (!whole && t % kColThreads == 0) {
                p.parts.stats[(long)part * 2 * kCols + col] = col_top;
                p.parts.stats[((long)part * 2 + 1) * kCols + col] = col_sum;
            }
            if (t == 0 && from > 0 && upto == w.per) {
                // the workgroup whose run holds the tile's first unit
                record[1] = tile;
                record[2] = run.owner(run.begin - from);
                record[0] = s;
            }
            __syncthreads();
        }
    }
}

// Joins the tile that workgroup blockIdx.x finished but did not begin: its sums are in part
// 2 first + 1 and in parts 2w of the workgroups w after the first.  A workgroup of this
// launch takes kJoinCols columns, 128 threads each.
constexpr int kJoinCols = 2, kColThreads = kLatentMax / 4;
template <bool BF16> __global__ __launch_bounds__(kJoinCols *kColThreads) void latent_join_kernel(Params p) {
    __shared__ float weights[kJoinCols][kMaxGroups];
    __shared__ float reds[kJoinCols][2][kColThreads / kWave];
    const int group = blockIdx.x, x = threadIdx.x / kColThreads, t = threadIdx.x % kColThreads;
    const int col = blockIdx.y * kJoinCols + x;
    const int *record = p.parts.records + kRecord * group;
    const int s = record[0], tile = record[1], first = record[2];
    if (s < 0) return;
    const LatentSeq seq = latent_seq(p.b, s, p.rows);
    const int count = group - first + 1;
    const auto part_of = [&](int i) { return i == 0 ? 2L * first + 1 : 2L * (first + i); };
    float top = -INFINITY;
    for (int i = t; i < count; i += kColThreads) {
        const float its = p.parts.stats[part_of(i) * 2 * kCols + col];
        weights[x][i] = its;
        top = fmaxf(top, its);
    }
    top = wave_max(top);
    if (t % kWave == 0) reds[x][0][t / kWave] = top;
    __syncthreads();
    top = fmaxf(reds[x][0][0], reds[x][0][1]);
    float sum = 0.0f;
    for (int i = t; i < count; i += kColThreads) {
        const float its = weights[x][i];
        const float by = its == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(its - top);
        sum += by * p.parts.stats[(part_of(i) * 2 + 1) * kCols + col];
        weights[x][i] = by;
    }
    sum = wave_sum(sum);
    if (t % kWave == 0) reds[x][1][t / kWave] = sum;
    __syncthreads();
    sum = reds[x][1][0] + reds[x][1][1];
    const unsigned pair = (unsigned)tile * kCols + col;
    if (pair >= (unsigned)seq.count * (unsigned)p.heads || 4 * t >= p.b.latent) return;
    const float *from = p.parts.sums + (long)col * kLatentMax + 4 * t;
    f32x4 v = weights[x][0] * load_f4(from + part_of(0) * kCols * kLatentMax);
    from += part_of(1) * kCols * kLatentMax;
#pragma unroll 8
    for (int i = 1; i < count; ++i) v += weights[x][i] * load_f4(from + (long)(i - 1) * 2 * kCols * kLatentMax);
    v *= top == -INFINITY && !(sum != sum) ? 0.0f : 1.0f / sum;
    store4<BF16>(p.out, ((long)seq.begin * p.heads + pair) * p.b.latent + 4 * t, v);
}

template <bool FP4, bool BF16, bool FULL> int launch(const Params &p, hipStream_t stream) {
    constexpr int threads = kWavesOf<BF16> * kWave;
    constexpr int bytes = kWavesOf<BF16> * kKeyBytes + kQueryBytes<BF16>;
    const auto kernel = latent_attend_kernel<FP4, BF16, FULL>;
    static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
    if (!ok) return kErrLaunch;
    kernel<<<p.groups, threads, bytes, stream>>>(p);
    if (hipGetLastError() != hipSuccess) return kErrLaunch;
    if (p.groups == 1) return kOk;
    latent_join_kernel<BF16><<<dim3(p.groups, kCols / kJoinCols), kJoinCols * kColThreads, 0, stream>>>(p);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace

size_t latent_attend_workspace() { return kSumsBytes + kStatsBytes + kRecordBytes; }

int latent_attend(const MlkLatentBatch &b, const LatentAttend &p, int cu_count, hipStream_t stream) {
    Params a;
    a.b = b;
    a.q = p.q;
    a.out = p.out;
    a.rows = p.rows;
    a.heads = p.heads;
    a.scale = p.scale * 1.44269504f;
    a.groups = cu_count < kMaxGroups ? cu_count : kMaxGroups;
    uint8_t *at = static_cast<uint8_t *>(p.workspace);
    a.parts.sums = reinterpret_cast<float *>(at);
    a.parts.stats = reinterpret_cast<float *>(at + kSumsBytes);
    a.parts.records = reinterpret_cast<int *>(at + kSumsBytes + kStatsBytes);
    const bool full = b.latent == kLatentMax && b.rope == kLatentRopeMax;
    if (b.type == MLK_FP4)
        return p.bf16 ? (full ? launch<true, true, true>(a, stream) : launch<true, true, false>(a, stream))
                      : (full ? launch<true, false, true>(a, stream) : launch<true, false, false>(a, stream));
    return p.bf16 ? (full ? launch<false, true, true>(a, stream) : launch<false, true, false>(a, stream))
                  : (full ? launch<false, false, true>(a, stream) : launch<false, false, false>(a, stream));
}

}  // namespace mlh
