// latent_attend.hip -- attention of a batch's token rows over a paged latent cache
// (gfx950, wave64).
//
//   s_j = scale * q . [latent_j | rope_j],  out = sum_j exp(s_j - m) latent_j / sum_j exp(s_j - m)
//
// for each (token row, head); a sequence's (row, head) pairs are taken 16 at a time
// (a tile: the 16 columns of a matrix instruction), and a tile's keys 64 at a time (a
// unit).  The units of all tiles, in order, are dealt out in equal runs to as many
// workgroups as the chip holds, so ragged lengths leave none of them idle; a tile whose
// units fell to several is joined by latent_join_kernel from their partial sums.
//
// In a workgroup each of the 4 waves takes 16 of a unit's 64 keys, with a running maximum
// and sum of its own, and the four meet at the end of a tile.  The keys are read straight
// into the matrix operand (lane (k, g): 8 values of key k at a step), so the scores
// S[key][column] come from v_mfma_f32_16x16x32_bf16; their registers hold 4 keys of a
// column, which is the operand layout of the second product O[latent][column] += V^T P on
// v_mfma_f32_16x16x16_bf16.  V^T, the same keys with the latent index across lanes, goes
// through a piece of LDS of the wave's own, written in rows and read transposed
// (ds_read_b64_tr_b16).
#include "bf16.h"
#include "latent.h"
#include "mlh_device.h"
#include "mlh_host.h"

namespace mlh {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kCols = 16;       // (row, head) pairs of a tile
constexpr int kTileKeys = 16;   // keys of a wave's step
constexpr int kUnitKeys = kWaves * kTileKeys;
constexpr int kSteps = kLatentMax / 32;          // product steps over a latent row
constexpr int kRopeSteps = kLatentRopeMax / 32;  // and over a rope row
constexpr int kDims = kLatentMax / 16;           // 16-value tiles of a latent row
constexpr int kMaxGroups = 512;                  // workgroups of a launch

// A wave's keys in LDS: rows 32 bytes apart from a multiple of the banks, so that neither
// the rows of a transposed read nor those of a write share them.
constexpr int kKeyStride = 2 * kLatentMax + 32;
constexpr int kKeyBytes = kTileKeys * kKeyStride;
// The waves' results in LDS, kJoinDims latent values of each column at a time.
constexpr int kJoinDims = 256;
constexpr int kJoinStride = kJoinDims + 4;
static_assert(kWaves * kCols * kJoinStride * 4 <= kWaves * kKeyBytes, "the results fit where the keys were");
// f32 queries in LDS, as three bf16 parts.
constexpr int kQueryStride = kLatentMax + kLatentRopeMax + 8;
constexpr int kQueryBytes = 3 * kCols * kQueryStride * 2;

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

__device__ __forceinline__ Work work_of(const Params &p, int s) {
    Work w;
    w.seq = latent_seq(p.b, s, p.rows);
    const long room = (long)p.b.table_width * p.b.page_size;
    const int length = w.seq.length < 0 ? 0 : w.seq.length;
    w.keys = length < room ? length : (int)room;
    w.per = w.keys > kUnitKeys ? (w.keys - 1) / kUnitKeys + 1 : 1;
    w.tiles = (int)(((long)w.seq.count * p.heads + kCols - 1) / kCols);
    return w;
}

__device__ __forceinline__ long wave_sum_long(long v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// Where a workgroup's run of units begins, and its length.
struct Run {
    int seq;      // the sequence that holds its first unit
    long offset;  // that unit's place among the sequence's
    long begin, end, total;
    int groups;   // workgroups that have one
};

__device__ __forceinline__ Run find_run(const Params &p, int group) {
    __shared__ long sums[kWaves];
    __shared__ long at[2];
    const int t = threadIdx.x, wave = t / kWave, lane = t % kWave;
    long mine = 0;
    for (int s = t; s < p.b.seqs; s += kThreads) mine += work_of(p, s).units();
    mine = wave_sum_long(mine);
    if (lane == 0) sums[wave] = mine;
    __syncthreads();
    Run r;
    r.total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    // (no workgroup's run is empty between those of a tile)
    r.groups = r.total < p.groups ? (int)r.total : p.groups;
    r.begin = r.end = 0;
    r.seq = 0;
    r.offset = 0;
    if (group >= r.groups) return r;
    r.begin = r.total * group / r.groups;
    r.end = r.total * (group + 1) / r.groups;
    long before = 0;
    for (int s0 = 0; s0 < p.b.seqs; s0 += kThreads) {
        const int s = s0 + t;
        const long units = s < p.b.seqs ? work_of(p, s).units() : 0;
        long upto = units;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const long below = __shfl_up(upto, o, kWave);
            if (lane >= o) upto += below;
        }
        __syncthreads();
        if (lane == kWave - 1) sums[wave] = upto;
        __syncthreads();
        long first = before;
        for (int w = 0; w < wave; ++w) first += sums[w];
        first += upto - units;
        if (r.begin >= first && r.begin < first + units) {
            at[0] = s;
            at[1] = r.begin - first;
        }
        before += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (r.begin < before) break;
    }
    __syncthreads();
    r.seq = (int)at[0];
    r.offset = at[1];
    __syncthreads();
    return r;
}

// Product step st, lane group g: the first of the 8 values that a lane holds.  Codes are
// taken 32 at a time, one scale, so four steps go over 128 values.
template <bool FP4> __device__ __forceinline__ int dim_of(int st, int g) {
    if (FP4 && st < kSteps) return 128 * (st / 4) + 32 * g + 8 * (st % 4);
    return 32 * st + 8 * g;
}

// One key as it is read, by the lane group's share, and as product operands.
template <bool FP4> struct Raw;
template <> struct Raw<false> {
    u32x4 v[kSteps + kRopeSteps];
};
template <> struct Raw<true> {
    u32x4 codes[kSteps / 4];
    unsigned scales;
    u32x4 rope[kRopeSteps];
};
struct Key {
    u32x4 v[kSteps + kRopeSteps];
};

template <bool FP4, bool FULL>
__device__ __forceinline__ void load_key(Raw<FP4> &raw, const uint8_t *row, int g, int latent, int rope) {
    const u32x4 none = {0, 0, 0, 0};
    if constexpr (FP4) {
#pragma unroll
        for (int j = 0; j < kSteps / 4; ++j) {
            const bool in = FULL || 128 * j + 32 * g < latent;
            raw.codes[j] = in ? *reinterpret_cast<const u32x4 *>(row + 64 * j + 16 * g) : none;
        }
        raw.scales = *reinterpret_cast<const unsigned *>(row + latent / 2 + 4 * g);
        const uint8_t *tail = row + latent_part_bytes(true, latent);
#pragma unroll
        for (int j = 0; j < kRopeSteps; ++j) {
            const bool in = FULL || 32 * j + 8 * g < rope;
            raw.rope[j] = in ? *reinterpret_cast<const u32x4 *>(tail + 64 * j + 16 * g) : none;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kSteps + kRopeSteps; ++j) {
            // (steps past the latent row are the rope's)
            const int at = j < kSteps ? 32 * j + 8 * g : 32 * (j - kSteps) + 8 * g;
            const bool in = FULL || at < (j < kSteps ? latent : rope);
            const uint8_t *from = row + 2 * (j < kSteps ? at : latent + at);
            raw.v[j] = in ? *reinterpret_cast<const u32x4 *>(from) : none;
        }
    }
}

template <bool FP4, bool FULL>
__device__ __forceinline__ void to_key(Key &key, const Raw<FP4> &raw, int g, int latent) {
    if constexpr (FP4) {
#pragma unroll
        for (int j = 0; j < kSteps / 4; ++j) {
            const bool in = FULL || 128 * j + 32 * g < latent;
            const float scale =
                __uint_as_float(in ? (raw.scales >> (8 * j) & 0xFFu) << 23 : 0x3F800000u);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned codes = raw.codes[j][w];
                const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
                const auto p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
                const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
                const auto p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
                u32x4 v;
                v[0] = __builtin_bit_cast(unsigned, p0);
                v[1] = __builtin_bit_cast(unsigned, p1);
                v[2] = __builtin_bit_cast(unsigned, p2);
                v[3] = __builtin_bit_cast(unsigned, p3);
                key.v[4 * j + w] = v;
            }
        }
#pragma unroll
        for (int j = 0; j < kRopeSteps; ++j) key.v[kSteps + j] = raw.rope[j];
    } else {
#pragma unroll
        for (int j = 0; j < kSteps + kRopeSteps; ++j) key.v[j] = raw.v[j];
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

// Running softmax of a wave's keys: lane (c, g) holds column c, its sums over keys
// 4 g .. 4 g + 3 of every step.
struct Soft {
    float top;  // in units of log2
    float sum;
};

template <bool FP4, bool BF16, bool FULL>
__global__ __launch_bounds__(kThreads, 1) void latent_attend_kernel(Params p) {
    constexpr int kParts = BF16 ? 1 : 3;  // bf16 parts of a query value and of a probability
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float tops[kWaves][kCols], sums[kWaves][kCols];
    const int t = threadIdx.x, wave = t / kWave, lane = t % kWave;
    const int g = lane / 16, c = lane % 16;
    const int latent = FULL ? kLatentMax : p.b.latent, rope = FULL ? kLatentRopeMax : p.b.rope;
    const int width = latent + rope, dims = latent / 16;
    const int row_bytes = latent_row_bytes(FP4, latent, rope);
    uint8_t *keys_lds = lds + wave * kKeyBytes;
    uint16_t *query_lds = reinterpret_cast<uint16_t *>(lds + kWaves * kKeyBytes);

    const int group = blockIdx.x;
    const Run run = find_run(p, group);
    int *record = p.parts.records + kRecord * group;
    if (t == 0) record[0] = -1;
    long left = run.end - run.begin, offset = run.offset;
    for (int s = run.seq; left > 0 && s < p.b.seqs; ++s, offset = 0) {
        const Work w = work_of(p, s);
        for (; left > 0 && offset < w.units();) {
            const int tile = (int)(offset / w.per), from = (int)(offset - (long)tile * w.per);
            const int upto = left < w.per - from ? from + (int)left : w.per;
            left -= upto - from;
            offset += upto - from;

            // the tile's columns
            const long pair0 = (long)tile * kCols, pairs = (long)w.seq.count * p.heads;
            const int used = pairs - pair0 < kCols ? (int)(pairs - pair0) : kCols;
            const long base = (long)w.seq.begin * p.heads + pair0;  // among all (row, head) pairs
            // keys that row i of the sequence sees, as far as the table goes
            const auto seen = [&](long pair) {
                const long n = (long)w.seq.length - w.seq.count + 1 + pair / p.heads;
                return n < 0 ? 0 : n < w.keys ? (int)n : w.keys;
            };
            const int limit = c < used ? seen(pair0 + c) : 0;
            const int least = seen(pair0), most = seen(pair0 + used - 1);
            // a row that sees more keys than the table can hold
            const bool beyond = c < used && (long)w.seq.length - w.seq.count + 1 + (pair0 + c) / p.heads > w.keys;

            // queries: in registers as they are, or in LDS in parts
            u32x4 query[BF16 ? kSteps + kRopeSteps : 1];
            if constexpr (BF16) {
                const uint16_t *q = static_cast<const uint16_t *>(p.q) + (base + (c < used ? c : 0)) * width;
#pragma unroll
                for (int j = 0; j < kSteps + kRopeSteps; ++j) {
                    const int at = j < kSteps ? dim_of<FP4>(j, g) : 32 * (j - kSteps) + 8 * g;
                    const bool in = c < used && (FULL || at < (j < kSteps ? latent : rope));
                    u32x4 v = {0, 0, 0, 0};
                    if (in) v = *reinterpret_cast<const u32x4_any *>(q + (j < kSteps ? at : latent + at));
                    query[j] = v;
                }
            } else {
                const float *q = static_cast<const float *>(p.q) + base * width;
                __syncthreads();  // (the tile before is read)
                for (int i = t; i < kCols * (kLatentMax + kLatentRopeMax); i += kThreads) {
                    const int col = i / (kLatentMax + kLatentRopeMax), d = i % (kLatentMax + kLatentRopeMax);
                    const bool in = col < used && (d < kLatentMax ? d < latent : d - kLatentMax < rope);
                    const float v = in ? q[(long)col * width + (d < kLatentMax ? d : latent + d - kLatentMax)] : 0.0f;
                    unsigned part[3];
                    split3(v, part);
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        query_lds[(k * kCols + col) * kQueryStride + d] = (uint16_t)part[k];
                }
                __syncthreads();
            }

            Soft soft = {-INFINITY, beyond ? NAN : 0.0f};
            f32x4 out[kDims];
#pragma unroll
            for (int d = 0; d < kDims; ++d) out[d] = f32x4{0.f, 0.f, 0.f, 0.f};

            for (int unit = from; unit < upto; ++unit) {
                const int key0 = unit * kUnitKeys + wave * kTileKeys;
                if (key0 >= most) continue;
                const int mine = key0 + c;
                long slot = mine < most ? latent_slot(p.b, s, (unsigned)mine) : 0;
                unsigned bad = (unsigned)__ballot(slot < 0) & 0xFFFFu;  // keys without a place
                Raw<FP4> raw;
                load_key<FP4, FULL>(raw, static_cast<const uint8_t *>(p.b.data) + (slot < 0 ? 0 : slot) * row_bytes,
                                    g, latent, rope);
                Key key;
                to_key<FP4, FULL>(key, raw, g, latent);
                f32x4 score = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < kSteps + kRopeSteps; ++j) {
#pragma unroll
                    for (int k = 0; k < kParts; ++k) {
                        if constexpr (BF16) {
                            score = mfma32(key.v[j], query[j], score);
                        } else {
                            const int at = j < kSteps ? dim_of<FP4>(j, g) : kLatentMax + 32 * (j - kSteps) + 8 * g;
                            score = mfma32(key.v[j], *reinterpret_cast<const u32x4 *>(
                                                         query_lds + (k * kCols + c) * kQueryStride + at), score);
                        }
                    }
                }
                float sc[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[i] = score[i] * p.scale;
                if (bad || key0 + kTileKeys > least) {
                    // Keys that not every column sees, or that have no place: those that a
                    // column does not see must not reach it by 0 * NaN either, so rows that
                    // are not finite (or not there) are taken out of the second product and
                    // make NaN of the scores of the columns that see them.
                    bool odd = false;
#pragma unroll
                    for (int j = 0; j < kSteps; ++j) odd |= not_finite(key.v[j]);
                    const unsigned long long which = __ballot(odd && mine < most);
                    bad |= (unsigned)(which | which >> 16 | which >> 32 | which >> 48) & 0xFFFFu;
                    const bool out_of_it = mine >= most || (bad >> c & 1u);
#pragma unroll
                    for (int j = 0; j < kSteps; ++j)
                        if (out_of_it) key.v[j] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (bad >> (4 * g + i) & 1u) sc[i] = NAN;
                        if (key0 + 4 * g + i >= limit) sc[i] = -INFINITY;
                    }
                }
                // rows of the second product
#pragma unroll
                for (int j = 0; j < kSteps; ++j)
                    *reinterpret_cast<u32x4 *>(keys_lds + c * kKeyStride + 2 * dim_of<FP4>(j, g)) = key.v[j];

                float top = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
                top = fmaxf(top, __shfl_xor(top, 16, kWave));
                top = fmaxf(top, __shfl_xor(top, 32, kWave));
                if (__any(top > soft.top)) {
                    const float next = fmaxf(soft.top, top);
                    const float by = soft.top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(soft.top - next);
                    soft.sum *= by;
                    soft.top = next;
#pragma unroll
                    for (int d = 0; d < kDims; ++d) out[d] *= by;
                }
                const float zero = soft.top == -INFINITY ? 0.0f : soft.top;
                float prob[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) prob[i] = __builtin_amdgcn_exp2f(sc[i] - zero);
                s16x4 probs[kParts];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (BF16) {
                        const unsigned bits = bf16_bits(prob[i]);
                        probs[0][i] = (short)bits;
                        soft.sum += bf16_value(bits);
                    } else {
                        unsigned part[3];
                        split3(prob[i], part);
#pragma unroll
                        for (int k = 0; k < 3; ++k) probs[k][i] = (short)part[k];
                        soft.sum += prob[i];
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                const uint8_t *from_lds = keys_lds + (4 * g + c / 4) * kKeyStride + 8 * (c % 4);
#pragma unroll
                for (int d = 0; d < kDims; ++d) {
                    if (FULL || d < dims) {
                        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s16x4 *)(from_lds + 32 * d));
#pragma unroll
                        for (int k = 0; k < kParts; ++k)
                            out[d] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(v, probs[k], out[d], 0, 0, 0);
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }

            // the four waves' sums: each to the largest of their maxima, then added
            soft.sum += __shfl_xor(soft.sum, 16, kWave);
            soft.sum += __shfl_xor(soft.sum, 32, kWave);
            if (g == 0) {
                tops[wave][c] = soft.top;
                sums[wave][c] = soft.sum;
            }
            __syncthreads();
            const float all = fmaxf(fmaxf(tops[0][c], tops[1][c]), fmaxf(tops[2][c], tops[3][c]));
            const float by = soft.top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(soft.top - all);
            const bool whole = from == 0 && upto == w.per;
            const int slot = 2 * group + (from == 0 ? 1 : 0);
            // thread: column t / 16, values 4 (t % 16) + 64 k of a round
            const int col = t / kCols;
            float col_top = fmaxf(fmaxf(tops[0][col], tops[1][col]), fmaxf(tops[2][col], tops[3][col]));
            float col_sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kWaves; ++k)
                col_sum += tops[k][col] == -INFINITY
                               ? sums[k][col] * 0.0f  // (0, or NaN where a column is)
                               : sums[k][col] * __builtin_amdgcn_exp2f(tops[k][col] - col_top);
            const float over = col_top == -INFINITY && !(col_sum != col_sum) ? 0.0f : 1.0f / col_sum;
            float *results = reinterpret_cast<float *>(lds);
            for (int round = 0; round < (latent + kJoinDims - 1) / kJoinDims; ++round) {
                if (round) __syncthreads();
#pragma unroll
                for (int d = 0; d < kDims; ++d)
                    if (d / (kJoinDims / 16) == round) {
                        const f32x4 v = out[d] * by;
                        *reinterpret_cast<f32x4 *>(results + (wave * kCols + c) * kJoinStride +
                                                   16 * (d % (kJoinDims / 16)) + 4 * g) = v;
                    }
                __syncthreads();
                for (int k = 0; k < kJoinDims / 64; ++k) {
                    const int at = 4 * (t % 16) + 64 * k, d = round * kJoinDims + at;
                    if (d >= latent) break;
                    f32x4 v = load_f4(results + (0 * kCols + col) * kJoinStride + at);
#pragma unroll
                    for (int x = 1; x < kWaves; ++x) v += load_f4(results + (x * kCols + col) * kJoinStride + at);
                    if (!whole) {
                        *reinterpret_cast<f32x4 *>(p.parts.sums + ((long)slot * kCols + col) * kLatentMax + d) = v;
                    } else if (col < used) {
                        v *= over;
                        if constexpr (BF16) {
                            uint16_t *to = static_cast<uint16_t *>(p.out) + (base + col) * latent + d;
#pragma unroll
                            for (int i = 0; i < 4; ++i) to[i] = (uint16_t)bf16_bits(v[i]);
                        } else {
                            float *to = static_cast<float *>(p.out) + (base + col) * latent + d;
#pragma unroll
                            for (int i = 0; i < 4; ++i) to[i] = v[i];
                        }
                    }
                }
            }
            if (!whole && t % 16 == 0) {
                p.parts.stats[(long)slot * 2 * kCols + col] = col_top;
                p.parts.stats[((long)slot * 2 + 1) * kCols + col] = col_sum;
            }
            if (t == 0 && from > 0 && upto == w.per) {
                // the tile's first unit, and the workgroup whose run holds it
                const long first = run.begin - from;
                record[1] = tile;
                record[2] = (int)(((first + 1) * run.groups - 1) / run.total);
                record[0] = s;
            }
            __syncthreads();
        }
    }
}

// Joins the tile that workgroup blockIdx.x finished but did not begin: its sums are in slot
// 2 first + 1 and in slots 2w of the workgroups w after the first.  A workgroup of this
// launch takes one column.
template <bool BF16> __global__ __launch_bounds__(kLatentMax / 4) void latent_join_kernel(Params p) {
    const int group = blockIdx.x, col = blockIdx.y;
    const int *record = p.parts.records + kRecord * group;
    const int s = record[0];
    if (s < 0) return;
    const int tile = record[1], first = record[2];
    const LatentSeq seq = latent_seq(p.b, s, p.rows);
    const long pair = (long)tile * kCols + col;
    if (pair >= (long)seq.count * p.heads) return;
    const int d = 4 * (int)threadIdx.x;
    if (d >= p.b.latent) return;
    const auto slot_of = [&](int w) { return w == first ? 2L * w + 1 : 2L * w; };
    float top = -INFINITY;
    for (int w = first; w <= group; ++w)
        top = fmaxf(top, p.parts.stats[slot_of(w) * 2 * kCols + col]);
    float sum = 0.0f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int w = first; w <= group; ++w) {
        const long slot = slot_of(w);
        const float its = p.parts.stats[slot * 2 * kCols + col];
        const float by = its == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(its - top);
        sum += by * p.parts.stats[(slot * 2 + 1) * kCols + col];
        v += by * load_f4(p.parts.sums + (slot * kCols + col) * kLatentMax + d);
    }
    v *= top == -INFINITY && !(sum != sum) ? 0.0f : 1.0f / sum;
    const long at = ((long)seq.begin * p.heads + pair) * p.b.latent + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) static_cast<uint16_t *>(p.out)[at + i] = (uint16_t)bf16_bits(v[i]);
        else static_cast<float *>(p.out)[at + i] = v[i];
    }
}

template <bool FP4, bool BF16, bool FULL> int launch(const Params &p, hipStream_t stream) {
    constexpr int bytes = kWaves * kKeyBytes + (BF16 ? 0 : kQueryBytes);
    const auto kernel = latent_attend_kernel<FP4, BF16, FULL>;
    static const bool ok = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
    if (!ok) return kErrLaunch;
    kernel<<<p.groups, kThreads, bytes, stream>>>(p);
    if (hipGetLastError() != hipSuccess) return kErrLaunch;
    if (p.groups == 1) return kOk;
    latent_join_kernel<BF16><<<dim3(p.groups, kCols), kLatentMax / 4, 0, stream>>>(p);
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
