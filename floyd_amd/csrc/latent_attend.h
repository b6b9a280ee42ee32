// latent_attend.h -- what the attention kernels over the latent cache share: a batch's work
// dealt to workgroups, its keys as they are read, partial sums and their join (internal).
#pragma once

#include "bf16.h"
#include "latent.h"
#include "mlh_device.h"
#include "mlh_host.h"

namespace mlh {

namespace latent_attention {

typedef u32x4 u32x4_any __attribute__((aligned(2)));

constexpr int kSteps = kLatentMax / 32;          // 32-value steps over a latent row
constexpr int kRopeSteps = kLatentRopeMax / 32;  // and over a rope row

// A tile is kCols (row, head) pairs of a sequence; its keys are taken 2^kStepShift at a time (a
// step), and a workgroup has at least 2^kLeastShift keys, where there are as many.
template <int COLS, int STEP_SHIFT, int LEAST_SHIFT, int GROUPS> struct Tiling {
    static constexpr int kCols = COLS, kStepShift = STEP_SHIFT, kStepKeys = 1 << STEP_SHIFT;
    static constexpr int kLeastShift = LEAST_SHIFT;
    static constexpr int kGroups = GROUPS;  // workgroups of a launch, at most
};
typedef Tiling<16, 4, 6, 512> Narrow;
typedef Tiling<64, 6, 7, 254> Wide;  // (its parts: in 64 MiB of workspace)

// What latent_join_kernel has to know of a tile, told by the workgroup that ends it: its
// sequence and number in it, and the workgroups that its units fell to (-1: to one, there is
// nothing to join).  Where a batch has few tiles a record belongs to the tile: of sequence s,
// the tile that begins with pair b of all (row, head) pairs has record b / kCols + s.  Those
// are different, but not every record has a tile, and one that has none tells of an
// earlier call's.  Else a record belongs to the workgroup, which ends at most one tile that
// another one began.
struct __attribute__((aligned(16))) Record {
    int seq, tile, first, last;
};
constexpr int kMaxTileRecords = 2048;

// Partial sums of tiles: slot 2w holds the tile that workgroup w found begun, slot 2w + 1
// the one that it left unfinished.
struct Parts {
    float *sums;    // [2 groups][kCols][kLatentMax]
    float *stats;   // [2 groups][2][kCols] maxima, then sums
    Record *records;
    int tiles;      // records of tiles, else 0: of workgroups
};
constexpr long kMaxPartCols = Narrow::kGroups * Narrow::kCols > Wide::kGroups * Wide::kCols ? 2 * Narrow::kGroups * Narrow::kCols
                                                                                        : 2 * Wide::kGroups * Wide::kCols;
constexpr size_t kSumsBytes = kMaxPartCols * kLatentMax * 4;
constexpr size_t kStatsBytes = kMaxPartCols * 2 * 4;
constexpr size_t kRecordBytes = (size_t)kMaxTileRecords * sizeof(Record);
static_assert(kSumsBytes + kStatsBytes + kRecordBytes <= 64 << 20, "the workspace");
static_assert(Narrow::kGroups <= kMaxTileRecords, "records of workgroups");

// n / d of n below 2^31 by a product: m is the whole number above 2^(31 + l) / d with l the
// least for which 2^l >= d.
struct Divisor {
    unsigned m, shift;
    __host__ static Divisor of(unsigned d) {
        unsigned l = 0;
        while ((1ull << l) < d) ++l;
        return {(unsigned)((1ull << (31 + l)) / d + 1), l};
    }
    // ((2^32 / 2) / d would not fit for d = 1)
    __device__ __forceinline__ unsigned quotient(unsigned n) const {
        return shift ? __umulhi(n, m) >> (shift - 1) : n;
    }
};

struct Params {
    MlkLatentBatch b;
    const void *q;
    void *out;
    int rows, heads;
    float scale;  // times log2(e)
    int groups;
    int keys;     // that a table can hold
    int shift;    // a unit is 2^shift steps
    Divisor page, head;
    Parts parts;
};

// A value that all lanes of a wave hold, known to be one: what depends on it is computed and
// branched on once for the wave.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A sequence's work.
struct Work {
    LatentSeq seq;
    int keys;    // that its table can hold
    int per;     // units of a tile
    int tiles;
};

template <class Til> __device__ __forceinline__ Work work_of(const Params &p, const LatentSeq &seq) {
    Work w;
    w.seq = seq;
    const int length = seq.length < 0 ? 0 : seq.length;
    w.keys = length < p.keys ? length : p.keys;
    w.per = w.keys > 0 ? ((w.keys - 1) >> (Til::kStepShift + p.shift)) + 1 : 1;
    // (rows * heads is below 2^31 - 15)
    w.tiles = (int)(((unsigned)seq.count * (unsigned)p.heads + (Til::kCols - 1)) / Til::kCols);
    return w;
}

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// A workgroup's run of units: `length` of them from the one that is `offset` after the first
// of sequence `seq`; `begin` is that one's place among all.
struct Run {
    int seq, offset, begin, length;
    int share, rest;  // workgroups have `share` units each, the first `rest` of them one more
    bool malformed;   // starts decrease: rows of several sequences could make more units than are counted
    // Of `total` units, dealt to no more workgroups than leaves each 2^least of them: then no run
    // between those of one tile is empty, and a tile has no more parts than pay.
    __device__ __forceinline__ void deal(int total, int groups, int group, int least) {
        const int most = ((total - 1) >> least) + 1;
        groups = most < groups ? most : groups;
        offset = begin = length = share = seq = rest = 0;
        if (group >= groups) return;
        share = (int)((unsigned)total / (unsigned)groups);
        rest = total - share * groups;
        begin = share * group + (group < rest ? group : rest);
        length = share + (group < rest ? 1 : 0);
    }
    __device__ __forceinline__ int owner(int unit) const {
        const int longer = (share + 1) * rest;
        return (int)(unit < longer ? (unsigned)unit / (unsigned)(share + 1)
                                   : rest + (unsigned)(unit - longer) / (unsigned)share);
    }
};

// The sequences are in LDS (`held`) where a workgroup has a thread for each.
template <class Til, int WAVES> __device__ __forceinline__ Run find_run(const Params &p, int group, LatentSeq *held) {
    constexpr int kWaves = WAVES, kThreads = kWaves * kWave, kLeast = Til::kLeastShift - Til::kStepShift;
    __shared__ int sums[kWaves], at[2];
    const int t = threadIdx.x, wave = uniform(t / kWave), lane = t % kWave;
    const auto seq_of = [&](int s) { return s < p.b.seqs ? latent_seq(p.b, s, p.rows) : LatentSeq{0, 0, 0}; };
    const auto units_of = [&](const LatentSeq &q) {
        const Work w = work_of<Til>(p, q);
        return w.per * w.tiles;
    };
    Run r;
    const LatentSeq mine = seq_of(t);
    int units = units_of(mine), all = units, total = 0;
    if (t == 0) at[0] = p.b.seqs;  // (no sequence, until one is found)
    bool decrease = mine.begin < 0;
    r.malformed = false;
    if (p.b.seqs <= kThreads) {
        held[t] = mine;
    } else {
        for (int s = t + kThreads; s < p.b.seqs; s += kThreads) {
            const LatentSeq seq = seq_of(s);
            all += units_of(seq);
            decrease |= seq.begin < 0;
        }
        all = __any(decrease) ? -1 : wave_sum_int(all);
        if (lane == 0) sums[wave] = all;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) {
            const int units = uniform(sums[w]);
            r.malformed |= units < 0;
            total += units;
        }
        r.deal(r.malformed ? 0 : total, p.groups, group, kLeast);
        decrease = false;
    }
    int before = 0;
    for (int s0 = 0;; s0 += kThreads) {
        if (s0) units = units_of(seq_of(s0 + t));
        const bool none = __any(decrease);
        const int upto = wave_scan(units);
        __syncthreads();
        if (lane == kWave - 1) sums[wave] = none ? -1 : upto;
        __syncthreads();
        int first = before + upto - units;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int all = uniform(sums[w]);
            r.malformed |= all < 0;
            if (w < wave) first += all;
            before += all;
        }
        if (p.b.seqs <= kThreads) r.deal(r.malformed ? 0 : before, p.groups, group, kLeast);
        if (r.begin >= first && r.begin < first + units) {
            at[0] = s0 + t;
            at[1] = r.begin - first;
        }
        if (r.begin < before || s0 + kThreads >= p.b.seqs) break;
    }
    __syncthreads();
    if (r.length > 0) {
        r.seq = uniform(at[0]);
        r.offset = uniform(at[1]);
    }
    return r;
}

// Records of workgroups begin without a tile; those of tiles that no workgroup is to do are told, or an
// earlier call's would be joined.
__device__ __forceinline__ void begin_records(const Params &p, const Run &run, int group) {
    if (threadIdx.x) return;
    if (!p.parts.tiles) p.parts.records[group].first = -1;
    else if (run.malformed)
        for (int i = group; i < p.parts.tiles; i += p.groups) p.parts.records[i].first = -1;
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
    u32x4 v[kSteps + kRopeSteps];
};
template <> struct Raw<true> {
    u32x4 codes[kSteps / 4];
    unsigned scales;
    u32x4 rope[kRopeSteps];
};

// Whether one of its latent values is not finite, and the key without its latent values.
__device__ __forceinline__ bool not_finite(const Raw<true> &raw, int g, int latent) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < kSteps / 4; ++j)  // (scales that a narrower row has not are any bytes)
        bad |= 128 * j + 32 * g < latent && (raw.scales >> (8 * j) & 0xFFu) == 0xFFu;
    return bad;
}
__device__ __forceinline__ bool not_finite(const Raw<false> &raw, int, int) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            bad |= (raw.v[j][i] & 0x7F80u) == 0x7F80u || (raw.v[j][i] & 0x7F800000u) == 0x7F800000u;
    return bad;
}
__device__ __forceinline__ void drop(Raw<true> &raw) {
    raw.scales = 0x7F7F7F7Fu;
#pragma unroll
    for (int j = 0; j < kSteps / 4; ++j) raw.codes[j] = u32x4{0, 0, 0, 0};
}
__device__ __forceinline__ void drop(Raw<false> &raw) {
#pragma unroll
    for (int j = 0; j < kSteps; ++j) raw.v[j] = u32x4{0, 0, 0, 0};
}

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
        for (int j = 0; j < kSteps + kRopeSteps; ++j) {
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
// it (in powers of 2): p stays below 2^25 and sums lose nothing by that (2^31 keys' are finite for
// values below 2^71), and most steps need not scale what is summed.
constexpr float kSlack = 24.0f;
// exp2(q . k scale - top) takes the product and the difference in one rounding, `top` is a rounded
// product: from here on they may be more than 1 apart, at 2^32 more than 2^7, which makes 0 or an
// infinity of the largest p.
constexpr float kLarge = 0x1p25f;
// (a score of -inf would be a key without weight: a score that is not finite is NaN)
__device__ __forceinline__ float large_score(float s) { return fabsf(s) < INFINITY ? s : NAN; }

// Joins the tile of record blockIdx.x: its sums are in part 2 first + 1 and in parts 2w of
// the workgroups w after the first.  128 threads take a column's values, and TEAMS such teams
// share its parts: a round of loads from what other workgroups wrote takes about a
// microsecond, so as many as can are under way at once: four teams where all workgroups are
// resident that way, and 16 loads a thread for the few tiles of small batches, whose parts are
// many; else 4 loads, for what a thread asks for beyond the last part is read again for nothing
// (17 tiles of about 15 parts 9.6 us with 16 loads, 6.1 with 4; 80 tiles of 64 columns and of about
// four parts 16.3 and 11.6).
constexpr int kTeam = kLatentMax / 4;
constexpr int kMaxTeams = 4;
template <class Til, bool BF16, int TEAMS, int LOADS> __global__ __launch_bounds__((kTeam * TEAMS)) void latent_join_kernel(Params p) {
    constexpr int kCols = Til::kCols, kThreads = kTeam * TEAMS, kLoads = LOADS, kStride = kLoads * TEAMS;
    __shared__ float tops[Til::kGroups], sums[Til::kGroups];
    __shared__ float reds[2][kThreads / kWave];
    __shared__ f32x4 shares[TEAMS][kTeam];
    const Record record = p.parts.records[blockIdx.x];
    if (record.first < 0) return;
    const int col = blockIdx.y, team = threadIdx.x / kTeam, t = threadIdx.x % kTeam;
    // (a record without a tile holds anything)
    const int first = record.first < p.groups ? record.first : 0;
    const int last = record.last < first ? first : record.last < p.groups ? record.last : p.groups - 1;
    const int count = last - first + 1;
    const auto part_of = [&](int i) { return 2 * (first + i) + (i == 0 ? 1 : 0); };
    const int s = (unsigned)record.seq < (unsigned)p.b.seqs ? record.seq : 0;
    const LatentSeq seq = latent_seq(p.b, s, p.rows);
    const int pairs = seq.count * p.heads, pair = record.tile * kCols + col;
    const long base = (long)seq.begin * p.heads;
    const float *from = p.parts.sums + col * kLatentMax + 4 * t;
    float top = -INFINITY, sum = 0.0f;
    f32x4 v[kLoads], result = {0.f, 0.f, 0.f, 0.f};
    // (entered a step early, for the loads; parts i0 + team + k TEAMS)
    for (int i0 = team - kStride; i0 < count; i0 += kStride) {
        if (i0 >= 0) {
#pragma unroll
            for (int k = 0; k < kLoads; ++k)
                if (i0 + k * TEAMS < count) result += tops[i0 + k * TEAMS] * v[k];
        }
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int i = i0 + kStride + k * TEAMS;
            v[k] = load_f4(from + (long)part_of(i < count ? i : count - 1) * (kCols * kLatentMax));
        }
        if (i0 >= 0) continue;
        // (what a record without a tile says of one is not true)
        if (p.parts.tiles && ((unsigned)record.tile > (unsigned)pairs / kCols ||
                              (int)((base + record.tile * kCols) / kCols) + s != (int)blockIdx.x))
            return;
        for (int i = threadIdx.x; i < count; i += kThreads) {
            const float *stats = p.parts.stats + part_of(i) * (2 * kCols) + col;
            tops[i] = stats[0];
            sums[i] = stats[kCols];
            top = fmaxf(top, stats[0]);
        }
        top = dpp_wave_max(top);
        if (threadIdx.x % kWave == 0) reds[0][threadIdx.x / kWave] = top;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kThreads / kWave; ++k) top = fmaxf(top, reds[0][k]);
        if (top == -INFINITY) top = 0.0f;
        for (int i = threadIdx.x; i < count; i += kThreads) {
            const float by = __builtin_amdgcn_exp2f(tops[i] - top);
            tops[i] = by;
            sum += by * sums[i];
        }
        sum = dpp_wave_sum(sum);
        if (threadIdx.x % kWave == 0) reds[1][threadIdx.x / kWave] = sum;
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kThreads / kWave; ++k) sum += reds[1][k];
    }
    if (TEAMS > 1) {
        if (team) shares[team - 1][t] = result;
        __syncthreads();
        if (team) return;
#pragma unroll
        for (int k = 1; k < TEAMS; ++k) result += shares[k - 1][t];
    }
    if (pair >= pairs || 4 * t >= p.b.latent) return;
    store4<BF16>(p.out, (base + pair) * p.b.latent + 4 * t, result * (sum == 0.0f ? 0.0f : 1.0f / sum));
}

// Behind the attention kernel's launch.
template <class Til, bool BF16> int launch_join(const Params &p, hipStream_t stream) {
    if (p.groups == 1) return kOk;
    const int records = p.parts.tiles ? p.parts.tiles : p.groups;
    const dim3 grid(records, Til::kCols);
    if ((long)records * Til::kCols * kTeam * kMaxTeams > (long)p.groups * 2048)
        latent_join_kernel<Til, BF16, 1, 4><<<grid, kTeam, 0, stream>>>(p);
    else if (records >= 16)
        latent_join_kernel<Til, BF16, kMaxTeams, 4><<<grid, kTeam * kMaxTeams, 0, stream>>>(p);
    else
        latent_join_kernel<Til, BF16, kMaxTeams, 16><<<grid, kTeam * kMaxTeams, 0, stream>>>(p);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

// The kernel for many (row, head) pairs a sequence, bf16 queries and full rows (latent_wide.hip).
int launch_wide(bool fp4, const Params &p, hipStream_t stream);

}  // namespace latent_attention

}  // namespace mlh
