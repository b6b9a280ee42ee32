// logprobs.hip -- log probabilities of given tokens, entropies and the most likely tokens
// of rows of logits (gfx950, wave64).
//
//   m = max x, Z = sum exp(x - m), T = sum (x - m) exp(x - m)
//   log p_t = (x_t - m) - log Z,   H = log Z - T / Z
//
// A row is cut into pieces, one a workgroup, which holds its piece in registers: one pass
// over the memory.  A second launch joins a row's pieces.  The sums go into 64 bits 16
// bytes of logits at a time; those among which the piece's maximum may be are added one by
// one, since next to its 1 what makes a likely token's log p would be lost.
//
// The top k: the k-th largest of a wave's threads' own largest is a bound that at least k
// values reach, and only k threads' values, so what is left to be put in order is few however
// the values lie.  It is found two bits at a time, by counting lanes.  (value, index) are
// compared as one whole number, all different.
//
// exp(d) is the hardware's 2^(d log2 e): d and the product are rounded to f32, which puts a
// term off by 2.1 |d| 2^-24 of itself.
//
// Measured, calls without the join and what it adds: 512 bf16 rows of 163840 logits, 168 MB, 36-40 and 2
// us, where a plain read takes 24: 14 vector instructions a logit, which keep the vector units busy
// 82 % of the time.  61 f32 rows of 50021 with 20 likely tokens 11.5 and 5.8 (without them 10 in all:
// what it takes to choose and order 20 of a piece, waves waiting 57 % of their time), one f32 row of
// 163840 with 5 likely tokens 6.8 and 4.2 (two launches and the trips to memory of each).
#include "bf16.h"
#include "latent.h"
#include "mlh_device.h"
#include "mlh_host.h"

namespace mlh {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kFew = 8, kMany = 32;  // values a thread holds
// Pieces of kMany values a thread, where that gives the chip's 256 CUs a workgroup each.  Calls in
// us with kMany and kFew: 512 bf16 rows of 163840 41 and 60; 61 f32 rows of 50021 (427 pieces of
// kMany) 10.1 and 11.5, with 20 likely tokens 17.1 and 17.4, with 32 19 and 27; 30 such rows
// (210) with 20 16.5 and 15; one f32 row of 163840 12.9 and 11.3.
constexpr long kManyFrom = 256;

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef unsigned long long Rank;  // value, then the lower index first; 0: none

__device__ __forceinline__ Rank rank_of(float v, unsigned index) {
    if (v != v) return 0;
    const unsigned u = __float_as_uint(v + 0.0f);  // (-0 is 0)
    return (Rank)(u ^ ((int)u < 0 ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ unsigned index_of(Rank r) { return 0xFFFFFFFFu - (unsigned)r; }
__device__ __forceinline__ float value_of(Rank r) {
    const unsigned u = (unsigned)(r >> 32);
    return __uint_as_float(u ^ ((int)u < 0 ? 0x80000000u : 0xFFFFFFFFu));
}

struct Stats {
    double sum, mean;  // Z, T
    float top;         // m
    float pad;
};

// The largest `top` ranks among `n` candidates in LDS, in order, into out[0 .. top).
__device__ __forceinline__ void put_in_order(const Rank *found, int n, int top, Rank *out) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const Rank mine = found[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += found[j] > mine;
        if (above < top) out[above] = mine;
    }
    for (int i = n + threadIdx.x; i < top; i += kThreads) out[i] = 0;
}

// The largest whole number below 2^(2 DIGITS) that `top` lanes or more, of those that count,
// reach, or 0, and how many reach it: two bits at a time, until `top` lanes are left.
template <int DIGITS, class Reaches> __device__ __forceinline__ unsigned reached_by(int top, Reaches reaches, int *lanes) {
    unsigned least = 0;
    int n = kWave;
    for (int shift = 2 * DIGITS - 2; shift >= 0 && n != top; shift -= 2) {
        const auto count = [&](unsigned digit) { return __popcll(__ballot(reaches(least | digit << shift))); };
        const int n1 = count(1), n2 = count(2), n3 = count(3);
        const unsigned digit = n3 >= top ? 3u : n2 >= top ? 2u : n1 >= top ? 1u : 0u;
        n = n3 >= top ? n3 : n2 >= top ? n2 : n1 >= top ? n1 : n;
        least |= digit << shift;
    }
    *lanes = n;
    return least;
}

// A bound that at least `top` of the workgroup's values reach, if it has as many, and values
// of at most `top` threads of each wave: the largest of what `top` threads of a wave reach
// (0 where fewer than `top` threads of each have a rank).  `high`: of a thread's largest rank (0:
// it has none), `low` gives the rest of it, by which equal values differ.
template <class Low> __device__ __forceinline__ Rank bound_of(unsigned high, Low low, int top, Rank *bounds) {
    int n;
    const unsigned least = reached_by<16>(top, [&](unsigned v) { return high >= v; }, &n);
    unsigned rest = 0;
    if (least && n != top) {
        // (indexes are below 2^22, which leaves ones above)
        const unsigned mine = low() & 0x3FFFFFu;
        rest = reached_by<11>(top, [&](unsigned v) { return high > least || (high == least && mine >= v); }, &n) | 0xFFC00000u;
    }
    if (threadIdx.x % kWave == 0) bounds[threadIdx.x / kWave] = (Rank)least << 32 | rest;
    __syncthreads();
    Rank bound = bounds[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) bound = bounds[w] > bound ? bounds[w] : bound;
    return bound;
}

__device__ __forceinline__ float from_bits(unsigned w, int half) {
    return __uint_as_float(half ? w & 0xFFFF0000u : w << 16);
}

// Log probability and entropy from a row's sums.
__device__ __forceinline__ void finish(const TokenLogprobs &p, int r, float top, double sum, double mean) {
    const double rest = log(sum);
    // (sums of a row with nothing above -inf, with +inf or NaN are NaN already)
    const int token = p.tokens[r];
    float at = NAN;
    if ((unsigned)token < (unsigned)p.vocab) {
        const long i = (long)r * p.stride + token;
        at = p.bf16 ? bf16_value(static_cast<const uint16_t *>(p.logits)[i]) : static_cast<const float *>(p.logits)[i];
    }
    p.logprobs[r] = (float)((double)at - (double)top - rest);
    if (p.entropy) p.entropy[r] = (float)(rest - mean / sum);
}

__device__ __forceinline__ void finish_top(const TokenLogprobs &p, int r, int k, Rank rank, float top, double sum) {
    const long at = (long)r * p.top + k;
    p.top_ids[at] = rank ? (int)index_of(rank) : -1;
    p.top_logprobs[at] = rank ? (float)((double)value_of(rank) - (double)top - log(sum)) : NAN;
}

template <bool BF16, bool TOP, int N>
__global__ __launch_bounds__(kThreads) void logprobs_piece_kernel(TokenLogprobs p, int pieces, Stats *stats,
                                                                  Rank *ranks) {
    constexpr int kVec = BF16 ? 8 : 4, kVecs = N / kVec;
    __shared__ float tops[kWaves];
    __shared__ double sums[kWaves][2];
    __shared__ Rank found[TOP ? kWaves * kLogprobsMaxTop * N : 1], sorted[TOP ? kLogprobsMaxTop : 1];
    __shared__ Rank bounds[kWaves];
    __shared__ int count;
    const int t = threadIdx.x, wave = t / kWave, lane = t % kWave;
    const int r = blockIdx.x / pieces, piece = blockIdx.x - r * pieces;
    using T = typename std::conditional<BF16, uint16_t, float>::type;
    const T *row = static_cast<const T *>(p.logits) + (long)r * p.stride;
    const int base = piece * kThreads * N;
    const auto first = [&](int k) { return base + (k * kThreads + t) * kVec; };
    u32x4 bits[kVecs];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int i = first(k);
        if (i + kVec <= p.vocab) {
            bits[k] = *reinterpret_cast<const u32x4_any *>(row + i);
        } else {
            constexpr unsigned kLowest = BF16 ? 0xFF80FF80u : 0xFF800000u;  // -inf
            bits[k] = u32x4{kLowest, kLowest, kLowest, kLowest};
#pragma unroll
            for (int x = 0; x < kVec; ++x) {
                if (i + x >= p.vocab) break;
                if constexpr (BF16)
                    bits[k][x / 2] = x % 2 ? (bits[k][x / 2] & 0xFFFFu) | (unsigned)row[i + x] << 16
                                           : (bits[k][x / 2] & 0xFFFF0000u) | row[i + x];
                else bits[k][x] = __float_as_uint(row[i + x]);
            }
        }
    }
    const auto value = [&](int k, int x) {
        if constexpr (BF16) return from_bits(bits[k][x / 2], x % 2);
        else return __uint_as_float(bits[k][x]);
    };
    float vec_top[kVecs], mine = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        vec_top[k] = -INFINITY;
#pragma unroll
        for (int x = 0; x < kVec; ++x) vec_top[k] = fmaxf(vec_top[k], value(k, x));
        mine = fmaxf(mine, vec_top[k]);
    }
    const float wave_top = dpp_wave_max(mine);
    if (lane == 0) tops[wave] = wave_top;
    if (TOP && t == 0) count = 0;
    __syncthreads();
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float base_top = top == -INFINITY ? 0.0f : top;  // (of a piece with nothing above)
    double sum = 0.0, mean = 0.0;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        float e[kVec], s = 0.0f, m = 0.0f;
#pragma unroll
        for (int x = 0; x < kVec; ++x) {
            // (a masked value's 0 times infinity is to be 0; NaN stays NaN, by e)
            const float d = value(k, x) - base_top;
            e[x] = __builtin_amdgcn_exp2f(d * 1.44269504f);
            m = fmaf(e[x], fmaxf(d, -1000.0f), m);
            s += e[x];
        }
        if (vec_top[k] - top > -0.7f) {
#pragma unroll
            for (int x = 0; x < kVec; ++x) sum += (double)e[x];
        } else {
            sum += (double)s;
        }
        mean += (double)m;
    }
    sum = dpp_wave_sum(sum);
    mean = dpp_wave_sum(mean);
    if (lane == 0) sums[wave][0] = sum, sums[wave][1] = mean;
    __syncthreads();
    sum = (sums[0][0] + sums[1][0]) + (sums[2][0] + sums[3][0]);
    mean = (sums[0][1] + sums[1][1]) + (sums[2][1] + sums[3][1]);
    if constexpr (TOP) {
        // (index of the thread's largest value; -1: it has none)
        const auto largest = [&] {
            int at = -1;
#pragma unroll
            for (int k = kVecs - 1; k >= 0; --k)
#pragma unroll
                for (int x = kVec - 1; x >= 0; --x)
                    if (value(k, x) == mine && first(k) + x < p.vocab) at = first(k) + x;
            return at;
        };
        const bool any = mine > -INFINITY || largest() >= 0;
        const Rank least = bound_of(any ? (unsigned)(rank_of(mine, 0) >> 32) : 0u,
                                    [&] { return 0xFFFFFFFFu - (unsigned)largest(); }, p.top, bounds);
        const float least_value = least ? value_of(least) : -INFINITY;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            if (vec_top[k] < least_value) continue;
#pragma unroll
            for (int x = 0; x < kVec; ++x) {
                const Rank rank = first(k) + x < p.vocab ? rank_of(value(k, x), first(k) + x) : 0;
                if (rank && rank >= least) found[atomicAdd(&count, 1)] = rank;
            }
        }
        __syncthreads();
        put_in_order(found, count, p.top, sorted);
        __syncthreads();
    }
    if (pieces == 1) {
        if (top == -INFINITY) sum = NAN;
        if (t == 0) finish(p, r, top, sum, mean);
        if (TOP && t < p.top) finish_top(p, r, t, sorted[t], top, sum);
        return;
    }
    if (t == 0) stats[blockIdx.x] = {sum, mean, top, 0.0f};
    if (TOP && t < p.top) ranks[(long)blockIdx.x * p.top + t] = sorted[t];
}

// Joins a row's pieces.
template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(TokenLogprobs p, int pieces, const Stats *stats,
                                                                 const Rank *ranks) {
    __shared__ float tops[kWaves];
    __shared__ double sums[kWaves][2];
    __shared__ Rank sorted[TOP ? kLogprobsMaxTop : 1];
    extern __shared__ __attribute__((aligned(16))) Rank found[];
    __shared__ Rank bounds[kWaves];
    __shared__ int count;
    const int t = threadIdx.x, wave = t / kWave, lane = t % kWave, r = blockIdx.x;
    const Stats *its = stats + (long)r * pieces;
    const Rank *from = ranks + (long)r * pieces * p.top;
    const int n = pieces * p.top;
    Rank best = 0;
    if constexpr (TOP)
        for (int i = t; i < n; i += kThreads) best = from[i] > best ? from[i] : best;
    float mine = -INFINITY;
    for (int i = t; i < pieces; i += kThreads) mine = fmaxf(mine, its[i].top);
    mine = dpp_wave_max(mine);
    if (lane == 0) tops[wave] = mine;
    if (TOP && t == 0) count = 0;
    __syncthreads();
    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double sum = 0.0, mean = 0.0;
    for (int i = t; i < pieces; i += kThreads) {
        const Stats s = its[i];
        // x - top = (x - s.top) + off: T moves by off Z
        if (s.top == -INFINITY) {
            sum += s.sum;  // 0, or NaN
            continue;
        }
        const double off = (double)s.top - (double)top, by = exp(off);
        sum += by * s.sum;
        mean += by == 0.0 ? 0.0 : by * (s.mean + off * s.sum);
    }
    sum = dpp_wave_sum(sum);
    mean = dpp_wave_sum(mean);
    if (lane == 0) sums[wave][0] = sum, sums[wave][1] = mean;
    __syncthreads();
    sum = (sums[0][0] + sums[1][0]) + (sums[2][0] + sums[3][0]);
    mean = (sums[0][1] + sums[1][1]) + (sums[2][1] + sums[3][1]);
    if (top == -INFINITY) sum = NAN;
    if (t == 0) finish(p, r, top, sum, mean);
    if constexpr (TOP) {
        const Rank least = bound_of((unsigned)(best >> 32), [&] { return (unsigned)best; }, p.top, bounds);
        for (int i = t; i < n; i += kThreads) {
            const Rank rank = from[i];
            if (rank && rank >= least) found[atomicAdd(&count, 1)] = rank;
        }
        __syncthreads();
        put_in_order(found, count, p.top, sorted);
        __syncthreads();
        if (t < p.top) finish_top(p, r, t, sorted[t], top, sum);
    }
}

int values_of(int rows, int vocab) {
    const long pieces = (vocab - 1) / (kThreads * kMany) + 1;
    return pieces * rows >= kManyFrom ? kMany : kFew;
}

// Ranks that the join of so many pieces may have to put in order: of the threads that reach the
// bound, at most `top` of a wave, all that they hold.
constexpr size_t most_found(size_t pieces, size_t top) {
    const size_t n = pieces * top, reach = kWaves * top * ((n + kThreads - 1) / kThreads);
    return n < reach ? n : reach;
}
// A call's pieces of kFew values, which are taken while those of kMany are fewer than kManyFrom; a
// row's of kMany.
constexpr size_t kMostFew = kMany / kFew * (kManyFrom - 1), kMostMany = kLogprobsMaxVocab / (kThreads * kMany);
constexpr size_t kMostFound = most_found(kMostFew > kMostMany ? kMostFew : kMostMany, kLogprobsMaxTop);
static_assert(sizeof(Rank) * kMostFound <= 128 << 10, "LDS, of 160 KB with the join's own arrays");

template <bool BF16, bool TOP, int N> int launch(const TokenLogprobs &p, hipStream_t stream) {
    const int pieces = (p.vocab - 1) / (kThreads * N) + 1;
    const size_t blocks = (size_t)pieces * p.rows;
    Stats *stats = static_cast<Stats *>(p.workspace);
    Rank *ranks = reinterpret_cast<Rank *>(stats + blocks);
    if (TOP && pieces > 1) {
        static const bool ok = allow_lds(logprobs_join_kernel<true>, sizeof(Rank) * kMostFound);
        if (!ok) return kErrLaunch;
    }
    logprobs_piece_kernel<BF16, TOP, N><<<(unsigned)blocks, kThreads, 0, stream>>>(p, pieces, stats, ranks);
    if (hipGetLastError() != hipSuccess) return kErrLaunch;
    if (pieces == 1) return kOk;
    const size_t found = TOP ? sizeof(Rank) * most_found(pieces, p.top) : 0;
    logprobs_join_kernel<TOP><<<p.rows, kThreads, found, stream>>>(p, pieces, stats, ranks);
    return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

template <bool BF16, bool TOP> int launch(const TokenLogprobs &p, hipStream_t stream) {
    return values_of(p.rows, p.vocab) == kMany ? launch<BF16, TOP, kMany>(p, stream) : launch<BF16, TOP, kFew>(p, stream);
}

}  // namespace

bool token_logprobs_fits(int rows, int vocab) {
    const long pieces = (vocab - 1) / (kThreads * values_of(rows, vocab)) + 1;
    return pieces * rows <= 0xFFFFFFFFl / kThreads;
}

static size_t piece_bytes(int top) { return sizeof(Stats) + sizeof(Rank) * top; }

size_t token_logprobs_needs(int rows, int vocab, int top) {
    const size_t pieces = (vocab - 1) / (kThreads * values_of(rows, vocab)) + 1;
    return pieces == 1 ? 0 : pieces * rows * piece_bytes(top);
}

// Of any call of at most `rows` rows of `vocab` logits.
size_t token_logprobs_workspace(int rows, int vocab, int top) {
    const size_t many = (vocab - 1) / (kThreads * kMany) + 1, few = (vocab - 1) / (kThreads * kFew) + 1;
    const size_t of_few = few == 1 ? 0 : few * rows < kMostFew ? few * rows : kMostFew;
    const size_t of_many = many == 1 ? 0 : many * rows;
    return (of_few > of_many ? of_few : of_many) * piece_bytes(top);
}

int token_logprobs(const TokenLogprobs &p, hipStream_t stream) {
    if (p.bf16) return p.top ? launch<true, true>(p, stream) : launch<true, false>(p, stream);
    return p.top ? launch<false, true>(p, stream) : launch<false, false>(p, stream);
}

}  // namespace mlh
