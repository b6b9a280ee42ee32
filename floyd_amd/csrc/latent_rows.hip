// latent_rows.hip -- rows of a paged latent cache: written with their norm and
// rotation, and read back (gfx950, wave64).
//
//   append  latent part  v = c / sqrt(mean(c^2) + eps) * w
//           rope part    k_i = x cos a - y sin a, k_(i + R/2) = y cos a + x sin a with
//                        (x, y) = pair i, a = position * inv_freq[i]; queries likewise
//
// in 64 bits: codes of 4 bits are a function of the inputs then, whatever order a sum is
// formed in, and the angle of a far position keeps its bits.  Results are rounded to f32, bf16
// ones from there.
#include "bf16.h"
#include "latent.h"
#include "mlh_device.h"
#include "mlh_host.h"

namespace mlh {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
static_assert(kThreads == kLatentRowThreads && kWaves == kLatentGatherRows, "the rows of a launch");

template <bool BF16> struct Elem { using type = float; };
template <> struct Elem<true> { using type = uint16_t; };

template <bool BF16> __device__ __forceinline__ double value(typename Elem<BF16>::type v) {
    if constexpr (BF16) return (double)bf16_value(v);
    else return (double)v;
}
// By way of f32, which the compiler is not to skip: its conversion of that is one instruction
// for two values (NaN stays NaN), of 64 bits a dozen.
__device__ __forceinline__ uint16_t to_bf16(double v) {
    float f = (float)v;
    asm("" : "+v"(f));
    return __builtin_bit_cast(uint16_t, (__bf16)f);
}
template <bool BF16> __device__ __forceinline__ void store(typename Elem<BF16>::type *p, double v) {
    if constexpr (BF16) *p = to_bf16(v);
    else *p = (float)v;
}
// Two neighbours, at any address of their type.
template <bool BF16> struct Pair {
    typename Elem<BF16>::type x, y;
};
template <bool BF16> __device__ __forceinline__ Pair<BF16> load_pair(const typename Elem<BF16>::type *p) {
    Pair<BF16> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}

// Key position of token row r (below 0: padding) and its place in the pages (-1: none), by every
// lane of a wave; false: r is no row of a sequence.  Its sequence is the number of those that end
// at r or before; their starts and lengths, 64 sequences at a time, are asked for together.
__device__ __forceinline__ bool place_of_row(const MlkLatentBatch &b, int r, int rows, int *position,
                                             long *slot) {
    int s = r, begin = r, end = r + 1, length = 0;
    if (!b.row_starts) {
        if (r >= b.seqs) return false;
        length = b.lengths[r];
    } else {
        const int lane = (int)(threadIdx.x % kWave);
        int before = kWave;
        for (int s0 = 0; before == kWave; s0 += kWave) {
            if (s0 >= b.seqs) return false;
            const int mine = s0 + lane < b.seqs ? s0 + lane : b.seqs - 1;
            const int first = b.row_starts[mine], last = b.row_starts[mine + 1], n = b.lengths[mine];
            before = __popcll(__ballot(s0 + lane < b.seqs && last <= r));
            s = s0 + before;
            begin = __builtin_amdgcn_readlane(first, before % kWave);
            end = __builtin_amdgcn_readlane(last, before % kWave);
            length = __builtin_amdgcn_readlane(n, before % kWave);
        }
        if (s >= b.seqs || begin < 0 || end > rows || r < begin || r >= end) return false;
    }
    const long j = (long)length - (end - r);
    *position = j < 0 ? -1 : (int)j;
    *slot = j < 0 ? -1 : latent_slot(b, s, (unsigned)j);
    return true;
}

// sin and cos of an angle below 2^32 in magnitude, to a few last places of 1: the nearest
// multiple of pi / 2 is taken off in two parts (products and differences exact by fma), and
// what is left, at most pi / 4, goes into the power series up to x^17 and x^16.
__device__ __forceinline__ void turn_of(double angle, double *sine, double *cosine) {
    constexpr double kHalfPi = 0x1.921fb54442d18p+0, kHalfPiRest = 0x1.1a62633145c07p-54;
    const double k = rint(angle * 0x1.45f306dc9c883p-1);
    const double x = fma(-k, kHalfPiRest, fma(-k, kHalfPi, angle)), y = x * x;
    double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;
    s = fma(s, y, -1.0 / 1307674368000.0);
    s = fma(s, y, 1.0 / 6227020800.0);
    s = fma(s, y, -1.0 / 39916800.0);
    s = fma(s, y, 1.0 / 362880.0);
    s = fma(s, y, -1.0 / 5040.0);
    s = fma(s, y, 1.0 / 120.0);
    s = fma(s, y, -1.0 / 6.0);
    s = fma(s * y, x, x);
    c = fma(c, y, -1.0 / 87178291200.0);
    c = fma(c, y, 1.0 / 479001600.0);
    c = fma(c, y, -1.0 / 3628800.0);
    c = fma(c, y, 1.0 / 40320.0);
    c = fma(c, y, -1.0 / 720.0);
    c = fma(c, y, 1.0 / 24.0);
    c = fma(c, y, -0.5);
    c = fma(c, y, 1.0);
    const int quarter = (int)((long long)k & 3);
    const double a = quarter & 1 ? c : s, b = quarter & 1 ? s : c;
    *sine = quarter & 2 ? -a : a;
    *cosine = (quarter + 1) & 2 ? -b : b;
}

// 2^e of a double, e in its normal range.
__device__ __forceinline__ double power2(int e) {
    return __longlong_as_double((long long)(e + 1023) << 52);
}

// A value cut off to f32 with its last bit set where that left something out: rounded to fewer
// bits it goes where the value goes.
__device__ __forceinline__ float to_odd(double v) {
    const float f = (float)v;
    const double back = (double)f;
    unsigned u = __float_as_uint(f);
    if (fabs(back) > fabs(v)) --u;
    return __uint_as_float(back != v ? u | 1u : u);
}
// The e2m1 codes nearest to two values of at most 6 in magnitude, ties to even.
__device__ __forceinline__ uint8_t fp4_codes(double v0, double v1) {
    return (uint8_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, to_odd(v0), to_odd(v1), 1.0f, 0);
}

// The largest of a row of 16 lanes.
template <int CTRL> __device__ __forceinline__ unsigned dpp_max(unsigned v) {
    const unsigned other = __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
    return other > v ? other : v;
}
__device__ __forceinline__ unsigned row_max(unsigned v) {
    v = dpp_max<0xB1>(v);   // quad_perm [1,0,3,2]
    v = dpp_max<0x4E>(v);   // quad_perm [2,3,0,1]
    v = dpp_max<0x141>(v);  // row_half_mirror
    return dpp_max<0x140>(v);  // row_mirror
}

// One token row a workgroup.  What it reads of the row is asked for at once, beside the way to
// its place (starts and length, then table, a microsecond each).  Queries: 32 threads for the
// pairs of a head, 8 heads a pass.  4095 bf16 rows with 16 heads into 4 bits, 23.1 MB, take 13-14 us
// (1.7 TB/s; the library's sine and cosine, loads in turn and codes in 64 bits 19), into bf16 rows, 26
// MB, 12: 8 workgroups a CU, in two rounds, whose waves wait 45 % of their time, for those trips one
// after the other and for the wave that makes sine and cosine.  The vector units are busy 33 % of the
// time; a fifth of their instructions are 64-bit arithmetic.  One row 3.0-3.2 us: a launch and those
// trips.
constexpr int kPairLanes = kLatentRopeMax / 2, kPassHeads = kThreads / kPairLanes;
constexpr int kTurns = 2;  // passes on their way at once
template <bool BF16, bool FP4>
__global__ __launch_bounds__(kThreads) void latent_append_kernel(MlkLatentBatch b, LatentAppend p) {
    using T = typename Elem<BF16>::type;
    __shared__ double part[kWaves];
    __shared__ double turn[kLatentRopeMax / 2][2];
    const int r = blockIdx.x, t = threadIdx.x;
    const int latent = b.latent, half = b.rope / 2, width = latent + b.rope;
    // thread t: latent values 2t and 2t + 1, rope pair t
    const T *kv = static_cast<const T *>(p.kv) + (long)r * p.kv_stride;
    const bool has = 2 * t < latent, turns = t < half;
    const auto latent_pair = load_pair<BF16>(kv + (has ? 2 * t : 0));
    const auto rope_pair = load_pair<BF16>(kv + (turns ? latent + 2 * t : 0));
    const float w0 = p.norm_w && has ? p.norm_w[2 * t] : 1.0f, w1 = p.norm_w && has ? p.norm_w[2 * t + 1] : 1.0f;
    const float freq = p.inv_freq[turns ? t : 0];
    const int lane_pair = t % kPairLanes, head0 = t / kPairLanes;
    const int heads = p.query && lane_pair < half ? p.heads : 0;
    const T *query = static_cast<const T *>(p.query) + (long)r * p.query_stride + p.head_width - b.rope + 2 * lane_pair;
    Pair<BF16> asked[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
        asked[k] = {};
        const int h = head0 + k * kPassHeads;
        if (h < heads) asked[k] = load_pair<BF16>(query + (long)h * p.head_width);
    }
    int position;
    long slot;
    if (!place_of_row(b, r, p.rows, &position, &slot) || position < 0) return;
    double cs = 1.0, sn = 0.0;
    if (turns) {
        turn_of((double)position * (double)freq, &sn, &cs);
        turn[t][0] = cs;
        turn[t][1] = sn;
    }
    double c0 = has ? value<BF16>(latent_pair.x) : 0.0, c1 = has ? value<BF16>(latent_pair.y) : 0.0;
    const double squares = dpp_wave_sum(c0 * c0 + c1 * c1);
    if (t % kWave == 0) part[t / kWave] = squares;
    __syncthreads();
    if (heads) {
        const double qc = turn[lane_pair][0], qs = turn[lane_pair][1];
        T *out = static_cast<T *>(p.q) + (long)r * p.heads * width + latent + lane_pair;
        const auto turn_query = [&](int h, Pair<BF16> q) {
            const double x = value<BF16>(q.x), y = value<BF16>(q.y);
            store<BF16>(out + (long)h * width, x * qc - y * qs);
            store<BF16>(out + (long)h * width + half, y * qc + x * qs);
        };
#pragma unroll
        for (int k = 0; k < kTurns; ++k)
            if (head0 + k * kPassHeads < heads) turn_query(head0 + k * kPassHeads, asked[k]);
        for (int h = head0 + kTurns * kPassHeads; h < heads; h += kPassHeads)
            turn_query(h, load_pair<BF16>(query + (long)h * p.head_width));
    }
    if (slot < 0) return;
    uint8_t *row = static_cast<uint8_t *>(b.data) + slot * latent_row_bytes(FP4, latent, b.rope);
    if (p.norm_w && has) {
        const double total = (part[0] + part[1]) + (part[2] + part[3]);
        const double inv = rsqrt(total / latent + (double)p.eps);
        c0 = c0 * inv * (double)w0;
        c1 = c1 * inv * (double)w1;
    }
    if constexpr (FP4) {
        // the 16 threads of 32 values.  Of a magnitude the upper half of its bits is enough, the
        // last one set if a lower one is: they are in the order of the magnitudes, NaN above
        // all, and show a mantissa of 1.5 and more than that apart.
        const auto upper = [](double v) {
            const unsigned long long u = __double_as_longlong(fabs(v));
            return (unsigned)(u >> 32) | ((unsigned)u != 0u ? 1u : 0u);
        };
        const unsigned u0 = upper(c0), u1 = upper(c1), top = row_max(u0 > u1 ? u0 : u1);
        const int exp = (int)(top >> 20) - 1023;  // top = 1.m * 2^exp <= 6 * 2^e = 1.5 * 2^(e + 2)
        const bool bad = exp >= 127;
        const int least = exp - ((top & 0xFFFFFu) > 0x80000u ? 1 : 2);
        const int e = bad ? 0 : least < kFp4LeastExp ? kFp4LeastExp : least;
        const double inv = power2(-e);
        if (has) {
            row[t] = bad ? (uint8_t)0 : fp4_codes(c0 * inv, c1 * inv);
            const int g = t / (kFp4Group / 2);
            if (t % (kFp4Group / 2) == 0)
                row[latent / 2 + 4 * (g % 4) + g / 4] = (uint8_t)(bad ? 255 : e + kFp4Bias);
        }
    } else if (has) {
        reinterpret_cast<unsigned *>(row)[t] = to_bf16(c0) | (unsigned)to_bf16(c1) << 16;
    }
    if (turns) {
        const double x = value<BF16>(rope_pair.x), y = value<BF16>(rope_pair.y);
        uint16_t *rope = reinterpret_cast<uint16_t *>(row + latent_part_bytes(FP4, latent));
        rope[t] = to_bf16(x * cs - y * sn);
        rope[half + t] = to_bf16(y * cs + x * sn);
    }
}

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// One token row a wave, 8 values a lane and step.  67 MB of ragged f32 rows 13.5-14 us (4.8-5.0 TB/s; a
// large copy reaches 5.2), 8192 rows of 4 bits, 13 MB, 5.3 (the way to a row and from it, three trips).
template <bool BF16, bool FP4>
__global__ __launch_bounds__(kThreads) void latent_gather_kernel(MlkLatentBatch b, int rows, void *to) {
    using T = typename Elem<BF16>::type;
    const long r = (long)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (r >= rows) return;
    int position;
    long slot;
    if (!place_of_row(b, (int)r, rows, &position, &slot)) return;
    const int latent = b.latent, width = latent + b.rope;
    const uint8_t *row = static_cast<const uint8_t *>(b.data) +
                         (slot < 0 ? 0 : slot) * latent_row_bytes(FP4, latent, b.rope);
    T *out = static_cast<T *>(to) + r * width;
    for (int c = 8 * (int)(threadIdx.x % kWave); c < width; c += 8 * kWave) {
        unsigned w[4];  // bf16 pairs
        if (slot < 0) {
            // padding, or a key that has no place
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = position < 0 ? 0u : 0x7FC07FC0u;
        } else if (FP4 && c < latent) {
            const unsigned codes = *reinterpret_cast<const unsigned *>(row + c / 2);
            const int g = c / kFp4Group;
            const float scale = __uint_as_float((unsigned)row[latent / 2 + 4 * (g % 4) + g / 4] << 23);
            const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
            const auto p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
            const auto p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
            const auto p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
            __builtin_memcpy(&w[0], &p0, 4);
            __builtin_memcpy(&w[1], &p1, 4);
            __builtin_memcpy(&w[2], &p2, 4);
            __builtin_memcpy(&w[3], &p3, 4);
        } else {
            const int at = FP4 ? latent_part_bytes(true, latent) + 2 * (c - latent) : 2 * c;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(row + at);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        }
        if constexpr (BF16) {
            *reinterpret_cast<u32x4_any *>(out + c) = u32x4_any{w[0], w[1], w[2], w[3]};
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<u32x4_any *>(out + c + 4 * h) =
                    u32x4_any{w[2 * h] << 16, w[2 * h] & 0xFFFF0000u, w[2 * h + 1] << 16,
                              w[2 * h + 1] & 0xFFFF0000u};
        }
    }
}

int launched() { return hipGetLastError() == hipSuccess ? kOk : kErrLaunch; }

}  // namespace

int latent_append(const MlkLatentBatch &b, const LatentAppend &p, hipStream_t stream) {
    const bool fp4 = b.type == MLK_FP4;
    auto kernel = p.bf16 ? (fp4 ? latent_append_kernel<true, true> : latent_append_kernel<true, false>)
                         : (fp4 ? latent_append_kernel<false, true> : latent_append_kernel<false, false>);
    kernel<<<p.rows, kThreads, 0, stream>>>(b, p);
    return launched();
}

int latent_gather(const MlkLatentBatch &b, bool bf16, int rows, void *out, hipStream_t stream) {
    const bool fp4 = b.type == MLK_FP4;
    auto kernel = bf16 ? (fp4 ? latent_gather_kernel<true, true> : latent_gather_kernel<true, false>)
                       : (fp4 ? latent_gather_kernel<false, true> : latent_gather_kernel<false, false>);
    kernel<<<(rows - 1) / kWaves + 1, kThreads, 0, stream>>>(b, rows, out);
    return launched();
}

}  // namespace mlh
