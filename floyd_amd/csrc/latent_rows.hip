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

template <bool BF16> struct Elem { using type = float; };
template <> struct Elem<true> { using type = uint16_t; };

template <bool BF16> __device__ __forceinline__ double value(typename Elem<BF16>::type v) {
    if constexpr (BF16) return (double)bf16_value(v);
    else return (double)v;
}
template <bool BF16> __device__ __forceinline__ void store(typename Elem<BF16>::type *p, double v) {
    if constexpr (BF16) *p = (uint16_t)bf16_bits((float)v);
    else *p = (float)v;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}

// The sequence of token row r (b.seqs: none), by every lane of a wave: the number of
// sequences that end at r or before.
__device__ __forceinline__ int seq_of_row(const MlkLatentBatch &b, int r) {
    if (!b.row_starts) return r < b.seqs ? r : b.seqs;
    int before = 0;
    for (int s0 = 0; s0 < b.seqs; s0 += kWave) {
        const int s = s0 + (int)(threadIdx.x % kWave);
        const bool ends = s < b.seqs && b.row_starts[s + 1] <= r;
        before += __popcll(__ballot(ends));
    }
    return before;
}

// Key position of token row r (below 0: padding) and its place in the pages (-1: none);
// false: r is no row of a sequence.
__device__ __forceinline__ bool place_of_row(const MlkLatentBatch &b, int r, int rows, int *position,
                                             long *slot) {
    const int s = seq_of_row(b, r);
    if (s >= b.seqs) return false;
    const LatentSeq q = latent_seq(b, s, rows);
    if (r < q.begin || r >= q.begin + q.count) return false;
    const long j = (long)q.length - (q.begin + q.count - r);
    *position = j < 0 ? -1 : (int)j;
    *slot = j < 0 ? -1 : latent_slot(b, s, (unsigned)j);
    return true;
}

// 2^e of a double, e in its normal range.
__device__ __forceinline__ double power2(int e) {
    return __longlong_as_double((long long)(e + 1023) << 52);
}

// The e2m1 code nearest to v (|v| <= 6), ties to even.
__device__ __forceinline__ unsigned fp4_code(double v) {
    const double a = fabs(v);
    const unsigned m = (a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) +
                       (a > 5.0);
    return m | (v < 0.0 ? 8u : 0u);
}

// One token row a workgroup.
template <bool BF16, bool FP4>
__global__ __launch_bounds__(kThreads) void latent_append_kernel(MlkLatentBatch b, LatentAppend p) {
    using T = typename Elem<BF16>::type;
    __shared__ double part[kWaves];
    __shared__ double turn[kLatentRopeMax / 2][2];
    const int r = blockIdx.x, t = threadIdx.x;
    const int latent = b.latent, half = b.rope / 2;
    // thread t: latent values 2t and 2t + 1
    const T *kv = static_cast<const T *>(p.kv) + (long)r * p.kv_stride;
    const bool has = 2 * t < latent;
    double c0 = has ? value<BF16>(kv[2 * t]) : 0.0, c1 = has ? value<BF16>(kv[2 * t + 1]) : 0.0;
    int position;
    long slot;
    if (!place_of_row(b, r, p.rows, &position, &slot) || position < 0) return;
    if (t < half) {
        double sn, cs;
        sincos((double)position * (double)p.inv_freq[t], &sn, &cs);
        turn[t][0] = cs;
        turn[t][1] = sn;
    }
    const double squares = wave_sum64(c0 * c0 + c1 * c1);
    if (t % kWave == 0) part[t / kWave] = squares;
    __syncthreads();
    if (p.query) {
        const T *query = static_cast<const T *>(p.query) + (long)r * p.query_stride;
        T *q = static_cast<T *>(p.q) + (long)r * p.heads * (latent + b.rope);
        for (int j = t; j < p.heads * half; j += kThreads) {
            const int h = j / half, i = j - h * half;
            const T *in = query + (long)(h + 1) * p.head_width - b.rope + 2 * i;
            const double x = value<BF16>(in[0]), y = value<BF16>(in[1]);
            T *out = q + (long)h * (latent + b.rope) + latent + i;
            store<BF16>(out, x * turn[i][0] - y * turn[i][1]);
            store<BF16>(out + half, y * turn[i][0] + x * turn[i][1]);
        }
    }
    if (slot < 0) return;
    uint8_t *row = static_cast<uint8_t *>(b.data) + slot * latent_row_bytes(FP4, latent, b.rope);
    if (p.norm_w && has) {
        const double total = (part[0] + part[1]) + (part[2] + part[3]);
        const double inv = 1.0 / sqrt(total / latent + (double)p.eps);
        c0 = c0 * inv * (double)p.norm_w[2 * t];
        c1 = c1 * inv * (double)p.norm_w[2 * t + 1];
    }
    if constexpr (FP4) {
        // the 16 threads of 32 values; magnitudes in the order of their bits, NaN above all
        const long long a0 = __double_as_longlong(fabs(c0)), a1 = __double_as_longlong(fabs(c1));
        long long top = a0 > a1 ? a0 : a1;
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {
            const long long other = __shfl_xor(top, o, kWave);
            top = other > top ? other : top;
        }
        const int exp = (int)(top >> 52) - 1023;  // top = 1.m * 2^exp <= 6 * 2^e = 1.5 * 2^(e + 2)
        const bool above = (top & 0xFFFFFFFFFFFFFLL) > 0x8000000000000LL;
        const bool bad = exp >= 127;
        const int least = exp - (above ? 1 : 2);
        const int e = bad ? 0 : least < kFp4LeastExp ? kFp4LeastExp : least;
        const double inv = power2(-e);
        if (has) {
            row[t] = bad ? (uint8_t)0 : (uint8_t)(fp4_code(c0 * inv) | (fp4_code(c1 * inv) << 4));
            const int g = t / (kFp4Group / 2);
            if (t % (kFp4Group / 2) == 0)
                row[latent / 2 + 4 * (g % 4) + g / 4] = (uint8_t)(bad ? 255 : e + kFp4Bias);
        }
    } else if (has) {
        reinterpret_cast<unsigned *>(row)[t] = bf16_bits((float)c0) | (bf16_bits((float)c1) << 16);
    }
    if (t < half) {
        const double x = value<BF16>(kv[latent + 2 * t]), y = value<BF16>(kv[latent + 2 * t + 1]);
        uint16_t *rope = reinterpret_cast<uint16_t *>(row + latent_part_bytes(FP4, latent));
        rope[t] = (uint16_t)bf16_bits((float)(x * turn[t][0] - y * turn[t][1]));
        rope[half + t] = (uint16_t)bf16_bits((float)(y * turn[t][0] + x * turn[t][1]));
    }
}

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// One token row a wave, 8 values a lane and step.
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
