// bf16.h -- bfloat16 bits and values on the device (internal).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlh {

__device__ __forceinline__ float bf16_value(unsigned bits) { return __uint_as_float(bits << 16); }

// to the nearest bf16, ties to even; a NaN stays one
__device__ __forceinline__ unsigned bf16_bits(float v) {
    const unsigned u = __float_as_uint(v);
    if (v != v) return (u >> 16) | 0x40u;
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// The same of a 64-bit value, rounded once: the f32 in between is cut off, with its last
// bit set where that left something out, so that no tie appears or is lost.
__device__ __forceinline__ unsigned bf16_bits(double v) {
    float f = (float)v;
    if ((double)f != v) {
        unsigned u = __float_as_uint(f);
        if (fabs((double)f) > fabs(v)) --u;
        f = __uint_as_float(u | 1u);
    }
    return bf16_bits(f);
}

}  // namespace mlh
