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

}  // namespace mlh
