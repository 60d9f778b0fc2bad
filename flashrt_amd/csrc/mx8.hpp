// The values of 8-bit codes with a power-of-two scale per 32.
#pragma once

#include "common.hpp"

namespace frt {

// The fp32 value of a scale byte (0: the subnormal 2^-127, 255: NaN)
__device__ __forceinline__ float mx8_scale(uint32_t b) {
    return __builtin_bit_cast(float, b == 255u ? 0x7fc00000u : b ? b << 23 : 0x00400000u);
}
// Four codes' values, of a word, and eight, of two
__device__ __forceinline__ auto mx8_values(uint32_t w, float scale) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    f4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = float(int(w << (24 - 8 * j)) >> 24) * scale;
    return v;
}
__device__ __forceinline__ auto mx8_values(uint32_t lo, uint32_t hi, float scale) {
    const auto l = mx8_values(lo, scale), h = mx8_values(hi, scale);
    return __builtin_shufflevector(l, h, 0, 1, 2, 3, 4, 5, 6, 7);
}

}  // namespace frt
