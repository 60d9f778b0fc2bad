// The values of 8-bit codes with a power-of-two scale per 32.
#pragma once

#include "common.hpp"

namespace frt {

// The fp32 value of a scale byte (0: the subnormal 2^-127, 255: NaN)
__device__ __forceinline__ float mx8_scale(uint32_t b) {
    return __builtin_bit_cast(float, b == 255u ? 0x7fc00000u : b ? b << 23 : 0x00400000u);
}
// Eight codes' values, two words of four codes each
__device__ __forceinline__ auto mx8_values(uint32_t lo, uint32_t hi, float scale) {
    typedef float f8 __attribute__((ext_vector_type(8)));
    f8 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = float(int(lo << (24 - 8 * j)) >> 24) * scale;
        v[j + 4] = float(int(hi << (24 - 8 * j)) >> 24) * scale;
    }
    return v;
}

}  // namespace frt
