// The E8M0 scale of a block, shared by BLOCK_SCALE_QUANTIZE and the 8-bit cache.
#pragma once

#include "common.cuh"

namespace dfgpu {
namespace {

// |x| bit patterns order like unsigned integers, and every NaN pattern is larger
// than +Inf, so an unsigned max over (bits & 0x7fffffff) is arith.maximumf over
// |x| with NaN propagation.
// `largest`: the largest finite value of the code type (448 for E4M3, 57344 for E5M2; SpecializedGraph.cpp:795-808).
__device__ __forceinline__ uint32_t scale_code_from_amax_bits(uint32_t amax_bits, float largest = 448.0f) {
    if (amax_bits > 0x7f800000u) return 0xffu;  // NaN block
    float desired = __fdiv_rn(__uint_as_float(amax_bits), largest);
    uint32_t bits = __float_as_uint(desired);
    if (bits == 0u) return 127u;            // desired > 0 is false -> scale 1.0
    if (bits == 0x7f800000u) return 0xfeu;  // +Inf saturates
    int exponent = static_cast<int>(bits >> 23);
    uint32_t mantissa = bits & 0x7fffffu;
    int n;  // ceil(log2(desired))
    if (exponent == 0) {
        int top = 31 - __clz(mantissa);
        n = top - 149 + ((mantissa & (mantissa - 1u)) != 0u ? 1 : 0);
    } else {
        n = exponent - 127 + (mantissa != 0u ? 1 : 0);
    }
    int code = n + 127;
    // 2^n below 2^-127 is nearest (in the linear distance the search uses) to code 0.
    return static_cast<uint32_t>(code < 0 ? 0 : (code > 254 ? 254 : code));
}

}  // namespace
}  // namespace dfgpu
