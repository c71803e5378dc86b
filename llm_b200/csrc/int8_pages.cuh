// A paged cache held in 8 bits: pages of LLMB_PAGE positions, whole numbers q [pages, kv heads, 64, dim] with 32-bit scales
// s [pages, kv heads, 64 / block]; q * s is the value that is held.
//
// Scales are powers of two, the smallest with which the largest value of a block of positions is at most 127 steps. So x / s has no
// rounding but that to a whole number, a block whose scale grows divides what it holds by a power of two, and q * s is exact in bfloat16 and in 32
// bits; what that costs is up to one of the 8 bits (127 steps become 64 just above a power of two). A block that took in a value that is not
// finite has a scale that is no number, and so is all that is read from it; its whole numbers are finite whatever they are.
#pragma once

#include "common.cuh"

namespace llmb {

constexpr uint32_t NOT_FINITE = 0x7f800000u;      // magnitudes (bits of |x|) from here on

// The scale for a largest magnitude, as bits: |x| = 1.f * 2^(e - 127) takes 2^(e - 133) while 1.f <= 127 / 64, twice that above.
__device__ __forceinline__ uint32_t scale_bits(uint32_t magnitude) {
    if (magnitude >= NOT_FINITE) return 0x7fffffffu;
    int exponent = (int)(magnitude >> 23) - 6 + ((magnitude & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return (uint32_t)max(exponent, 1) << 23;
}
__device__ __forceinline__ bool is_number(float s) { return (__float_as_uint(s) & 0x7fffffffu) < NOT_FINITE; }

}  // namespace llmb
