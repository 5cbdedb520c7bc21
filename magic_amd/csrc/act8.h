// Exponent and codes of a block of 32 columns kept in 8 bits (act8.hip has the format), for every kernel that writes them.
#pragma once
#include "common.h"

namespace magic {
namespace act8 {

__device__ __forceinline__ float pow2f(int e) {  // 2^e, -126 <= e <= 127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// amax of a block (its bits as an unsigned number: magnitudes compare like integers, NaN above infinity) -> stored exponent
__device__ __forceinline__ int block_exp(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255;
    const int k = (int)(amax_bits >> 23);                        // biased exponent, 0 for subnormals and zero
    int e = k - 6;
    if ((amax_bits & 0x7fffffu) >= 0x7f0000u) ++e;               // mantissa >= 127.5 / 64: would round to 128
    return e < 1 ? 1 : e;
}

// Codes of four values under stored exponent e (1 .. 249, or 255: zeros) in the bytes of a word.  x 2^-e is exact and at
// most 127 in size: added to 1.5 2^23 in a fused step it is rounded once, to the nearest even integer, which the sum's low
// byte then holds in two's complement.  Seven instructions for four codes; rounding, converting and shifting take twenty.
__device__ __forceinline__ uint32_t codes4(float x0, float x1, float x2, float x3, int e) {
    const float s = pow2f(127 - e), big = 12582912.f;
    const uint32_t a = __float_as_uint(fmaf(x0, s, big)), b = __float_as_uint(fmaf(x1, s, big));
    const uint32_t c = __float_as_uint(fmaf(x2, s, big)), d = __float_as_uint(fmaf(x3, s, big));
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return e == 255 ? 0u : lo | hi;
}

// largest of eight consecutive lanes (the swaps go through the lanes' own pipe, not the LDS)
__device__ __forceinline__ uint32_t max8(uint32_t m) {
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));        // quad: lanes 1 0 3 2
    m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));        // quad: lanes 2 3 0 1
    return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));    // the half row mirrored
}

}  // namespace act8
}  // namespace magic
