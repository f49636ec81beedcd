// Integers of the 8-bit key/value cache as halves.
#pragma once
#include "common.h"

namespace cpmk {

// sixteen bytes as integers -> halves, exactly: 1024 + 128 + q has q in its last bits
__device__ __forceinline__ void halves_of(uint4_t p, half8_t& lo, half8_t& hi) {
    uint32_t h[8];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const uint32_t u = p[d] ^ 0x80808080u;
        h[2 * d] = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
        h[2 * d + 1] = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    }
    const half2_t off = {(half_t)1152.0f, (half_t)1152.0f};
    uint4_t a, b;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        a[d] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, h[d]) - off);
        b[d] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, h[4 + d]) - off);
    }
    lo = __builtin_bit_cast(half8_t, a);
    hi = __builtin_bit_cast(half8_t, b);
}

}  // namespace cpmk
