// The rounding of the 8-bit key/value cache (kv_cache.hip): q = round(127 x / a) and q' = round(q a / a'), halves away from zero, in one fused operation an element.
//
// 127 x / a (and q a / a') has numerator and denominator of at most 18 and 11 bits beside powers of two, so it lies exactly half-way between two integers or is off that
// point by at least 1 / (2 * 127 * 2047) = 2^-19 of its size.  The factor is (127 / a) (1 + 2^-21), rounded twice, so above 127 / a by 2^-21.5 to 2^-20.6 of itself; its product with x is not rounded before the
// addition of 1.5 * 2^23, whose last bit is 1: halves come out above the half-way point by 2^-21.5 at least, everything else stays on its side.  As every step is odd in x, halves of either
// sign go away from zero.  Plain C++, so that a program on the host can go through every pair with these same functions.
#pragma once

namespace cpmk {

// num / den for kv_shifted (den > 0)
template <class Float>
constexpr Float kv_factor(Float num, Float den) {
    return num / den * (1.0f + 0x1p-21f);
}

// The integer lies in the low bits of the result's (its low byte in the low byte).  An fma by name: left to the compiler, a product and an addition are one rounding or two.
template <class Float>
constexpr Float kv_shifted(Float x, Float factor) {
    return __builtin_fmaf(x, factor, 12582912.0f);
}

}  // namespace cpmk
