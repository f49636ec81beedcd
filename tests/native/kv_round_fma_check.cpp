/* The rounding of the 8-bit key/value cache as its kernels compile it (csrc/kv_round.h) against exact integer arithmetic:
 *     round(127 x / a)  for every pair of finite fp16 numbers |x| <= a,
 *     round(q a / b)    for every q in -127 .. 127 and every pair of significands a, b with a's exponent at most 9 below b's (further below every result is 0),
 * halves away from zero; and the powers of two that the pairs leave out: exponents at both ends of the fp16 range. */
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include "kv_round.h"

static int low_byte(float x, float factor) {
    const float t = cpmk::kv_shifted(x, factor);
    uint32_t b;
    std::memcpy(&b, &t, 4);
    return (int8_t)(b & 0xff);
}

/* a positive fp16 number as significand * 2^exponent */
static void parts(int bits, int64_t* m, int* e) {
    const int x = bits >> 10;
    *m = (bits & 1023) | (x ? 1024 : 0);
    *e = (x ? x : 1) - 25;
}
static float value(int bits) {
    int64_t m;
    int e;
    parts(bits, &m, &e);
    return std::ldexp((float)m, e);
}
/* num / (den * 2^down), halves up */
static int64_t nearest(int64_t num, int64_t den, int down) {
    if (down > 40) return 0;
    den <<= down;
    return (2 * num + den) / (2 * den);
}

int main() {
    long long differ = 0, pairs = 0;
#pragma omp parallel for schedule(dynamic, 64) reduction(+ : differ, pairs)
    for (int a = 1; a <= 0x7bff; ++a) {
        int64_t ma, mx;
        int ea, ex;
        parts(a, &ma, &ea);
        const float y = cpmk::kv_factor(127.0f, value(a));
        for (int x = 0; x <= a; ++x) {
            parts(x, &mx, &ex);
            const int64_t want = nearest(127 * mx, ma, ea - ex);
            differ += low_byte(value(x), y) != want;
            differ += low_byte(-value(x), y) != -want;
            ++pairs;
        }
    }
    printf("%lld pairs of a value and a magnitude\n", pairs);
    pairs = 0;
#pragma omp parallel for schedule(dynamic, 64) reduction(+ : differ, pairs)
    for (int b = 1024; b <= 2047; ++b)
        for (int down = 0; down <= 9; ++down)
            for (int a = 1024; a <= (down ? 2047 : b); ++a) {
                const float r = cpmk::kv_factor(std::ldexp((float)a, -down), (float)b);
                for (int q = 0; q <= 127; ++q) {
                    const int64_t want = nearest((int64_t)q * a, b, down);
                    differ += low_byte((float)q, r) != want;
                    differ += low_byte((float)-q, r) != -want;
                    ++pairs;
                }
            }
    printf("%lld pairs of an integer and two magnitudes\n", pairs);
    /* the same quotients from magnitudes at the ends of the range, subnormal ones among them */
    const int ends[] = {1, 2, 3, 0x3ff, 0x400, 0x401, 0x7fff >> 4, 0x7bfe, 0x7bff};
    for (int b : ends)
        for (int a = 0; a <= b; ++a) {
            int64_t ma, mb;
            int ea, eb;
            parts(a, &ma, &ea);
            parts(b, &mb, &eb);
            const float r = cpmk::kv_factor(value(a), value(b));
            for (int q = 0; q <= 127; ++q) differ += low_byte((float)q, r) != nearest(q * ma, mb, eb - ea);
        }
    printf("%lld differ\n", differ);
    return differ != 0;
}
