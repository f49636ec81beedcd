/* The rounding of the 8-bit key/value cache in exact integer arithmetic against the kernels' one product and one addition:
 *     round(127 x / a)  for every pair of positive finite fp16 numbers x <= a,
 *     round(q a / b)    for every q in 1 .. 127 and every pair a <= b whose exponents are at most 9 apart (further apart every result is 0),
 * halves away from zero.  (Both are odd functions of x and q: the product and the addition of 1.5 * 2^23, to nearest with ties to even, see no tie.) */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

static int low_byte(float q) {
    float t = q + 12582912.0f;
    uint32_t b;
    memcpy(&b, &t, 4);
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
    return ldexpf((float)m, e);
}

int main(void) {
    const float up = 1.0f + 0x1p-21f;
    long long differ = 0, pairs = 0;
#pragma omp parallel for schedule(dynamic, 64) reduction(+ : differ, pairs)
    for (int a = 1; a <= 0x7bff; ++a) {
        int64_t ma, mx;
        int ea, ex;
        parts(a, &ma, &ea);
        const float y = 127.0f / value(a) * up;
        for (int x = 0; x <= a; ++x) {
            parts(x, &mx, &ex);
            const int down = ea - ex;       /* >= 0 */
            const int64_t den = down > 40 ? 0 : ma << down;
            const int64_t want = den == 0 ? 0 : (2 * 127 * mx + den) / (2 * den);
            const float p = value(x) * y;
            differ += low_byte(p) != want;
            differ += low_byte(-p) != (int8_t)-want;
            ++pairs;
        }
    }
#pragma omp parallel for schedule(dynamic, 64) reduction(+ : differ, pairs)
    for (int b = 1024; b <= 2047; ++b)
        for (int down = 0; down <= 9; ++down)
            for (int a = 1024; a <= (down ? 2047 : b); ++a) {
                const float r = ldexpf((float)a, -down) / (float)b * up;
                for (int q = 1; q <= 127; ++q) {
                    const int64_t den = (int64_t)b << down, want = (2 * (int64_t)q * a + den) / (2 * den);
                    differ += low_byte((float)q * r) != want;
                    ++pairs;
                }
            }
    printf("%lld pairs, %lld differ\n", pairs, differ);
    return differ != 0;
}
