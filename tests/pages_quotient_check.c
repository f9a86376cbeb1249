/*
 * Exhaustive host check of the quantizers' quotient (hy-nomas_amd/csrc/hn_common.h, struct
 * Quot) for the scale rule amax * fl(1 / 448) (127) of the paged write: for every bf16 row
 * maximum amax > 0 and every bf16 x with |x| <= amax, both signs,
 *
 *     y = fl(x * r), r = fl(1 / s);  e = fma(-s, y, x);  q = copysign(fma(e, r, y), x)
 *
 * gives the code of fl32(x / s). Rows with s < 2^-100 take the IEEE division in the
 * kernels and are skipped here.
 *
 * Build: gcc -O2 -fopenmp -ffp-contract=off pages_quotient_check.c ../oracle/fp8_oracle.c -lm
 */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

uint8_t hn_oracle_e4m3_encode(float f);

static float from_bits(uint32_t u) { float x; memcpy(&x, &u, 4); return x; }

static int int8_code(float v)
{
    float r = v >= 0.0f ? floorf(v + 0.5f) : ceilf(v - 0.5f);
    return (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

int main(void)
{
    int failed = 0;
    for (int int8 = 0; int8 < 2; ++int8) {
        const float inv = 1.0f / (int8 ? 127.0f : 448.0f);
        unsigned long long pairs = 0, bad = 0, past = 0;
#pragma omp parallel for schedule(dynamic, 64) reduction(+ : pairs, bad, past)
        for (uint32_t ab = 1; ab < 0x7F80u; ++ab) {
            const float amax = from_bits(ab << 16), s = amax * inv;
            if (!(s >= 0x1p-100f)) continue;
            const float r = 1.0f / s;
            /* the hardware conversion is checked up to 448.5 */
            past += !int8 && amax / s > 448.5f;
            for (uint32_t xs = 0; xs <= 2 * ab + 1; ++xs) {
                const float x = from_bits(((xs >> 1) << 16) | ((xs & 1u) << 31));
                const float exact = x / s, y = x * r, e = fmaf(-s, y, x), q = copysignf(fmaf(e, r, y), x);
                ++pairs;
                if (int8) bad += int8_code(q) != int8_code(exact);
                else bad += hn_oracle_e4m3_encode(q) != hn_oracle_e4m3_encode(exact);
            }
        }
        printf("%s: %llu pairs checked, %llu code mismatches, %llu rows past 448.5\n", int8 ? "amax*(1/127)" : "amax*(1/448)",
               pairs, bad, past);
        failed |= bad != 0 || past != 0;
    }
    return failed;
}
