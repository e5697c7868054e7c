// The 32-byte record of a gaussian's 48 SH coefficients (include/gsplat.h, "Packed SH"), encoded and decoded in
// registers.  Shared by the conversion and colour kernels (sh_pack.hip), K1 (preprocess.hip) and K8 (param_bwd.hip), so
// every reader gets the same floats.
//
//   q0      half(c0 of r) | half(c0 of g) << 16 | half(c0 of b) << 32 | scale r << 48 | scale g << 56
//   q1..q3  channel r, g, b: E2M1 code of coefficient k = 1..15 at bit 4 (k - 1); bits 60..63 hold the low (r) and high
//           (g) half of scale b, 0 (b)
// A scale byte s stands for 2^(s - 127), 255 for NaN; a code is sign, two exponent bits, one mantissa bit:
// 0, .5, 1, 1.5, 2, 3, 4, 6.  The constant term carries the base colour (its magnitude is several times the others'), so
// it stays out of the block that shares a scale and keeps 11 significant bits.
#pragma once
#include "common.h"

constexpr int GS_SH_SCALE_MAX = 252;      // 6 * 2^(252 - 127) is finite
constexpr uint32_t GS_SH_SCALE_NAN = 255;
constexpr float GS_HALF_MAX = 65504.0f;

struct gs_sh_record {
    uint32_t w[8];
};

__device__ __forceinline__ gs_sh_record gs_sh_load(const uint4 *__restrict__ words, size_t i) {
    const uint4 a = words[2 * i], b = words[2 * i + 1];
    return gs_sh_record{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}

__device__ __forceinline__ uint32_t gs_sh_scale(const gs_sh_record &r, int ch) {
    return ch == 0 ? (r.w[1] >> 16) & 255u : ch == 1 ? r.w[1] >> 24 : (r.w[3] >> 28) | ((r.w[5] >> 28) << 4);
}

__device__ __forceinline__ float gs_half_bits(uint32_t h) {
    union { uint16_t u; _Float16 f; } c;
    c.u = (uint16_t)h;
    return (float)c.f;
}

// the 48 coefficients [channel][k], as floats
__device__ __forceinline__ void gs_sh_decode(const gs_sh_record &r, float (&coef)[48]) {
#pragma unroll
    for (int ch = 0; ch < 3; ch++) {
        coef[16 * ch] = gs_half_bits(ch == 0 ? r.w[0] & 0xffffu : ch == 1 ? r.w[0] >> 16 : r.w[1] & 0xffffu);
        const uint32_t s = gs_sh_scale(r, ch);
        const bool bad = s == GS_SH_SCALE_NAN;
#pragma unroll
        for (int k = 1; k < 16; k++) {
            const uint32_t c = r.w[2 + 2 * ch + (k - 1) / 8] >> (4 * ((k - 1) & 7));
            // the code's exponent and mantissa as the top bits of a float: 2^-126 of its value (.5 is a denormal there)
            const float f = __uint_as_float(((c & 8u) << 28) | ((c & 7u) << 22));
            coef[16 * ch + k] = bad ? __uint_as_float(0x7fc00000u) : ldexpf(f, (int)s - 1);
        }
    }
}

// scale byte of a block whose largest magnitude has the bits `amax`: the exponent of amax rounded to one mantissa bit
// (so that nothing up to 7/8 of the next power of two is pushed above 6), minus E2M1's largest exponent 2.
// The saturation that is left is that of magnitudes between 6 and 7 scales, to 6.
__device__ __forceinline__ uint32_t gs_sh_block_scale(uint32_t amax) {
    if (amax >= 0x7f800000u) return GS_SH_SCALE_NAN;
    const int e = (int)((amax + 0x00200000u) >> 23) - 2;
    return (uint32_t)(e < 0 ? 0 : e > GS_SH_SCALE_MAX ? GS_SH_SCALE_MAX : e);
}

// E2M1 code of v in a block of scale s (not NaN): to nearest, ties to the even code, 6 at most
__device__ __forceinline__ uint32_t gs_e2m1_code(float v, uint32_t s) {
    const float x = fabsf(v) * __uint_as_float((254u - s) << 23);     // exact, or below half the smallest step
    uint32_t c = (x > 0.25f) + (x >= 0.75f) + (x > 1.25f) + (x >= 1.75f) + (x > 2.5f) + (x >= 3.5f) + (x > 5.0f);
    return c | ((__float_as_uint(v) >> 28) & 8u);
}

// half-precision bits of a constant term: to nearest even; finite values saturate, infinities and NaN stay
__device__ __forceinline__ uint32_t gs_half_code(float v) {
    if (fabsf(v) < __uint_as_float(0x7f800000u)) v = fminf(fmaxf(v, -GS_HALF_MAX), GS_HALF_MAX);
    union { uint16_t u; _Float16 f; } c;
    c.f = (_Float16)v;
    return c.u;
}
