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

typedef float gs_float2 __attribute__((ext_vector_type(2)));

// two codes (byte B of w) times the scale whose exponent bits `scale` holds: exact for every scale byte, NaN for 255
template <int B>
__device__ __forceinline__ void gs_e2m1_pair(uint32_t w, float scale, float &a, float &b) {
    const gs_float2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, B);
    a = v.x;
    b = v.y;
}

// The 48 coefficients [channel][k], as floats: 24 conversions by the hardware's own E2M1 instruction.
__device__ __forceinline__ void gs_sh_decode(const gs_sh_record &r, float (&coef)[48]) {
#pragma unroll
    for (int ch = 0; ch < 3; ch++) {
        float *c = coef + 16 * ch;
        c[0] = gs_half_bits(ch == 0 ? r.w[0] & 0xffffu : ch == 1 ? r.w[0] >> 16 : r.w[1] & 0xffffu);
        const float scale = __uint_as_float(gs_sh_scale(r, ch) << 23);
        const uint32_t lo = r.w[2 + 2 * ch], hi = r.w[3 + 2 * ch];
        float unused;                       // the last nibble belongs to a scale byte
        gs_e2m1_pair<0>(lo, scale, c[1], c[2]);
        gs_e2m1_pair<1>(lo, scale, c[3], c[4]);
        gs_e2m1_pair<2>(lo, scale, c[5], c[6]);
        gs_e2m1_pair<3>(lo, scale, c[7], c[8]);
        gs_e2m1_pair<0>(hi, scale, c[9], c[10]);
        gs_e2m1_pair<1>(hi, scale, c[11], c[12]);
        gs_e2m1_pair<2>(hi, scale, c[13], c[14]);
        gs_e2m1_pair<3>(hi, scale, c[15], unused);
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

// The 15 codes of a channel (c[1..15]) in a block of scale byte s, 255 excepted: to nearest, ties to the even code, 6 scales
// at most -- what the hardware's conversion does.
__device__ __forceinline__ void gs_sh_codes(const float *c, uint32_t s, uint32_t &lo, uint32_t &hi) {
    const float scale = __uint_as_float(s << 23);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, c[1], c[2], scale, 0);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, c[3], c[4], scale, 1);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, c[5], c[6], scale, 2);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(lo, c[7], c[8], scale, 3);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, c[9], c[10], scale, 0);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(hi, c[11], c[12], scale, 1);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(hi, c[13], c[14], scale, 2);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(hi, c[15], 0.0f, scale, 3);
}

// half-precision bits of a constant term: to nearest even; finite values saturate, infinities and NaN stay
__device__ __forceinline__ uint32_t gs_half_code(float v) {
    if (fabsf(v) < __uint_as_float(0x7f800000u)) v = fminf(fmaxf(v, -GS_HALF_MAX), GS_HALF_MAX);
    union { uint16_t u; _Float16 f; } c;
    c.f = (_Float16)v;
    return c.u;
}
