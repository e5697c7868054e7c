// View-dependent colour of one gaussian (py_compute_color, forward_pass.py:168-215), in fp64: shared by K1 and the
// stand-alone colour product, which therefore give the same floats and clamp flags.  Files that include it are compiled
// with -ffp-contract=off.
#pragma once
#include "precam.h"

// the 16 basis values of the unit direction (dx, dy, dz); those above `degree` are left unset
__device__ __forceinline__ void gs_sh_basis(int degree, double dx, double dy, double dz, double (&basis)[16]) {
    basis[0] = SH_C0;
    if (degree > 0) {
        basis[1] = -dy * SH_C1; basis[2] = dz * SH_C1; basis[3] = -dx * SH_C1;
        if (degree > 1) {
            const double xx = dx * dx, yy = dy * dy, zz = dz * dz, xy = dx * dy, yz = dy * dz, xz = dx * dz;
            basis[4] = SH_C2_0 * xy; basis[5] = SH_C2_1 * yz;
            basis[6] = SH_C2_2 * (2.0 * zz - xx - yy);
            basis[7] = SH_C2_3 * xz; basis[8] = SH_C2_4 * (xx - yy);
            if (degree > 2) {
                basis[9] = SH_C3_0 * dy * (3.0 * xx - yy);
                basis[10] = SH_C3_1 * xy * dz;
                basis[11] = SH_C3_2 * dy * (4.0 * zz - xx - yy);
                basis[12] = SH_C3_3 * dz * (2.0 * zz - 3.0 * xx - 3.0 * yy);
                basis[13] = SH_C3_4 * dx * (4.0 * zz - xx - yy);
                basis[14] = SH_C3_5 * dz * (xx - yy);
                basis[15] = SH_C3_6 * dx * (xx - 3.0 * yy);
            }
        }
    }
}

// colour and clamp flag of the three channels.  The colour is a float output (tolerance, not bits; the reference's own
// sums associate differently, :178-203): fused multiply-adds for the 48-term sums.
__device__ __forceinline__ void gs_sh_channels(int degree, const double (&basis)[16], const float (&coef)[48],
                                               float (&col)[3], uint8_t (&clamped)[3]) {
    const int nb = (degree + 1) * (degree + 1);
#pragma unroll
    for (int ch = 0; ch < 3; ch++) {
        double r = 0.0;
#pragma unroll
        for (int k = 0; k < 16; k++)
            if (k < nb) {
                float cf = coef[16 * ch + k];
#ifdef GS_K1_CVT_IN_LOOP
                asm volatile("" : "+v"(cf));        // keep the coefficient a float across views (48 VGPRs, not 96)
#endif
                r = __builtin_fma(basis[k], (double)cf, r);
            }
        r += .5;
        if (r < 0) { r = 0; clamped[ch] = 1; }
        col[ch] = (float)r;
    }
}
