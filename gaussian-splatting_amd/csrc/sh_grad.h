// The SH basis and its partial derivatives in fp32 (setup_gpu.py:256-303 differentiates the same polynomials): shared by
// K8 and the stand-alone colour gradient.
#pragma once
#include "precam.h"

// values and d/dx, d/dy, d/dz of the 16 basis polynomials at the unit direction (dx, dy, dz); zero above `degree`
__device__ __forceinline__ void gs_sh_basis_grad(int degree, float dx, float dy, float dz, float (&basis)[16],
                                                 float (&bx)[16], float (&by)[16], float (&bz)[16]) {
#pragma unroll
    for (int k = 0; k < 16; k++) basis[k] = bx[k] = by[k] = bz[k] = 0.0f;
    constexpr float C0 = (float)SH_C0, C1 = (float)SH_C1;
    constexpr float C20 = (float)SH_C2_0, C21 = (float)SH_C2_1, C22 = (float)SH_C2_2, C23 = (float)SH_C2_3,
                    C24 = (float)SH_C2_4;
    constexpr float C30 = (float)SH_C3_0, C31 = (float)SH_C3_1, C32 = (float)SH_C3_2, C33 = (float)SH_C3_3,
                    C34 = (float)SH_C3_4, C35 = (float)SH_C3_5, C36 = (float)SH_C3_6;
    basis[0] = C0;
    if (degree > 0) {
        basis[1] = -dy * C1; by[1] = -C1;
        basis[2] = dz * C1;  bz[2] = C1;
        basis[3] = -dx * C1; bx[3] = -C1;
        if (degree > 1) {
            const float xx = dx * dx, yy = dy * dy, zz = dz * dz, xy = dx * dy, yz = dy * dz, xz = dx * dz;
            basis[4] = C20 * xy; bx[4] = C20 * dy; by[4] = C20 * dx;
            basis[5] = C21 * yz; by[5] = C21 * dz; bz[5] = C21 * dy;
            basis[6] = C22 * (2.0f * zz - xx - yy);
            bx[6] = -2.0f * C22 * dx; by[6] = -2.0f * C22 * dy; bz[6] = 4.0f * C22 * dz;
            basis[7] = C23 * xz; bx[7] = C23 * dz; bz[7] = C23 * dx;
            basis[8] = C24 * (xx - yy); bx[8] = 2.0f * C24 * dx; by[8] = -2.0f * C24 * dy;
            if (degree > 2) {
                basis[9] = C30 * dy * (3.0f * xx - yy);
                bx[9] = C30 * 6.0f * xy; by[9] = C30 * (3.0f * xx - 3.0f * yy);
                basis[10] = C31 * xy * dz;
                bx[10] = C31 * yz; by[10] = C31 * xz; bz[10] = C31 * xy;
                basis[11] = C32 * dy * (4.0f * zz - xx - yy);
                bx[11] = C32 * (-2.0f * xy); by[11] = C32 * (4.0f * zz - xx - 3.0f * yy); bz[11] = C32 * 8.0f * yz;
                basis[12] = C33 * dz * (2.0f * zz - 3.0f * xx - 3.0f * yy);
                bx[12] = C33 * (-6.0f * xz); by[12] = C33 * (-6.0f * yz); bz[12] = C33 * (6.0f * zz - 3.0f * xx - 3.0f * yy);
                basis[13] = C34 * dx * (4.0f * zz - xx - yy);
                bx[13] = C34 * (4.0f * zz - 3.0f * xx - yy); by[13] = C34 * (-2.0f * xy); bz[13] = C34 * 8.0f * xz;
                basis[14] = C35 * dz * (xx - yy);
                bx[14] = C35 * 2.0f * xz; by[14] = C35 * (-2.0f * yz); bz[14] = C35 * (xx - yy);
                basis[15] = C36 * dx * (xx - 3.0f * yy);
                bx[15] = C36 * (3.0f * xx - 3.0f * yy); by[15] = C36 * (-6.0f * xy);
            }
        }
    }
}
