// Packed SH (include/gsplat.h): conversion of the 48 SH coefficients of a gaussian to and from their 32-byte record, the
// view-dependent colour computed from the record (the colour part of forward_pass, forward_pass.py:168-215) and its
// gradients (sh_backpass + kernel sh_grads, backward_pass.py:70-97, setup_gpu.py:256-303).  The reference keeps its
// coefficients in full precision only.
//
// All four kernels are bound by HBM: per gaussian 192 + 32 bytes (conversions), 44 + 15 V (colour of V views),
// 44 + 15 V + 204 (its gradients).  One thread per gaussian.
#include "common.h"
#include "sh_basis.h"
#include "sh_grad.h"
#include "sh_pack.h"

namespace {

// N may be the largest int32
unsigned blocks_of(int32_t N) { return ((unsigned)N + 255u) / 256u; }

constexpr int MAX_COLOR_VIEWS = 32;      // camera positions that one launch takes by value
struct Cameras {
    double pos[MAX_COLOR_VIEWS][3];
    int n;
};

__global__ __launch_bounds__(256) void sh_quantize_kernel(int N, const float4 *__restrict__ sh, uint4 *__restrict__ words) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)N) return;
    float c[48];
#pragma unroll
    for (int v = 0; v < 12; v++) {
        const float4 f = sh[(size_t)i * 12 + v];
        c[4 * v] = f.x; c[4 * v + 1] = f.y; c[4 * v + 2] = f.z; c[4 * v + 3] = f.w;
    }
    gs_sh_record r;
    uint32_t s[3];
#pragma unroll
    for (int ch = 0; ch < 3; ch++) {
        uint32_t amax = 0;
#pragma unroll
        for (int k = 1; k < 16; k++) amax = max(amax, __float_as_uint(c[16 * ch + k]) & 0x7fffffffu);
        s[ch] = gs_sh_block_scale(amax);
        uint32_t lo = 0, hi = 0;
        if (s[ch] != GS_SH_SCALE_NAN) {
#pragma unroll
            for (int k = 1; k < 16; k++) {
                const uint32_t code = gs_e2m1_code(c[16 * ch + k], s[ch]);
                if (k < 9) lo |= code << (4 * (k - 1)); else hi |= code << (4 * (k - 9));
            }
        }
        r.w[2 + 2 * ch] = lo; r.w[3 + 2 * ch] = hi;
    }
    r.w[0] = gs_half_code(c[0]) | gs_half_code(c[16]) << 16;
    r.w[1] = gs_half_code(c[32]) | s[0] << 16 | s[1] << 24;
    r.w[3] |= s[2] << 28;
    r.w[5] |= (s[2] >> 4) << 28;
    words[2 * (size_t)i] = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    words[2 * (size_t)i + 1] = make_uint4(r.w[4], r.w[5], r.w[6], r.w[7]);
}

__global__ __launch_bounds__(256) void sh_dequantize_kernel(int N, const uint4 *__restrict__ words, float4 *__restrict__ sh) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)N) return;
    float c[48];
    gs_sh_decode(gs_sh_load(words, i), c);
#pragma unroll
    for (int v = 0; v < 12; v++) sh[(size_t)i * 12 + v] = make_float4(c[4 * v], c[4 * v + 1], c[4 * v + 2], c[4 * v + 3]);
}

__global__ __launch_bounds__(256) void sh_color_kernel(int N, const uint4 *__restrict__ words, const float *__restrict__ means,
                                                       int degree, const Cameras cams, float *__restrict__ colors,
                                                       uint8_t *__restrict__ clamped) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)N) return;
    float coef[48];
    gs_sh_decode(gs_sh_load(words, i), coef);
    const double x = means[3 * (size_t)i], y = means[3 * (size_t)i + 1], z = means[3 * (size_t)i + 2];
#pragma unroll 1
    for (int v = 0; v < cams.n; v++) {
        double dx = x - cams.pos[v][0], dy = y - cams.pos[v][1], dz = z - cams.pos[v][2];
        const double inv = 1.0 / sqrt((dx * dx + dy * dy) + dz * dz);
        dx *= inv; dy *= inv; dz *= inv;
        double basis[16];
        gs_sh_basis(degree, dx, dy, dz, basis);
        float col[3];
        uint8_t cl[3] = {0, 0, 0};
        gs_sh_channels(degree, basis, coef, col, cl);
        const size_t o = 3 * ((size_t)v * N + i);
#pragma unroll
        for (int ch = 0; ch < 3; ch++) { colors[o + ch] = col[ch]; clamped[o + ch] = cl[ch]; }
    }
}

__global__ __launch_bounds__(256) void sh_color_backward_kernel(int N, const uint4 *__restrict__ words,
                                                                const float *__restrict__ means, int degree,
                                                                const Cameras cams, const uint8_t *__restrict__ clamped,
                                                                const float *__restrict__ d_colors, int accumulate,
                                                                float4 *__restrict__ d_sh, float *__restrict__ d_means) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)N) return;
    float coef[48], acc[48];
    gs_sh_decode(gs_sh_load(words, i), coef);
#pragma unroll
    for (int k = 0; k < 48; k++) acc[k] = 0.0f;
    const double x = means[3 * (size_t)i], y = means[3 * (size_t)i + 1], z = means[3 * (size_t)i + 2];
    double g_mean[3] = {0, 0, 0};
#pragma unroll 1
    for (int v = 0; v < cams.n; v++) {
        double dx = x - cams.pos[v][0], dy = y - cams.pos[v][1], dz = z - cams.pos[v][2];
        const double inv = 1.0 / sqrt((dx * dx + dy * dy) + dz * dz);
        dx *= inv; dy *= inv; dz *= inv;
        float basis[16], bx[16], by[16], bz[16], g[3];
        gs_sh_basis_grad(degree, (float)dx, (float)dy, (float)dz, basis, bx, by, bz);
        const size_t o = 3 * ((size_t)v * N + i);
#pragma unroll
        for (int ch = 0; ch < 3; ch++) g[ch] = clamped[o + ch] ? 0.0f : d_colors[o + ch];
        // w_k = sum over the channels of gradient x coefficient; dL/d(direction) = sum_k w_k grad Y_k
        const int nb = (degree + 1) * (degree + 1);
        float ex = 0.0f, ey = 0.0f, ez = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++)
            if (k < nb) {
                const float w = __builtin_fmaf(g[2], coef[32 + k], __builtin_fmaf(g[1], coef[16 + k], g[0] * coef[k]));
                ex = __builtin_fmaf(bx[k], w, ex);
                ey = __builtin_fmaf(by[k], w, ey);
                ez = __builtin_fmaf(bz[k], w, ez);
#pragma unroll
                for (int ch = 0; ch < 3; ch++) acc[16 * ch + k] = __builtin_fmaf(g[ch], basis[k], acc[16 * ch + k]);
            }
        // d = v / |v|: dL/dv = (dL/dd - d (d . dL/dd)) / |v|
        const double dot = dx * ex + dy * ey + dz * ez;
        g_mean[0] += ((double)ex - dx * dot) * inv;
        g_mean[1] += ((double)ey - dy * dot) * inv;
        g_mean[2] += ((double)ez - dz * dot) * inv;
    }
    float4 *out = d_sh + (size_t)i * 12;
#pragma unroll
    for (int v = 0; v < 12; v++) {
        float4 f = make_float4(acc[4 * v], acc[4 * v + 1], acc[4 * v + 2], acc[4 * v + 3]);
        if (accumulate) {
            const float4 old = out[v];
            f.x += old.x; f.y += old.y; f.z += old.z; f.w += old.w;
        }
        out[v] = f;
    }
#pragma unroll
    for (int k = 0; k < 3; k++) {
        const size_t o = 3 * (size_t)i + k;
        d_means[o] = accumulate ? d_means[o] + (float)g_mean[k] : (float)g_mean[k];
    }
}

int check_records(gs_ctx *ctx, const char *who, int32_t N, const void *words) {
    GS_REQUIRE(ctx, "%s: ctx is NULL", who);
    GS_REQUIRE(N >= 0, "%s: N=%d < 0", who, N);
    if (N == 0) return GS_OK;
    GS_REQUIRE(words, "%s: the packed records are NULL", who);
    GS_REQUIRE(((uintptr_t)words & 15) == 0, "%s: the packed records must be 16-byte aligned", who);
    return GS_OK;
}

int check_views(const char *who, int32_t degree, int32_t n_views, const double *cam_pos) {
    GS_REQUIRE(degree >= 0 && degree <= 3, "%s: degree %d not in 0..3", who, degree);
    GS_REQUIRE(n_views >= 0, "%s: n_views=%d < 0", who, n_views);
    GS_REQUIRE(n_views == 0 || cam_pos, "%s: the camera positions are NULL", who);
    return GS_OK;
}

int take_cameras(Cameras *c, const double *cam_pos, int first, int n_views) {
    c->n = n_views - first < MAX_COLOR_VIEWS ? n_views - first : MAX_COLOR_VIEWS;
    for (int v = 0; v < c->n; v++)
        for (int k = 0; k < 3; k++) c->pos[v][k] = cam_pos[3 * (first + v) + k];
    return c->n;
}

}  // namespace

extern "C" int gs_sh_quantize(gs_ctx *ctx, int32_t N, const float *sh, uint32_t *words) {
    const int rc = check_records(ctx, "gs_sh_quantize", N, words);
    if (rc || N == 0) return rc;
    GS_REQUIRE(sh && ((uintptr_t)sh & 15) == 0, "gs_sh_quantize: sh must be a 16-byte aligned array");
    GS_HIP(hipSetDevice(ctx->device));
    { gs_prof_scope prof_(ctx, GS_K_SH_PACK);
      hipLaunchKernelGGL(sh_quantize_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N,
                         reinterpret_cast<const float4 *>(sh), reinterpret_cast<uint4 *>(words)); }
    GS_HIP(hipGetLastError());
    return GS_OK;
}

extern "C" int gs_sh_dequantize(gs_ctx *ctx, int32_t N, const uint32_t *words, float *sh) {
    const int rc = check_records(ctx, "gs_sh_dequantize", N, words);
    if (rc || N == 0) return rc;
    GS_REQUIRE(sh && ((uintptr_t)sh & 15) == 0, "gs_sh_dequantize: sh must be a 16-byte aligned array");
    GS_HIP(hipSetDevice(ctx->device));
    { gs_prof_scope prof_(ctx, GS_K_SH_PACK);
      hipLaunchKernelGGL(sh_dequantize_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N,
                         reinterpret_cast<const uint4 *>(words), reinterpret_cast<float4 *>(sh)); }
    GS_HIP(hipGetLastError());
    return GS_OK;
}

extern "C" int gs_sh_color(gs_ctx *ctx, int32_t N, const uint32_t *words, const float *means, int32_t degree, int32_t n_views,
                           const double *cam_pos, float *colors, uint8_t *clamped) {
    int rc = check_records(ctx, "gs_sh_color", N, words);
    if (!rc) rc = check_views("gs_sh_color", degree, n_views, cam_pos);
    if (rc || N == 0 || n_views == 0) return rc;
    GS_REQUIRE(means && colors && clamped, "gs_sh_color: NULL array argument");
    GS_HIP(hipSetDevice(ctx->device));
    for (int done = 0; done < n_views;) {
        Cameras cams;
        const int n = take_cameras(&cams, cam_pos, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_SH_COLOR);
          hipLaunchKernelGGL(sh_color_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N,
                             reinterpret_cast<const uint4 *>(words), means, degree, cams, colors + 3 * (size_t)N * done,
                             clamped + 3 * (size_t)N * done); }
        GS_HIP(hipGetLastError());
        done += n;
    }
    return GS_OK;
}

extern "C" int gs_sh_color_backward(gs_ctx *ctx, int32_t N, const uint32_t *words, const float *means, int32_t degree,
                                    int32_t n_views, const double *cam_pos, const uint8_t *clamped, const float *dL_dcolors,
                                    int32_t accumulate, float *dL_dsh, float *dL_dmeans) {
    int rc = check_records(ctx, "gs_sh_color_backward", N, words);
    if (!rc) rc = check_views("gs_sh_color_backward", degree, n_views, cam_pos);
    if (rc || N == 0) return rc;
    GS_REQUIRE(means && dL_dsh && dL_dmeans && (n_views == 0 || (clamped && dL_dcolors)),
               "gs_sh_color_backward: NULL array argument");
    GS_REQUIRE(((uintptr_t)dL_dsh & 15) == 0, "gs_sh_color_backward: dL_dsh must be 16-byte aligned");
    GS_HIP(hipSetDevice(ctx->device));
    int done = 0;
    do {      // no views: one launch that writes zeros (or adds nothing)
        Cameras cams;
        const int n = take_cameras(&cams, cam_pos, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_SH_COLOR);
          hipLaunchKernelGGL(sh_color_backward_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N,
                             reinterpret_cast<const uint4 *>(words), means, degree, cams,
                             clamped + 3 * (size_t)N * done, dL_dcolors + 3 * (size_t)N * done,
                             (accumulate || done > 0) ? 1 : 0, reinterpret_cast<float4 *>(dL_dsh), dL_dmeans); }
        GS_HIP(hipGetLastError());
        done += n;
    } while (done < n_views);
    return GS_OK;
}
