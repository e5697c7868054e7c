// Packed SH (include/gsplat.h): conversion of the 48 SH coefficients of a gaussian to and from their 32-byte record, the
// view-dependent colour computed from the record (the colour part of forward_pass, forward_pass.py:168-215) and its
// gradients (sh_backpass + kernel sh_grads, backward_pass.py:70-97, setup_gpu.py:256-303).  The reference keeps its
// coefficients in full precision only.
//
// What they have to move per gaussian: 192 + 32 bytes (conversions), 44 + 15 V (colour of V views), 44 + 15 V + 204 (its
// gradients).  All are bound by HBM, at the 5.0-5.2 TB/s a large copy reaches or above, but for colours and gradients of many
// views, which the arithmetic of the view loop bounds (figures at the kernels).
#include "common.h"
#include "precam.h"
#include "sh_pack.h"

namespace {

// N may be the largest int32
unsigned blocks_of(int32_t N, unsigned per_block = 256) { return ((unsigned)N + per_block - 1) / per_block; }

constexpr int MAX_COLOR_VIEWS = 32;      // camera positions that one launch takes by value
struct Cameras {
    double pos[MAX_COLOR_VIEWS][3];
    int n;
};

// Outputs that nothing on the chip reads again before they have left its caches: non-temporal stores (dequantising 5 M
// gaussians 178 us against 192, gradients 1 view 10 M 426 against 446).
__device__ __forceinline__ void store_streaming(float4 *p, const float4 f) {
    typedef float vec4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(vec4{f.x, f.y, f.z, f.w}, reinterpret_cast<vec4 *>(p));
}

// The [N][48] floats that a wave's 64 threads hold leave through LDS: a column per thread on one side, memory order (12
// stores of 1 KiB of whole lines) on the other.  Threads that store their own 192 bytes write 64 quarter lines per store
// instead (dequantising 5 M gaussians 205 us against 302).  No other wave uses its columns: a fence of the wave on either side
// of the reads, no barrier.  The odd pitch keeps both sides free of bank conflicts.
// ROUNDS 2: 32 threads at a time, half the LDS, for a kernel that its waves gain by; where LDS does not limit them it costs
// (dequantising 5 M 208 us against 178).
template <int ROUNDS>
struct Columns {
    float4 q[12][256 / ROUNDS + 5];
};

// wave-uniform: the wave's first gaussian and how many it has (64, or fewer in the last wave)
struct Rows {
    uint32_t first, n;
};
__device__ __forceinline__ Rows wave_rows(int N) {
    const uint32_t first = blockIdx.x * 256u + (threadIdx.x & ~63u);
    return {first, first >= (uint32_t)N ? 0u : min(64u, (uint32_t)N - first)};
}

template <bool ADD, int ROUNDS>
__device__ __forceinline__ void registers_to_rows(Columns<ROUNDS> &s, const Rows r, const float (&c)[48], float4 *__restrict__ dst) {
    constexpr int COLS = 64 / ROUNDS;                    // the wave's columns
    const int lane = threadIdx.x & 63, col0 = (threadIdx.x >> 6) * COLS;
    float4 *p = dst + (size_t)r.first * 12;
#pragma unroll
    for (int round = 0; round < ROUNDS; round++) {
        wave_lds_fence();      // the previous round's columns have been read
        if (ROUNDS == 1 || lane / COLS == round) {
#pragma unroll
            for (int v = 0; v < 12; v++)
                s.q[v][col0 + lane % COLS] = make_float4(c[4 * v], c[4 * v + 1], c[4 * v + 2], c[4 * v + 3]);
        }
        wave_lds_fence();
#pragma unroll
        for (int k = 0; k < 12 / ROUNDS; k++) {
            const uint32_t j = k * 64 + lane;            // float4 j of the round: gaussian j / 12, quarter j % 12
            const uint32_t at = round * COLS * 12 + j;
            if (at < r.n * 12) {
                float4 f = s.q[j % 12][col0 + j / 12];
                if (ADD) {
                    const float4 old = p[at];
                    f.x += old.x; f.y += old.y; f.z += old.z; f.w += old.w;
                }
                store_streaming(p + at, f);
            }
        }
    }
}

// A thread per channel: its 64 bytes in four loads.  The three threads of a gaussian, which may sit in different waves, meet
// in LDS, and the records leave 16 bytes per thread.  5 M gaussians 200 us = 5.6 TB/s.  (1 M and 5 M when this was chosen: 40
// and 205 us; a thread per gaussian, twelve loads 192 bytes apart: 43 and 208; non-temporal loads drop the lines between
// them: 100 and 487.)
constexpr int QUANT_GAUSSIANS = 64;
__global__ __launch_bounds__(3 * QUANT_GAUSSIANS) void sh_quantize_kernel(int N, const float4 *__restrict__ sh,
                                                                          uint4 *__restrict__ words) {
    __shared__ uint4 s_row[3 * QUANT_GAUSSIANS];      // codes lo, hi; scale; half-precision constant
    const uint32_t first = blockIdx.x * (uint32_t)QUANT_GAUSSIANS;
    const uint32_t n = min((uint32_t)QUANT_GAUSSIANS, (uint32_t)N - first);
    if (threadIdx.x < 3 * n) {
        const float4 *p = sh + ((size_t)first * 3 + threadIdx.x) * 4;
        float c[16];
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const float4 f = p[v];
            c[4 * v] = f.x; c[4 * v + 1] = f.y; c[4 * v + 2] = f.z; c[4 * v + 3] = f.w;
        }
        uint32_t amax = 0;
#pragma unroll
        for (int k = 1; k < 16; k++) amax = max(amax, __float_as_uint(c[k]) & 0x7fffffffu);
        const uint32_t s = gs_sh_block_scale(amax);
        const bool bad = s == GS_SH_SCALE_NAN;
        uint32_t lo, hi;
        gs_sh_codes(c, s, lo, hi);
        s_row[threadIdx.x] = make_uint4(bad ? 0u : lo, bad ? 0u : hi, s, gs_half_code(c[0]));
    }
    __syncthreads();
    if (threadIdx.x >= 2 * n) return;
    const uint4 r = s_row[3 * (threadIdx.x >> 1)], g = s_row[3 * (threadIdx.x >> 1) + 1], b = s_row[3 * (threadIdx.x >> 1) + 2];
    words[2 * (size_t)first + threadIdx.x] =
        threadIdx.x & 1 ? make_uint4(g.x, g.y | (b.z >> 4) << 28, b.x, b.y)
                        : make_uint4(r.w | g.w << 16, b.w | r.z << 16 | g.z << 24, r.x, r.y | b.z << 28);
}

// 5 M gaussians 175 us = 6.4 TB/s.
__global__ __launch_bounds__(256) void sh_dequantize_kernel(int N, const uint4 *__restrict__ words, float4 *__restrict__ sh) {
    __shared__ Columns<1> s_col;
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    float c[48];
    gs_sh_decode(gs_sh_load(words, min(i, (uint32_t)N - 1)), c);
    registers_to_rows<false>(s_col, wave_rows(N), c, sh);
}

// ---- colour.  On the unit sphere the 16 basis functions are constants times these polynomials (x^2 + y^2 + z^2 = 1 turns
// 2zz - xx - yy into 3zz - 1 and so on); the signs are in the constants.
//   m0..3   1, y, z, x           m4..8  xy, yz, 3zz - 1, xz, xx - yy
//   m9..15  y (3xx - yy), xyz, y (5zz - 1), z (5zz - 3), x (5zz - 1), z (xx - yy), x (xx - 3yy)
__device__ constexpr double BASIS_CONST[16] = {SH_C0, -SH_C1, SH_C1, -SH_C1, SH_C2_0, SH_C2_1, SH_C2_2, SH_C2_3, SH_C2_4,
                                               SH_C3_0, SH_C3_1, SH_C3_2, SH_C3_3, SH_C3_4, SH_C3_5, SH_C3_6};

template <int DEGREE, typename T>
__device__ __forceinline__ void basis_polynomials(T x, T y, T z, T (&m)[16]) {
    m[0] = 1;
    if (DEGREE > 0) { m[1] = y; m[2] = z; m[3] = x; }
    if (DEGREE > 1) {
        const T xx = x * x, yy = y * y, zz = z * z;
        m[4] = x * y; m[5] = y * z; m[6] = 3 * zz - 1; m[7] = x * z; m[8] = xx - yy;
        if (DEGREE > 2) {
            const T q = 5 * zz - 1;
            m[9] = y * (3 * xx - yy); m[10] = m[4] * z; m[11] = y * q; m[12] = z * (q - 2); m[13] = x * q;
            m[14] = z * m[8]; m[15] = x * (xx - 3 * yy);
        }
    }
}

// 1 / sqrt(x) to the last bits of fp64: the hardware's 24-bit estimate and one step of third order
__device__ __forceinline__ double inverse_sqrt(double x) {
    const double y = __builtin_amdgcn_rsq(x);
    const double e = __builtin_fma(-x * y, y, 1.0);
    return __builtin_fma(y * e, __builtin_fma(0.375, e, 0.5), y);
}

struct Direction {
    double x, y, z, inv;      // unit vector from the camera, 1 / distance
};
__device__ __forceinline__ Direction direction(double x, double y, double z, const double (&cam)[3]) {
    Direction d{x - cam[0], y - cam[1], z - cam[2], 0};
    d.inv = inverse_sqrt(__builtin_fma(d.x, d.x, __builtin_fma(d.y, d.y, d.z * d.z)));
    d.x *= d.inv; d.y *= d.inv; d.z *= d.inv;
    return d;
}

// The colour as a polynomial a(x, y) + z b(x, y): zz = 1 - xx - yy leaves ten terms of degree 3 in a and six of degree 2 in
// b, as many as there are coefficients, and Horner's rule needs no monomials: 15 multiply-adds per channel and view.
struct Polynomial {
    double a[10], b[6];      // a: 1, x, xx, xxx, y, xy, xxy, yy, xyy, yyy;  b: 1, x, xx, y, xy, yy
};
template <int DEGREE>
__device__ __forceinline__ Polynomial polynomial(const float *coef) {
    double c[16];
#pragma unroll
    for (int k = 0; k < 16; k++) c[k] = k < (DEGREE + 1) * (DEGREE + 1) ? BASIS_CONST[k] * (double)coef[k] : 0.0;
    Polynomial p{};
    p.a[0] = 0.5 + c[0];
    if (DEGREE > 0) { p.a[1] = c[3]; p.a[4] = c[1]; p.b[0] = c[2]; }
    if (DEGREE > 1) {
        p.a[0] += 2 * c[6]; p.a[2] = c[8] - 3 * c[6]; p.a[5] = c[4]; p.a[7] = -c[8] - 3 * c[6];
        p.b[1] = c[7]; p.b[3] = c[5];
    }
    if (DEGREE > 2) {
        p.a[1] += 4 * c[13]; p.a[3] = c[15] - 5 * c[13]; p.a[4] += 4 * c[11]; p.a[6] = 3 * c[9] - 5 * c[11];
        p.a[8] = -3 * c[15] - 5 * c[13]; p.a[9] = -c[9] - 5 * c[11];
        p.b[0] += 2 * c[12]; p.b[2] = c[14] - 5 * c[12]; p.b[4] = c[10]; p.b[5] = -c[14] - 5 * c[12];
    }
    return p;
}
template <int DEGREE>
__device__ __forceinline__ double evaluate(const Polynomial &p, double x, double y, double z) {
    auto fma = [](double a, double b, double c) { return __builtin_fma(a, b, c); };
    if (DEGREE == 0) return p.a[0];
    if (DEGREE == 1) return fma(x, p.a[1], fma(y, p.a[4], fma(z, p.b[0], p.a[0])));
    if (DEGREE == 2) {
        const double a = fma(y, fma(y, p.a[7], fma(x, p.a[5], p.a[4])), fma(x, fma(x, p.a[2], p.a[1]), p.a[0]));
        return fma(z, fma(y, p.b[3], fma(x, p.b[1], p.b[0])), a);
    }
    const double a0 = fma(x, fma(x, fma(x, p.a[3], p.a[2]), p.a[1]), p.a[0]), a1 = fma(x, fma(x, p.a[6], p.a[5]), p.a[4]);
    const double a = fma(y, fma(y, fma(y, p.a[9], fma(x, p.a[8], p.a[7])), a1), a0);
    const double b = fma(y, fma(y, p.b[5], fma(x, p.b[4], p.b[3])), fma(x, fma(x, p.b[2], p.b[1]), p.b[0]));
    return fma(z, b, a);
}

// In fp64 from the difference of the positions on, as K1 evaluates colours: the flag is the sign of the sum.
// SEVERAL views are bound by the fp64 arithmetic of the view loop, and turning the coefficients into a Polynomial in front of
// it pays: 1 M gaussians x 8 views 33 us = 5.0 TB/s (39 without), 3 M x 4 views 59 (63).  Two views are even (1 M 15 us either
// way, 5 M 68 with, 64 without).  A single view does not earn it back and stays at the memory's rate without: 10 M gaussians
// 104 us (119 with; fastest launches, both sides under the profiler: outside it a call takes 96 us = 6.1 TB/s).
template <int DEGREE, bool SEVERAL>
__global__ __launch_bounds__(256, 4) void sh_color_kernel(int N, const uint4 *__restrict__ words, const float *__restrict__ means,
                                                          const Cameras cams, float *__restrict__ colors,
                                                          uint8_t *__restrict__ clamped) {
    constexpr int NB = (DEGREE + 1) * (DEGREE + 1);
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)N) return;
    float coef[48];
    gs_sh_decode(gs_sh_load(words, i), coef);
    const double x = means[3 * (size_t)i], y = means[3 * (size_t)i + 1], z = means[3 * (size_t)i + 2];
    const size_t o = 3 * (size_t)i;
    auto store = [&](size_t at, double r) {
        const bool c = r < 0;
        __builtin_nontemporal_store(c ? 0.0f : (float)r, colors + at);
        clamped[at] = c;
    };
    if (SEVERAL) {
        const Polynomial p[3] = {polynomial<DEGREE>(coef), polynomial<DEGREE>(coef + 16), polynomial<DEGREE>(coef + 32)};
#pragma unroll 1
        for (int v = 0; v < cams.n; v++) {
            const Direction d = direction(x, y, z, cams.pos[v]);
#pragma unroll
            for (int ch = 0; ch < 3; ch++) store(3 * (size_t)N * v + o + ch, evaluate<DEGREE>(p[ch], d.x, d.y, d.z));
        }
    } else {
        const Direction d = direction(x, y, z, cams.pos[0]);
        double m[16];
        basis_polynomials<DEGREE, double>(d.x, d.y, d.z, m);
#pragma unroll
        for (int ch = 0; ch < 3; ch++) {
            double r = 0.5;
#pragma unroll
            for (int k = 0; k < NB; k++) r = __builtin_fma(m[k] * BASIS_CONST[k], (double)coef[16 * ch + k], r);
            store(o + ch, r);
        }
    }
}

// fp32 behind the fp64 direction, as in K8: products and sums of a few dozen terms.  The constants of the basis are taken
// out of the sums: they are multiplied in behind the view loop.
// Few views are bound by the rows that are written: the coefficients are decoded once (10 M gaussians x 1 view 425 us = 6.2
// TB/s).  SEVERAL views are bound by the loop's loads and its 200 vector instructions, and gain more by a fourth wave per SIMD
// than they lose by decoding the record in every view (45 registers less) and storing in two rounds: 1 M x 8 views 77 us
// against 85, 3 M x 4 163 against 170, 1 M x 3 52 against 53; 10 M x 1 438 against 417, two views the same (1 M 42, 5 M 230).
template <int DEGREE, bool SEVERAL>
__global__ __launch_bounds__(256, SEVERAL ? 4 : 1) void sh_color_backward_kernel(
    int N, const uint4 *__restrict__ words, const float *__restrict__ means, const Cameras cams,
    const uint8_t *__restrict__ clamped, const float *__restrict__ d_colors, int accumulate, float4 *__restrict__ d_sh,
    float *__restrict__ d_means) {
    constexpr int NB = (DEGREE + 1) * (DEGREE + 1);
    __shared__ Columns<SEVERAL ? 2 : 1> s_col;
    const uint32_t own = blockIdx.x * 256u + threadIdx.x;
    const uint32_t i = min(own, (uint32_t)N - 1);      // threads behind the last gaussian repeat it and store nothing
    float coef[48], acc[48];
    gs_sh_record record = gs_sh_load(words, i);
    if (!SEVERAL) gs_sh_decode(record, coef);
#pragma unroll
    for (int k = 0; k < 48; k++) acc[k] = 0.0f;
    const double x = means[3 * (size_t)i], y = means[3 * (size_t)i + 1], z = means[3 * (size_t)i + 2];
    double g_mean[3] = {0, 0, 0};
    // a view's gradients and flags are fetched one view ahead of their use, flags or no flags: three loads whose latency
    // the view in front of them covers
    struct Inputs {
        float g[3];
        uint8_t clamped[3];
    };
    auto fetch = [&](int v) {
        Inputs in;
        const size_t o = 3 * ((size_t)v * N + i);
#pragma unroll
        for (int ch = 0; ch < 3; ch++) { in.g[ch] = d_colors[o + ch]; in.clamped[ch] = clamped[o + ch]; }
        return in;
    };
    Inputs next = {};
    if (cams.n > 0) next = fetch(0);
#pragma unroll 1
    for (int v = 0; v < cams.n; v++) {
        const Inputs in = next;
        next = fetch(min(v + 1, cams.n - 1));
        const Direction d = direction(x, y, z, cams.pos[v]);
        const float dx = (float)d.x, dy = (float)d.y, dz = (float)d.z;
        float m[16], w[16], g[3];
        basis_polynomials<DEGREE, float>(dx, dy, dz, m);
#pragma unroll
        for (int ch = 0; ch < 3; ch++) g[ch] = in.clamped[ch] ? 0.0f : in.g[ch];
        if (SEVERAL) {
#pragma unroll
            for (int k = 0; k < 8; k++) asm volatile("" : "+v"(record.w[k]));      // decoded here, not in front of the loop
            gs_sh_decode(record, coef);
        }
#pragma unroll
        for (int k = 0; k < NB; k++) {
            w[k] = (float)BASIS_CONST[k] * __builtin_fmaf(g[2], coef[32 + k], __builtin_fmaf(g[1], coef[16 + k], g[0] * coef[k]));
#pragma unroll
            for (int ch = 0; ch < 3; ch++) acc[16 * ch + k] = __builtin_fmaf(g[ch], m[k], acc[16 * ch + k]);
        }
        if (DEGREE == 0) continue;
        // e = sum_k w_k grad m_k.  The polynomials agree with the basis on the sphere only; the component along d, where
        // they differ, is projected out below.
        float ex = w[3], ey = w[1], ez = w[2];
        if (DEGREE > 1) {
            ex += dy * w[4] + dz * w[7] + 2 * dx * w[8];
            ey += dx * w[4] + dz * w[5] - 2 * dy * w[8];
            ez += dy * w[5] + 6 * dz * w[6] + dx * w[7];
        }
        if (DEGREE > 2) {
            const float q = 5 * dz * dz - 1, xy6 = 6 * m[4], xxyy3 = 3 * m[8];
            ex += xy6 * w[9] + m[5] * w[10] + q * w[13] + 2 * m[7] * w[14] + xxyy3 * w[15];
            ey += xxyy3 * w[9] + m[7] * w[10] + q * w[11] - 2 * m[5] * w[14] - xy6 * w[15];
            ez += m[4] * w[10] + 10 * m[5] * w[11] + 3 * q * w[12] + 10 * m[7] * w[13] + m[8] * w[14];
        }
        // d = v / |v|: dL/dv = (e - d (d . e)) / |v|
        const double dot = d.x * ex + d.y * ey + d.z * ez;
        g_mean[0] += (ex - d.x * dot) * d.inv;
        g_mean[1] += (ey - d.y * dot) * d.inv;
        g_mean[2] += (ez - d.z * dot) * d.inv;
    }
#pragma unroll
    for (int k = 0; k < 48; k++) acc[k] *= (float)BASIS_CONST[k & 15];
    if (accumulate) registers_to_rows<true>(s_col, wave_rows(N), acc, d_sh);
    else registers_to_rows<false>(s_col, wave_rows(N), acc, d_sh);
    if (own >= (uint32_t)N) return;
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
      hipLaunchKernelGGL(sh_quantize_kernel, dim3(blocks_of(N, QUANT_GAUSSIANS)), dim3(3 * QUANT_GAUSSIANS), 0, ctx->stream, N,
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
    // the degree is a template argument: its tests are a select per term otherwise
    constexpr decltype(&sh_color_kernel<0, false>) kernels[2][4] = {
        {sh_color_kernel<0, false>, sh_color_kernel<1, false>, sh_color_kernel<2, false>, sh_color_kernel<3, false>},
        {sh_color_kernel<0, true>, sh_color_kernel<1, true>, sh_color_kernel<2, true>, sh_color_kernel<3, true>}};
    for (int done = 0; done < n_views;) {
        Cameras cams;
        const int n = take_cameras(&cams, cam_pos, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_SH_COLOR);
          hipLaunchKernelGGL(kernels[n > 1][degree], dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N,
                             reinterpret_cast<const uint4 *>(words), means, cams, colors + 3 * (size_t)N * done,
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
    constexpr decltype(&sh_color_backward_kernel<0, false>) kernels[2][4] = {
        {sh_color_backward_kernel<0, false>, sh_color_backward_kernel<1, false>, sh_color_backward_kernel<2, false>,
         sh_color_backward_kernel<3, false>},
        {sh_color_backward_kernel<0, true>, sh_color_backward_kernel<1, true>, sh_color_backward_kernel<2, true>,
         sh_color_backward_kernel<3, true>}};
    int done = 0;
    do {      // no views: one launch that writes zeros (or adds nothing)
        Cameras cams;
        const int n = take_cameras(&cams, cam_pos, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_SH_COLOR);
          hipLaunchKernelGGL(kernels[n > 2][degree], dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N,
                             reinterpret_cast<const uint4 *>(words), means, cams,
                             clamped + 3 * (size_t)N * done, dL_dcolors + 3 * (size_t)N * done,
                             (accumulate || done > 0) ? 1 : 0, reinterpret_cast<float4 *>(dL_dsh), dL_dmeans); }
        GS_HIP(hipGetLastError());
        done += n;
    } while (done < n_views);
    return GS_OK;
}
