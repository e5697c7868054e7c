// Opacity dropout (include/gsplat.h, "Opacity dropout"): leaves gaussian i out of view s with probability p and divides
// the opacities that stay by 1 - p.  No counterpart in the reference.
//
// The mask is never stored: gaussian i stays in view s iff word (s & 3) of Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011), evaluated at the counter (i, 0, low and high half of s >> 2) under
// the 64-bit seed as key, is at least round(p 2^32).  It depends on (seed, i, s) alone: not on the device, the rank that
// renders the view, the launch, or the number of gaussians.
//
// They have to move 4 + 4 V bytes per gaussian forward, 8 + 4 V backward, and to evaluate the generator once per gaussian
// and block of four view numbers -- once per view for the views a rank of a multi-rank job renders, whose numbers lie apart.
// That evaluation, some 70 instructions, bounds them: 10 M gaussians x 4 views of different blocks 60 us = 3.3 TB/s, the
// gradient 63 us; 1 M x 8 views 18.5 us.  A thread takes four gaussians (one: 86 and 151 us, two: 69 and 93).
#include "common.h"
#include <math.h>
#include <string.h>

namespace {

// N may be the largest int32
unsigned blocks_of(int32_t N) { return ((unsigned)N + 1023u) / 1024u; }      // 256 threads of PER_THREAD gaussians

// The views of a launch, grouped by the evaluation of the generator they share: up to four views of one block s >> 2, each
// with another word.  Built on the host; a number that is there twice starts a group of its own.
constexpr int MAX_DROP_GROUPS = 32, MAX_DROP_VIEWS = 64;
struct ViewGroups {
    uint64_t block[MAX_DROP_GROUPS];
    int8_t view[MAX_DROP_GROUPS][4];      // the launch's view that takes word k, -1: none
    int n;
};

// Nine of the generator's ten rounds; a view's word needs one of the last round's two products.
// The 64-bit products are what it spends its time on (17 that depend on the gaussian, at a quarter of the rate of other
// instructions), the exclusive ors come second: three operands each (two by two: 76 us instead of 60).
constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

struct State {
    uint32_t c0, c1, c2, c3;
};
__device__ __forceinline__ State nine_rounds(uint32_t index, uint64_t block, uint64_t seed) {
    State s{index, 0, (uint32_t)block, (uint32_t)(block >> 32)};
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 9; r++) {
        const uint64_t a = (uint64_t)M0 * s.c0, b = (uint64_t)M1 * s.c2;
        s = State{xor3((uint32_t)(b >> 32), s.c1, k0), (uint32_t)b, xor3((uint32_t)(a >> 32), s.c3, k1), (uint32_t)a};
        k0 += W0;
        k1 += W1;
    }
    return s;
}
// words 0, 1 (PAIR 0) or 2, 3 (PAIR 1) of the tenth round
template <int PAIR>
__device__ __forceinline__ void last_round(const State &s, uint64_t seed, uint32_t &first, uint32_t &second) {
    const uint64_t p = PAIR == 0 ? (uint64_t)M1 * s.c2 : (uint64_t)M0 * s.c0;
    first = PAIR == 0 ? xor3((uint32_t)(p >> 32), s.c1, (uint32_t)seed + 9u * W0)
                      : xor3((uint32_t)(p >> 32), s.c3, (uint32_t)(seed >> 32) + 9u * W1);
    second = (uint32_t)p;
}

__device__ __forceinline__ float activated(float x, int is_logit) { return is_logit ? 1.0f / (1.0f + expf(-x)) : x; }

// four neighbouring gaussians per thread: rows of N floats start at any multiple of 4 bytes
constexpr int PER_THREAD = 4;
typedef float row4 __attribute__((ext_vector_type(4), aligned(4)));

__global__ __launch_bounds__(256) void opacity_dropout_kernel(int N, const float *__restrict__ opacity, int is_logit,
                                                              uint32_t limit, float scale, uint64_t seed, const ViewGroups groups,
                                                              float *__restrict__ out) {
    const uint32_t i = (blockIdx.x * 256u + threadIdx.x) * PER_THREAD;
    if (i >= (uint32_t)N) return;
    const uint32_t n = min((uint32_t)PER_THREAD, (uint32_t)N - i);
    row4 x = {0, 0, 0, 0};
    if (n == PER_THREAD) x = *reinterpret_cast<const row4 *>(opacity + i);
    else
        for (uint32_t e = 0; e < n; e++) x[e] = opacity[i + e];
#pragma unroll
    for (int e = 0; e < PER_THREAD; e++) x[e] = activated(x[e], is_logit) * scale;
#pragma unroll 1
    for (int g = 0; g < groups.n; g++) {
        State s[PER_THREAD];
#pragma unroll
        for (int e = 0; e < PER_THREAD; e++) s[e] = nine_rounds(i + e, groups.block[g], seed);
#pragma unroll
        for (int pair = 0; pair < 2; pair++) {
            if (groups.view[g][2 * pair] < 0 && groups.view[g][2 * pair + 1] < 0) continue;
            uint32_t w[2][PER_THREAD];
#pragma unroll
            for (int e = 0; e < PER_THREAD; e++) {
                if (pair == 0) last_round<0>(s[e], seed, w[0][e], w[1][e]);
                else last_round<1>(s[e], seed, w[0][e], w[1][e]);
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int v = groups.view[g][2 * pair + k];
                if (v < 0) continue;
                row4 y;
#pragma unroll
                for (int e = 0; e < PER_THREAD; e++) y[e] = w[k][e] >= limit ? x[e] : 0.0f;
                float *p = out + ((size_t)v * N + i);
                if (n == PER_THREAD) *reinterpret_cast<row4 *>(p) = y;
                else
                    for (uint32_t e = 0; e < n; e++) p[e] = y[e];
            }
        }
    }
}

__global__ __launch_bounds__(256) void opacity_dropout_backward_kernel(int N, const float *__restrict__ opacity, int is_logit,
                                                                       uint32_t limit, float scale, uint64_t seed,
                                                                       const ViewGroups groups, const float *__restrict__ d_out,
                                                                       int accumulate, float *__restrict__ d_opacity) {
    const uint32_t i = (blockIdx.x * 256u + threadIdx.x) * PER_THREAD;
    if (i >= (uint32_t)N) return;
    const uint32_t n = min((uint32_t)PER_THREAD, (uint32_t)N - i);
    row4 sum = {0, 0, 0, 0};
#pragma unroll 1
    for (int g = 0; g < groups.n; g++) {
        row4 d[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {                   // in flight while the generator runs
            const int v = groups.view[g][k];
            d[k] = row4{0, 0, 0, 0};
            if (v < 0) continue;
            const float *p = d_out + ((size_t)v * N + i);
            if (n == PER_THREAD) d[k] = *reinterpret_cast<const row4 *>(p);
            else
                for (uint32_t e = 0; e < n; e++) d[k][e] = p[e];
        }
        State s[PER_THREAD];
#pragma unroll
        for (int e = 0; e < PER_THREAD; e++) s[e] = nine_rounds(i + e, groups.block[g], seed);
#pragma unroll
        for (int pair = 0; pair < 2; pair++) {
            if (groups.view[g][2 * pair] < 0 && groups.view[g][2 * pair + 1] < 0) continue;
#pragma unroll
            for (int e = 0; e < PER_THREAD; e++) {
                uint32_t w0, w1;
                if (pair == 0) last_round<0>(s[e], seed, w0, w1);
                else last_round<1>(s[e], seed, w0, w1);
                // selected: a NaN of a dropped gaussian stays out
                sum[e] += w0 >= limit ? d[2 * pair][e] : 0.0f;
                sum[e] += w1 >= limit ? d[2 * pair + 1][e] : 0.0f;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < PER_THREAD; e++) {
        if (e >= (int)n) break;
        float f = sum[e];
        if (is_logit) {
            const float o = activated(opacity[i + e], 1);
            f *= o * (1.0f - o);
        }
        f *= scale;
        d_opacity[i + e] = accumulate ? d_opacity[i + e] + f : f;
    }
}

int check_dropout(const char *who, gs_ctx *ctx, int32_t N, double p, int32_t n_views, const uint64_t *view_ids, uint32_t *limit,
                  float *scale) {
    GS_REQUIRE(ctx, "%s: ctx is NULL", who);
    GS_REQUIRE(N >= 0 && n_views >= 0, "%s: negative N or n_views", who);
    GS_REQUIRE(p >= 0.0 && p < 1.0 && floor(p * 4294967296.0 + 0.5) < 4294967296.0, "%s: p=%g not in [0, 1)", who, p);
    GS_REQUIRE(n_views == 0 || view_ids, "%s: the view numbers are NULL", who);
    *limit = (uint32_t)floor(p * 4294967296.0 + 0.5);
    *scale = (float)(1.0 / (1.0 - p));
    return GS_OK;
}

// the groups of view_ids[first..], as many as a launch takes; returns the number of views in them
int take_views(ViewGroups *out, const uint64_t *ids, int first, int n_views) {
    memset(out, 0, sizeof *out);
    int v = 0;
    for (; first + v < n_views && v < MAX_DROP_VIEWS; v++) {
        const uint64_t id = ids[first + v];
        int g = out->n - 1;
        if (g < 0 || out->block[g] != id >> 2 || out->view[g][id & 3] >= 0) {
            if (out->n == MAX_DROP_GROUPS) break;
            g = out->n++;
            out->block[g] = id >> 2;
            for (int k = 0; k < 4; k++) out->view[g][k] = -1;
        }
        out->view[g][id & 3] = (int8_t)v;
    }
    return v;
}

}  // namespace

extern "C" int gs_opacity_dropout(gs_ctx *ctx, int32_t N, const float *opacity, int32_t opacity_is_logit, double p, uint64_t seed,
                                  int32_t n_views, const uint64_t *view_ids, float *out) {
    uint32_t limit;
    float scale;
    const int rc = check_dropout("gs_opacity_dropout", ctx, N, p, n_views, view_ids, &limit, &scale);
    if (rc || N == 0 || n_views == 0) return rc;
    GS_REQUIRE(opacity && out, "gs_opacity_dropout: NULL array argument");
    GS_HIP(hipSetDevice(ctx->device));
    for (int done = 0; done < n_views;) {
        ViewGroups groups;
        const int n = take_views(&groups, view_ids, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_DROPOUT);
          hipLaunchKernelGGL(opacity_dropout_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N, opacity,
                             opacity_is_logit, limit, scale, seed, groups, out + (size_t)N * done); }
        GS_HIP(hipGetLastError());
        done += n;
    }
    return GS_OK;
}

extern "C" int gs_opacity_dropout_backward(gs_ctx *ctx, int32_t N, const float *opacity, int32_t opacity_is_logit, double p,
                                           uint64_t seed, int32_t n_views, const uint64_t *view_ids, const float *dL_dout,
                                           int32_t accumulate, float *dL_dopacity) {
    uint32_t limit;
    float scale;
    const int rc = check_dropout("gs_opacity_dropout_backward", ctx, N, p, n_views, view_ids, &limit, &scale);
    if (rc || N == 0) return rc;
    GS_REQUIRE(opacity && dL_dopacity && (n_views == 0 || dL_dout), "gs_opacity_dropout_backward: NULL array argument");
    GS_HIP(hipSetDevice(ctx->device));
    int done = 0;
    do {      // no views: one launch that writes zeros (or adds nothing)
        ViewGroups groups;
        const int n = take_views(&groups, view_ids, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_DROPOUT);
          hipLaunchKernelGGL(opacity_dropout_backward_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N, opacity,
                             opacity_is_logit, limit, scale, seed, groups, dL_dout + (size_t)N * done,
                             (accumulate || done > 0) ? 1 : 0, dL_dopacity); }
        GS_HIP(hipGetLastError());
        done += n;
    } while (done < n_views);
    return GS_OK;
}
