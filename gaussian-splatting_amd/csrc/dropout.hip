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
// That evaluation, some 70 instructions, bounds them where every view needs its own: 10 M gaussians x 4 views 56 us = 3.6
// TB/s, the gradient 61 us; 1 M x 8 views 15 us and 16 us.  Consecutive view numbers, as a training on one GPU counts them,
// share evaluations and come to the memory's rate: 35 us = 5.7 TB/s and 44 us = 5.5 TB/s; 9.6 us and 10.5 us.
#include "common.h"
#include <math.h>
#include <string.h>

namespace {

// The views of a launch, grouped by the evaluation of the generator they share: up to four views of one block s >> 2, each
// with another word.  Built on the host; a number that is there twice starts a group of its own.  A group is one 16-byte
// scalar load in the kernels.
constexpr int MAX_DROP_GROUPS = 32, MAX_DROP_VIEWS = 64;
constexpr uint32_t NO_VIEW = 255;
struct alignas(16) ViewGroup {
    uint64_t block;
    uint32_t views;           // byte k: the launch's view that takes word k, or NO_VIEW
    uint32_t unused;
    __host__ __device__ uint32_t view(int k) const { return (views >> (8 * k)) & 255u; }
};
struct ViewGroups {
    ViewGroup g[MAX_DROP_GROUPS];
    int n;
};

// Nine of the generator's ten rounds; a view's word needs one of the last round's two products.
// The 64-bit products are what it spends its time on (17 that depend on the gaussian, at a quarter of the rate of other
// instructions), the exclusive ors come second: three operands each (two by two: 76 us instead of 57).
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

// sigmoid'(x) = e / (1 + e)^2 with e = exp(-|x|): six roundings at every x.  (o (1 - o) cancels where o is close to 1: 1 % off
// at x = 12, exactly 0 from 17.4 on, where the value is 2.8e-8.)
__device__ __forceinline__ float sigmoid_derivative(float x) {
    const float e = expf(-fabsf(x)), d = 1.0f + e;
    return e / (d * d);
}

// PER neighbouring gaussians per thread, loaded and stored together; rows of N floats start at any multiple of 4 bytes.
// `all` is uniform in a block: the last block of a launch goes element by element.
template <int PER>
struct Row {
    typedef float vec __attribute__((ext_vector_type(PER), aligned(4)));
    float v[PER];
    __device__ __forceinline__ void load(const float *p, bool all, uint32_t n) {
        if (all) {
            const vec t = *reinterpret_cast<const vec *>(p);
#pragma unroll
            for (int e = 0; e < PER; e++) v[e] = t[e];
        } else {
#pragma unroll
            for (int e = 0; e < PER; e++) v[e] = e < (int)n ? p[e] : 0.0f;
        }
    }
    __device__ __forceinline__ void store(float *p, bool all, uint32_t n) const {
        if (all) {
            vec t;
#pragma unroll
            for (int e = 0; e < PER; e++) t[e] = v[e];
            *reinterpret_cast<vec *>(p) = t;
        } else {
#pragma unroll
            for (int e = 0; e < PER; e++)
                if (e < (int)n) p[e] = v[e];
        }
    }
};
template <>
struct Row<1> {
    float v[1];
    __device__ __forceinline__ void load(const float *p, bool, uint32_t) { v[0] = *p; }
    __device__ __forceinline__ void store(float *p, bool, uint32_t) const { *p = v[0]; }
};

template <int PER>
__global__ __launch_bounds__(256) void opacity_dropout_kernel(int N, const float *__restrict__ opacity, int is_logit,
                                                              uint32_t limit, float scale, uint64_t seed, const ViewGroups groups,
                                                              float *__restrict__ out) {
    const uint32_t i = (blockIdx.x * 256u + threadIdx.x) * PER;
    if (i >= (uint32_t)N) return;
    const bool all = (blockIdx.x + 1) * (256u * PER) <= (uint32_t)N;
    const uint32_t n = min((uint32_t)PER, (uint32_t)N - i);
    Row<PER> x;
    x.load(opacity + i, all, n);
#pragma unroll
    for (int e = 0; e < PER; e++) x.v[e] = activated(x.v[e], is_logit) * scale;
#pragma unroll 1
    for (int g = 0; g < groups.n; g++) {
        const ViewGroup group = groups.g[g];
        State s[PER];
#pragma unroll
        for (int e = 0; e < PER; e++) s[e] = nine_rounds(i + e, group.block, seed);
#pragma unroll
        for (int pair = 0; pair < 2; pair++) {
            if (group.view(2 * pair) == NO_VIEW && group.view(2 * pair + 1) == NO_VIEW) continue;
            uint32_t w[2][PER];
#pragma unroll
            for (int e = 0; e < PER; e++) {
                if (pair == 0) last_round<0>(s[e], seed, w[0][e], w[1][e]);
                else last_round<1>(s[e], seed, w[0][e], w[1][e]);
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t v = group.view(2 * pair + k);
                if (v == NO_VIEW) continue;
                Row<PER> y;
#pragma unroll
                for (int e = 0; e < PER; e++) y.v[e] = w[k][e] >= limit ? x.v[e] : 0.0f;
                y.store(out + ((size_t)v * N + i), all, n);
            }
        }
    }
}

template <int PER>
__global__ __launch_bounds__(256) void opacity_dropout_backward_kernel(int N, const float *__restrict__ opacity, int is_logit,
                                                                       uint32_t limit, float scale, uint64_t seed,
                                                                       const ViewGroups groups, const float *__restrict__ d_out,
                                                                       int accumulate, float *__restrict__ d_opacity) {
    const uint32_t i = (blockIdx.x * 256u + threadIdx.x) * PER;
    if (i >= (uint32_t)N) return;
    const bool all = (blockIdx.x + 1) * (256u * PER) <= (uint32_t)N;
    const uint32_t n = min((uint32_t)PER, (uint32_t)N - i);
    Row<PER> sum = {};
    bool kept[PER] = {};                                // by one of the views
#pragma unroll 1
    for (int g = 0; g < groups.n; g++) {
        const ViewGroup group = groups.g[g];
        Row<PER> d[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {                   // in flight while the generator runs
            const uint32_t v = group.view(k);
            d[k] = {};
            if (v != NO_VIEW) d[k].load(d_out + ((size_t)v * N + i), all, n);
        }
        State s[PER];
#pragma unroll
        for (int e = 0; e < PER; e++) s[e] = nine_rounds(i + e, group.block, seed);
#pragma unroll
        for (int pair = 0; pair < 2; pair++) {
            const bool has0 = group.view(2 * pair) != NO_VIEW, has1 = group.view(2 * pair + 1) != NO_VIEW;
            if (!has0 && !has1) continue;
#pragma unroll
            for (int e = 0; e < PER; e++) {
                uint32_t w0, w1;
                if (pair == 0) last_round<0>(s[e], seed, w0, w1);
                else last_round<1>(s[e], seed, w0, w1);
                // selected: a NaN of a dropped gaussian stays out
                sum.v[e] += w0 >= limit ? d[2 * pair].v[e] : 0.0f;
                sum.v[e] += w1 >= limit ? d[2 * pair + 1].v[e] : 0.0f;
                kept[e] |= (has0 && w0 >= limit) || (has1 && w1 >= limit);
            }
        }
    }
    Row<PER> r;
    if (is_logit) {
        r.load(opacity + i, all, n);
#pragma unroll
        for (int e = 0; e < PER; e++) sum.v[e] = kept[e] ? sum.v[e] * sigmoid_derivative(r.v[e]) : 0.0f;      // 0 times a NaN
    }
    if (accumulate) r.load(d_opacity + i, all, n);
#pragma unroll
    for (int e = 0; e < PER; e++) r.v[e] = accumulate ? r.v[e] + sum.v[e] * scale : sum.v[e] * scale;
    r.store(d_opacity + i, all, n);
}

// Gaussians per thread: four share a view's scalar work and store 16 bytes at once, but leave small scenes with few waves.
// us forward / backward of the kernels with one and with four (profiler, fastest launches): 10 k x 8 views 4.4 / 5.1 and
// 6.9 / 8.4, 300 k x 8 7.2 / 7.8 and 9.2 / 9.0, 524 k x 8 9.0 / 10.0 and 9.9 / 10.7, 1 M x 8 14.3 / 15.1 and 14.1 / 15.1,
// 10 M x 4 64 / 82 and 54 / 61.
inline int per_thread(int32_t N) { return N >= (1 << 19) ? 4 : 1; }

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
        const int k = (int)(id & 3);
        ViewGroup *g = out->n ? &out->g[out->n - 1] : nullptr;
        if (!g || g->block != id >> 2 || g->view(k) != NO_VIEW) {
            if (out->n == MAX_DROP_GROUPS) break;
            g = &out->g[out->n++];
            *g = {id >> 2, 0xffffffffu, 0};
        }
        g->views = (g->views & ~(255u << (8 * k))) | (uint32_t)v << (8 * k);
    }
    return v;
}

// blocks of 256 threads; N may be the largest int32
unsigned blocks_of(int32_t N, int per) { return ((unsigned)N + 256u * per - 1) / (256u * per); }

}  // namespace

extern "C" int gs_opacity_dropout(gs_ctx *ctx, int32_t N, const float *opacity, int32_t opacity_is_logit, double p, uint64_t seed,
                                  int32_t n_views, const uint64_t *view_ids, float *out) {
    uint32_t limit;
    float scale;
    const int rc = check_dropout("gs_opacity_dropout", ctx, N, p, n_views, view_ids, &limit, &scale);
    if (rc || N == 0 || n_views == 0) return rc;
    GS_REQUIRE(opacity && out, "gs_opacity_dropout: NULL array argument");
    GS_HIP(hipSetDevice(ctx->device));
    const int per = per_thread(N);
    for (int done = 0; done < n_views;) {
        ViewGroups groups;
        const int n = take_views(&groups, view_ids, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_DROPOUT);
          hipLaunchKernelGGL(per == 4 ? opacity_dropout_kernel<4> : opacity_dropout_kernel<1>, dim3(blocks_of(N, per)), dim3(256), 0, ctx->stream, N, opacity,
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
    const int per = per_thread(N);
    int done = 0;
    do {      // no views: one launch that writes zeros (or adds nothing)
        ViewGroups groups;
        const int n = take_views(&groups, view_ids, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_DROPOUT);
          hipLaunchKernelGGL(per == 4 ? opacity_dropout_backward_kernel<4> : opacity_dropout_backward_kernel<1>, dim3(blocks_of(N, per)), dim3(256), 0, ctx->stream, N, opacity,
                             opacity_is_logit, limit, scale, seed, groups, dL_dout + (size_t)N * done,
                             (accumulate || done > 0) ? 1 : 0, dL_dopacity); }
        GS_HIP(hipGetLastError());
        done += n;
    } while (done < n_views);
    return GS_OK;
}
