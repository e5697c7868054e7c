// Opacity dropout (include/gsplat.h, "Opacity dropout"): leaves gaussian i out of view s with probability p and divides
// the opacities that stay by 1 - p.  No counterpart in the reference.
//
// The mask is never stored: gaussian i stays in view s iff word (s & 3) of Philox4x32-10 (Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011), evaluated at the counter (i, 0, low and high half of s >> 2) under
// the 64-bit seed as key, is at least round(p 2^32).  It depends on (seed, i, s) alone: not on the device, the rank that
// renders the view, the launch, or the number of gaussians.
//
// Bound by HBM: 4 + 4 V bytes per gaussian forward, 8 + 4 V backward.  One thread per gaussian.
#include "common.h"
#include <math.h>

namespace {

// N may be the largest int32
unsigned blocks_of(int32_t N) { return ((unsigned)N + 255u) / 256u; }

constexpr int MAX_DROP_VIEWS = 64;       // view numbers that one launch takes by value
struct ViewIds {
    uint64_t id[MAX_DROP_VIEWS];
    int n;
};

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint32_t index, uint64_t block, uint64_t seed) {
    uint32_t c0 = index, c1 = 0, c2 = (uint32_t)block, c3 = (uint32_t)(block >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// The words of one gaussian: four consecutive view numbers share an evaluation of the generator.
struct Mask {
    uint32_t index, limit;
    uint64_t seed, block;
    bool have;
    Words words;
    __device__ __forceinline__ Mask(uint32_t i, uint32_t lim, uint64_t s) : index(i), limit(lim), seed(s), block(0), have(false) {}
    __device__ __forceinline__ bool keeps(uint64_t view) {
        if (!have || block != (view >> 2)) {     // the same decision in every lane: the view numbers are uniform
            block = view >> 2;
            have = true;
            words = philox(index, block, seed);
        }
        const uint32_t k = (uint32_t)view & 3u;
        return (k == 0 ? words.w[0] : k == 1 ? words.w[1] : k == 2 ? words.w[2] : words.w[3]) >= limit;
    }
};

__device__ __forceinline__ float activated(float x, int is_logit) { return is_logit ? 1.0f / (1.0f + expf(-x)) : x; }

__global__ __launch_bounds__(256) void opacity_dropout_kernel(int N, const float *__restrict__ opacity, int is_logit,
                                                              uint32_t limit, float scale, uint64_t seed, const ViewIds views,
                                                              float *__restrict__ out) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)N) return;
    const float o = activated(opacity[i], is_logit) * scale;
    Mask mask(i, limit, seed);
#pragma unroll 1
    for (int v = 0; v < views.n; v++) out[(size_t)v * N + i] = mask.keeps(views.id[v]) ? o : 0.0f;
}

__global__ __launch_bounds__(256) void opacity_dropout_backward_kernel(int N, const float *__restrict__ opacity, int is_logit,
                                                                       uint32_t limit, float scale, uint64_t seed,
                                                                       const ViewIds views, const float *__restrict__ d_out,
                                                                       int accumulate, float *__restrict__ d_opacity) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= (uint32_t)N) return;
    Mask mask(i, limit, seed);
    float g = 0.0f;
#pragma unroll 1
    for (int v = 0; v < views.n; v++) {
        const float d = d_out[(size_t)v * N + i];
        if (mask.keeps(views.id[v])) g += d;        // selected, not multiplied: a NaN of a dropped gaussian stays out
    }
    if (is_logit) {
        const float o = activated(opacity[i], 1);
        g *= o * (1.0f - o);
    }
    g *= scale;
    d_opacity[i] = accumulate ? d_opacity[i] + g : g;
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

int take_views(ViewIds *out, const uint64_t *ids, int first, int n_views) {
    out->n = n_views - first < MAX_DROP_VIEWS ? n_views - first : MAX_DROP_VIEWS;
    for (int v = 0; v < out->n; v++) out->id[v] = ids[first + v];
    return out->n;
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
        ViewIds ids;
        const int n = take_views(&ids, view_ids, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_DROPOUT);
          hipLaunchKernelGGL(opacity_dropout_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N, opacity,
                             opacity_is_logit, limit, scale, seed, ids, out + (size_t)N * done); }
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
        ViewIds ids;
        const int n = take_views(&ids, view_ids, done, n_views);
        { gs_prof_scope prof_(ctx, GS_K_DROPOUT);
          hipLaunchKernelGGL(opacity_dropout_backward_kernel, dim3(blocks_of(N)), dim3(256), 0, ctx->stream, N, opacity,
                             opacity_is_logit, limit, scale, seed, ids, dL_dout + (size_t)N * done,
                             (accumulate || done > 0) ? 1 : 0, dL_dopacity); }
        GS_HIP(hipGetLastError());
        done += n;
    } while (done < n_views);
    return GS_OK;
}
