/* gsplat.h -- C ABI of libgsplat_hip.so: the MI355X (gfx950) hot path of a 3D Gaussian Splatting
 * rasteriser, a drop-in for the Python hot-path functions of AubreyFeldker/gaussian-splatting.
 *
 * Conventions
 *   - every pointer is a DEVICE pointer owned by the caller unless the comment says "host";
 *   - every call is asynchronous on the ctx's HIP stream except where noted (gs_bin_count
 *     synchronises once to return D);
 *   - return 0 on success, <0 on error; gs_last_error() returns the message (thread-local);
 *   - one ctx per stream; calls on one ctx are serialised by the caller; ctxs are independent;
 *   - images are [W][H][3] x-major exactly as the reference (rasterize.c:93,130,
 *     rasterization.py:29,96,122);
 *   - the blend kernels take tile_size 16 (rasterize.c:5 TILE_SIZE), 32 (the render entry,
 *     gaussian.py:44-50) or any 16 << k: a tile is blended as 16x16 blocks sharing its list.
 *
 * Each entry point cites the reference interface it replaces (file:line under the reference).
 */
#ifndef GSPLAT_H
#define GSPLAT_H
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct gs_ctx gs_ctx;

/* Camera + frame description: the (camera, camera_r, camera_t, result_size, tile_size,
 * gaussians.degrees) arguments of forward_pass (forward_pass.py:25). Host struct. */
typedef struct gs_camera {
    double R[9];          /* camera_r, row-major, as passed to forward_pass                  */
    double t[3];          /* camera_t                                                         */
    double fx, fy;        /* camera.params[0], camera.params[1]                               */
    int32_t cam_width;    /* camera.width  (fov, forward_pass.py:43)                          */
    int32_t cam_height;   /* camera.height (fov, forward_pass.py:44)                          */
    int32_t res_w, res_h; /* result_size                                                      */
    int32_t tile_size;    /* 16                                                               */
    int32_t sh_degree;    /* gaussians.degrees, 0..3                                          */
    int32_t flags;        /* 0 = the reference's live forward path, bit for bit (strict).  "Sane"
                           * variants of two of its quirks, as constant branches of the same kernels
                           * (no reference counterpart; K8 differentiates whichever is selected):
                           * GS_CAM_APPLY_VIEW  the 2D centre is projected from VIEW-space coordinates
                           *   (the reference projects world coordinates: forward_pass.py:57 is
                           *   commented out, :59-61 use the world position);
                           * GS_CAM_DIAG_SCALE  the scale matrix is diag(s) * scale_mod (the reference
                           *   fills the off-diagonals with 1, forward_pass.py:75). */
} gs_camera;
#define GS_CAM_APPLY_VIEW 1
#define GS_CAM_DIAG_SCALE 2

/* Replaces setup_gpu() (setup_gpu.py:3-6,370): device context = device id + stream + workspace
 * arena. `stream` is a hipStream_t (NULL = default stream). */
int gs_ctx_create(int device, void *stream, gs_ctx **out);
/* The stream must have the DEFAULT priority (hipStreamGetPriority == 0): anything else is refused with an error.
 * (No reference counterpart: the reference has one OpenCL queue, setup_gpu.py:4-5.) */
int gs_ctx_set_stream(gs_ctx *ctx, void *stream);
int gs_ctx_destroy(gs_ctx *ctx);
/* Workspace accounting (no reference counterpart): name "workspace_bytes" = device bytes the ctx holds,
 * "allocations" = hipMallocs it has made since it was created (a grow-only arena: a training loop that
 * reserved ahead checks that a step adds none).  Returns -1 for an unknown name. */
int64_t gs_ctx_info(gs_ctx *ctx, const char *name);
/* Reserve ahead (no reference counterpart): sizes the ctx's workspace once for views of up to N_max gaussians and
 * D_max list entries at this frame, so that no later call on the ctx allocates -- without it a buffer that has
 * become too small is regrown in the middle of a step (stream synchronisation + hipFree + hipMalloc), which is
 * what a training loop with a growing gaussian count would otherwise pay after every
 * densification.  array_api != 0 also reserves the packed records and gradient rows that the array-based entry
 * points keep (64 bytes per gaussian each); callers that hand over records and rows (gs_ctx_use_records,
 * gs_blend_backward_rows) pass 0.  batch_views > 0 also sizes the ctx for gs_bin_prepare_begin / _end batches of that
 * many views (24 more bytes per gaussian and view).  The ordered K7 reduction's buffers (option
 * deterministic_backward) are not covered.  About 28 bytes per gaussian + 20 bytes per list entry. */
int gs_ctx_reserve(gs_ctx *ctx, int32_t N_max, int64_t D_max, int32_t res_w, int32_t res_h, int32_t tile_size,
                   int32_t array_api, int32_t batch_views);
/* Tuning knobs (no reference counterpart).  "pixels_per_thread": 1, 2 or 4 pixels of a tile
 * column per thread in the blend kernels (default 4 = one wavefront per 16x16 tile; also read
 * from the environment variable GSPLAT_PPT at ctx creation).
 * "deterministic_backward": 1 = gs_blend_backward* sum the per-(tile, gaussian) partial gradients in a
 * fixed order instead of with float atomics (the reference's kernel accumulates with compare-and-swap
 * atomics in arrival order, setup_gpu.py:9-21): the wave of a tile stores its partials next to the
 * tile's list entries, the entries are sorted by gaussian and each gaussian's run is added up in list
 * order.  Bitwise reproducible from run to run; about three times the time of the atomics form and
 * 48 bytes of workspace per list entry.  tile_size 16 or 32 only; one-wave-per-tile kernels only.
 * "tile_order": 1 (default; also GSPLAT_TILE_ORDER) = gs_blend_backward* hand their launch slots to the
 * 16x16 blocks heaviest-first (by the deepest last-contributor of the block, from n_contrib), for frames
 * of 2048..16384 blocks; results are unchanged (float atomics arrive in another order).
 * "tile_histogram": 1 (default) = gs_bin_fill* take the tile ranges from a per-tile histogram counted in the first
 * pass of the tile sort (frames of up to 32 768 tiles, keys == NULL) instead of writing the sorted tile ids and
 * reading them back; 0 = always the latter.  Same ranges bit for bit.
 * "sorted_count_from": gaussians from which gs_bin_count*_begin sorts by depth FIRST (all 32 key bits) and counts in
 * that order, so that the scan and emit kernels of gs_bin_fill* stream depth-ordered arrays (48 bytes of workspace
 * per gaussian) instead of gathering rect / depth / record per gaussian again -- once those arrays outgrow the caches a
 * gather costs a 128-byte line per item.  Default 2 097 152 (also GSPLAT_SORTED_COUNT_FROM); 0 = always.  Same lists
 * bit for bit.
 * "cull_shrink_rect": 1 (default) = the culled count / emit passes walk the tiles inside the axis-aligned bounding box
 * of the gaussian's own ellipse at its alpha threshold (grown by 0.1 % and a pixel) instead of the whole reference rect;
 * it only skips pairs the exact box test rejects, so the lists are the same with 0. */
int gs_ctx_set_option(gs_ctx *ctx, const char *name, int32_t value);
/* Per-kernel timing with HIP events on the ctx stream (no reference counterpart; the reference
 * only prints perf_counter deltas per stage, train.py:29-60).  While enabled every kernel launch
 * is bracketed by two events; gs_ctx_profile_read synchronises the stream, returns the summed
 * milliseconds and launch counts per kernel (arrays of gs_profile_kernel_count() entries, names
 * from gs_profile_kernel_name) and resets the counters. */
int gs_profile_kernel_count(void);
const char *gs_profile_kernel_name(int i);
int gs_ctx_profile(gs_ctx *ctx, int32_t enable);
int gs_ctx_profile_read(gs_ctx *ctx, double *ms_sum_host, int64_t *launches_host);
const char *gs_last_error(void);
int gs_version(void);

/* Replaces forward_pass (forward_pass.py:25-136) incl. py_compute_color (:168-215).
 * Inputs (fp32): means[N,3], log_scales[N,3], quats[N,4] (w,x,y,z), sh[N,3,16].
 * Outputs: centers[N,2] f32 (pixels), depths[N] i32, colors[N,3] f32, conics[N,3] f32,
 * clamped[N,3] u8, tiles_touched[N,4] i32 = [xmin,ymin,xmax,ymax] (the reference's [N,2,2]),
 * radii[N] i32.  The discontinuous chain (depth key, radius, tile rect) is evaluated in fp64 so
 * the integer outputs equal the reference's.  Training extras (forward_pass.py:89-94,134) are
 * written when non-NULL: Ws[N,6], Ms[N,9], Ts[N,3], cov2d[N,3], cov3d[N,6], dirs[N,3] (f32). */
int gs_preprocess(gs_ctx *ctx, int32_t N, const float *means, const float *log_scales,
                  const float *quats, const float *sh, const gs_camera *cam,
                  float *centers, int32_t *depths, float *colors, float *conics,
                  uint8_t *clamped, int32_t *tiles_touched, int32_t *radii,
                  float *Ws, float *Ms, float *Ts, float *cov2d, float *cov3d, float *dirs);

/* Multi-view form of gs_preprocess (no counterpart in the reference, which projects one view per
 * iteration, train.py:18-28): the parameters are read once and projected for every view of the
 * batch (launches of up to 8 views); per view the outputs equal gs_preprocess's bit for bit.
 * `views` is a HOST array; the output pointers are device pointers (no training extras). */
typedef struct gs_view_preprocess {
    const gs_camera *cam;
    float *centers; int32_t *depths; float *colors; float *conics; uint8_t *clamped;
    int32_t *tiles_touched; int32_t *radii;
} gs_view_preprocess;
int gs_preprocess_batch(gs_ctx *ctx, int32_t N, const float *means, const float *log_scales,
                        const float *quats, const float *sh, int32_t n_views,
                        const gs_view_preprocess *views);

/* Record-writing form of gs_preprocess_batch (no counterpart in the reference): instead of centers /
 * colors / conics each view receives records[N][16] floats, the 64-byte per-gaussian records the
 * blend and culled-binning kernels read (centre, opacity, alpha threshold, log2-scaled conic, colour; the last
 * 16 bytes repeat the tile rect as four int32, which the culled tile count of large scenes reads from there),
 * built from `opacities` (activated, [N]).  Records handed to gs_ctx_use_records must have been written by this
 * call.  gs_ctx_use_records(ctx, N, records) then makes the
 * culled-binning and blend calls on that ctx take their per-gaussian inputs from `records` and
 * ignore their centers / colors / opacities / conics arguments (which may be NULL), so no pack pass
 * runs per view; gs_ctx_use_records(ctx, 0, NULL) returns to the arrays.  The records must stay
 * unchanged while calls that use them are in flight. */
typedef struct gs_view_records {
    const gs_camera *cam;
    float *records; int32_t *depths; uint8_t *clamped; int32_t *tiles_touched; int32_t *radii;
} gs_view_records;
int gs_preprocess_batch_records(gs_ctx *ctx, int32_t N, const float *means, const float *log_scales,
                                const float *quats, const float *sh, const float *opacities,
                                int32_t n_views, const gs_view_records *views);
int gs_ctx_use_records(gs_ctx *ctx, int32_t N, const float *records);

/* Replaces match_gaus_to_tiles (rasterization.py:6-25) + kernel tile_match (setup_gpu.py:23-44)
 * + the per-tile filter and RadixSort (rasterization.py:57,66-71), in O(D) instead of
 * O(tiles*N).  Two phases so the caller owns the D-sized outputs:
 *   gs_bin_count: tiles-per-gaussian; returns D = their sum (host int64; one stream sync).
 *   gs_bin_fill : stable radix sort of the gaussians by u32(depth), duplication in that order
 *                 into (tile_id, gaussian) pairs, stable radix sort by tile_id;
 *                 vals[D] = gaussian ids, ranges[tile] = [start,end), tile_id = tx*tiles_y + ty;
 *                 keys[D] = (tile_id<<32)|u32(depth) of each entry, or NULL when not wanted.
 * Per tile the order is (depth asc, gaussian asc) = the reference's stable low-32-bit sort of
 * (g<<32)+depth; entries with u32(depth)==0 are dropped (rasterization.py:67).
 * gs_bin_fill must follow gs_bin_count on the same ctx with the same inputs. */
int gs_bin_count(gs_ctx *ctx, int32_t N, const int32_t *tiles_touched, const int32_t *depths,
                 int32_t res_w, int32_t res_h, int32_t tile_size, int64_t *D_host);
int gs_bin_fill(gs_ctx *ctx, int32_t N, const int32_t *tiles_touched, const int32_t *depths,
                int32_t res_w, int32_t res_h, int32_t tile_size, int64_t D,
                uint64_t *keys, int32_t *vals, int32_t *ranges);

/* Culled form of the two calls above (no counterpart in the reference): a (gaussian, tile) pair of
 * the reference's rect (forward_pass.py:114-120: the bounding square of 3 sigma of the LARGER axis)
 * is emitted only if the gaussian can reach alpha >= 1/255 (rasterize.c:114) somewhere in the tile's
 * pixel box -- the test the blend kernels apply when they stage a list.  The result is the list of
 * gs_bin_fill with those pairs removed, in the same order: gs_blend_forward / gs_blend_backward
 * give the same image and gradients from either list (n_contrib counts positions of the list it was
 * produced from, so forward and backward must use the same one), while D -- what is sorted, written
 * and staged -- is about halved.  centers / colors / opacities / conics are the arrays the blend
 * calls will be given (they are packed into the ctx's blend records here; a gs_blend_forward that
 * directly follows gs_bin_fill_culled on this ctx with the same arrays reuses them; any other call on
 * the ctx in between ends that reuse.  The cache is keyed on the four pointers and N only: the arrays'
 * CONTENTS must be unchanged between gs_bin_count_culled, gs_bin_fill_culled and that gs_blend_forward,
 * and between a gs_blend_forward and the gs_blend_backward* that consumes its n_contrib / t_final). */
int gs_bin_count_culled(gs_ctx *ctx, int32_t N, const int32_t *tiles_touched, const int32_t *depths,
                        const float *centers, const float *colors, const float *opacities,
                        const float *conics, int32_t res_w, int32_t res_h, int32_t tile_size,
                        float pixel_offset, int64_t *D_host);
int gs_bin_fill_culled(gs_ctx *ctx, int32_t N, const int32_t *tiles_touched, const int32_t *depths,
                       const float *centers, const float *colors, const float *opacities,
                       const float *conics, int32_t res_w, int32_t res_h, int32_t tile_size,
                       float pixel_offset, int64_t D, uint64_t *keys, int32_t *vals, int32_t *ranges);

/* gs_bin_count_culled in two halves, for callers that keep several views in flight on one stream (no
 * counterpart in the reference): _begin launches the count and records an event behind the copy of
 * D to pinned memory; gs_bin_count_end waits for THAT event only -- work enqueued on the stream after
 * _begin (another view's blend kernels on another ctx) keeps running -- and returns D.  One count
 * may be pending per ctx; gs_bin_fill_culled follows gs_bin_count_end as it follows
 * gs_bin_count_culled. */
int gs_bin_count_culled_begin(gs_ctx *ctx, int32_t N, const int32_t *tiles_touched, const int32_t *depths,
                              const float *centers, const float *colors, const float *opacities,
                              const float *conics, int32_t res_w, int32_t res_h, int32_t tile_size,
                              float pixel_offset);
/* the same first half for the reference's own lists (gs_bin_count = gs_bin_count_begin + gs_bin_count_end) */
int gs_bin_count_begin(gs_ctx *ctx, int32_t N, const int32_t *tiles_touched, const int32_t *depths,
                       int32_t res_w, int32_t res_h, int32_t tile_size);
/* The host wait is bounded: if the count has not completed after GSPLAT_WAIT_TIMEOUT_MS (environment, default
 * 30000) the call returns an error instead of blocking for ever. */
int gs_bin_count_end(gs_ctx *ctx, int64_t *D_host);

/* The culled lists of up to GS_BIN_MAX_VIEWS views per call, built by launches that each cover every view of the
 * batch, with no host wait (no counterpart in the reference, which builds one view's lists at a time on the host:
 * rasterization.py:6-25,57-71).  A training step is bound by the number of short dependent launches its views
 * need, and the per-view calls above need about 25 per view plus one host wait; this form needs about 20 per
 * BATCH and none.
 *   records        the view's 64-byte blend records (gs_preprocess_batch_records); the box test reads them
 *   vals[capacity] gaussian ids, per tile in (depth, gaussian) order -- the array gs_bin_fill_culled writes
 *   ranges[tiles,2]
 *   D_dev[2]       DEVICE memory: [0] = pairs in the list, [1] = pairs found ([1] > [0]: capacity was too small and
 *                  the list holds the first `capacity` pairs in depth order -- never an out-of-bounds access)
 * gs_bin_bounds_batch returns per view (bounds_host[2v], bounds_host[2v+1]) = (number of rect pairs of
 * rasterization.py:6-25 -- an upper bound of the culled count, to size vals with --, largest u32(depth) among
 * them), with ONE host wait for the whole batch.  gs_bin_culled_batch sorts the low depth_bits bits of the depth
 * keys (bits_of(max depth) from the bounds; 32 is always right) and waits for nothing.  The blend calls take
 * D = capacity for lists built this way (ranges bound every read of vals); the deterministic backward needs the
 * list's true length and is not supported on them. */
#define GS_BIN_MAX_VIEWS 8
typedef struct {
    const int32_t *tiles_touched;   /* [N,4]  */
    const int32_t *depths;          /* [N]    */
    const float *records;           /* [N,16] */
    int32_t *vals;                  /* [capacity] out */
    int32_t *ranges;                /* [tiles,2]  out */
    int64_t *D_dev;                 /* [2]        out, device */
} gs_view_bin;
int gs_bin_bounds_batch(gs_ctx *ctx, int32_t N, int32_t n_views, const gs_view_bin *views, int32_t res_w,
                        int32_t res_h, int32_t tile_size, int64_t *bounds_host);
int gs_bin_culled_batch(gs_ctx *ctx, int32_t N, int32_t n_views, const gs_view_bin *views, int32_t res_w,
                        int32_t res_h, int32_t tile_size, float pixel_offset, int32_t depth_bits, int64_t capacity);

/* The lists of a batch of views in two halves (no counterpart in the reference, which builds one view's lists at a
 * time on the host: rasterization.py:6-25,57-71).  What does not scale with the number of pairs -- the count, the
 * depth order of the gaussians, the scanned offsets -- is done for up to GS_BIN_MAX_VIEWS views by launches that
 * each cover every view (about 12 launches per BATCH and one host wait, instead of 12 short dependent launches
 * and one host wait per VIEW); what does -- emitting the pairs, the tile sort, the ranges -- stays per view, so
 * that the views of a training step can run it on their own streams next to other views' blend kernels.
 *   gs_bin_prepare_begin   launches the counts (records != NULL: the culled count of gs_bin_count_culled; NULL: the
 *                          rect count of gs_bin_count; the same for every view of a batch) and the copy of the
 *                          per-view totals to pinned memory; returns at once.  One batch may be pending per ctx.
 *   gs_bin_prepare_end     waits for that copy only (bounded, as gs_bin_count_end), then launches the depth sort and
 *                          the scan of every view; perm[N] (gaussians in (u32(depth), id) order) and offsets[N]
 *                          (exclusive prefix of pairs in that order) are caller-owned DEVICE arrays;
 *                          D_host[v] = pairs of view v.
 *   gs_bin_fill_prepared   K3 + K4b + K5 of ONE view from its perm / offsets / D, on any ctx of the device, stream-
 *                          ordered behind gs_bin_prepare_end by the caller: the result is bit for bit that of
 *                          gs_bin_fill (records == NULL) or gs_bin_fill_culled (records given). */
typedef struct {
    const int32_t *tiles_touched;   /* [N,4]  */
    const int32_t *depths;          /* [N]    */
    const float *records;           /* [N,16] or NULL */
    int32_t *perm;                  /* [N] out */
    uint32_t *offsets;              /* [N] out */
} gs_view_prepare;
int gs_bin_prepare_begin(gs_ctx *ctx, int32_t N, int32_t n_views, const gs_view_prepare *views, int32_t res_w,
                         int32_t res_h, int32_t tile_size, float pixel_offset);
int gs_bin_prepare_end(gs_ctx *ctx, int32_t N, int32_t n_views, const gs_view_prepare *views, int32_t res_w,
                       int32_t res_h, int32_t tile_size, int64_t *D_host);
int gs_bin_fill_prepared(gs_ctx *ctx, int32_t N, const int32_t *tiles_touched, const int32_t *depths,
                         const float *records, const int32_t *perm, const uint32_t *offsets, int64_t D,
                         int32_t res_w, int32_t res_h, int32_t tile_size, float pixel_offset, uint64_t *keys,
                         int32_t *vals, int32_t *ranges);

/* Replaces gpu_rasterize forward (rasterization.py:27-107 + kernel rasterize,
 * setup_gpu.py:46-100), c_rasterize/rasterize_tile (rasterization.py:109-153, rasterize.c:27-132)
 * and rasterize (rasterization.py:155-215): one launch for the whole frame.
 * pixel_offset: dist = c - x + pixel_offset; +0.5 = rasterize.c:103-104, -0.5 =
 * rasterization.py:187-191, 0 = setup_gpu.py:75-76.
 * Outputs: image[W,H,3] f32; n_contrib[W,H] i32: bits 0..30 = the reference's
 * last_contributors (rasterize.c:99-130), bit 31 set iff the pixel left the loop through the
 * transmittance break (rasterize.c:118-119); t_final[W,H] f32. */
int gs_blend_forward(gs_ctx *ctx, int32_t N, const float *centers, const float *colors,
                     const float *opacities, const float *conics, const int32_t *vals,
                     const int32_t *ranges, int64_t D, const float *background_host3,
                     int32_t res_w, int32_t res_h, int32_t tile_size, float pixel_offset,
                     float *image, int32_t *n_contrib, float *t_final);

/* gs_blend_forward with the training loss in the kernel's epilogue (no counterpart in the reference, whose loop
 * forms an L1 figure on uint8 copies on the host, train.py:45-49, and no dL/dimage at all): every pixel is compared
 * with target[W,H,3] while it is still in registers; dL_dimage[W,H,3] and the loss are those of gs_image_loss
 * (kind 0: mean |image - target|, dL = scale * sign(diff) / n; kind 1: mean diff^2, dL = scale * 2 diff / n;
 * n = W*H*3), except that loss_out[0] (device float) is ADDED to -- zero it first -- with one float atomic per
 * 16x16 block, so its last bits depend on the arrival order.  One pass over the image and two launches per view
 * less than gs_blend_forward + gs_image_loss. */
int gs_blend_forward_loss(gs_ctx *ctx, int32_t N, const float *centers, const float *colors,
                          const float *opacities, const float *conics, const int32_t *vals,
                          const int32_t *ranges, int64_t D, const float *background_host3,
                          int32_t res_w, int32_t res_h, int32_t tile_size, float pixel_offset,
                          float *image, int32_t *n_contrib, float *t_final, const float *target,
                          int32_t kind, float scale, float *dL_dimage, float *loss_out);

/* Replaces the backward half of kernel rasterize (setup_gpu.py:105-165, intent; defects B4-B8
 * not reproduced): reverse-order traversal from each pixel's last contributor.
 * dL_dimage[W,H,3] is an explicit input (B4).  Outputs are zeroed by the call, then accumulated:
 * dL_dcenters[N,2] (per pixel unit), dL_dconics[N,3], dL_dopacities[N], dL_dcolors[N,3]. */
int gs_blend_backward(gs_ctx *ctx, int32_t N, const float *centers, const float *colors,
                      const float *opacities, const float *conics, const int32_t *vals,
                      const int32_t *ranges, int64_t D, const float *background_host3,
                      int32_t res_w, int32_t res_h, int32_t tile_size, float pixel_offset,
                      const int32_t *n_contrib, const float *t_final, const float *dL_dimage,
                      float *dL_dcenters, float *dL_dconics, float *dL_dopacities,
                      float *dL_dcolors);

/* Replaces backward_pass (backward_pass.py:19-68), cov_2d_backpass + kernel cov_2d_grads
 * (backward_pass.py:99-133, setup_gpu.py:168-253), sh_backpass + kernel sh_grads
 * (backward_pass.py:70-97, setup_gpu.py:256-303) and the host d_scales/d_rots loop
 * (backward_pass.py:40-66); intent, defects B3/B9/B10/B13 not reproduced.  Forward
 * intermediates are recomputed from the parameters (fp64) instead of being re-read.
 * Inputs: parameters as gs_preprocess; radii[N], clamped[N,3] from gs_preprocess;
 * dL_dcenters[N,2] (pixel units), dL_dconics[N,3], dL_dcolors[N,3] from gs_blend_backward.
 * Outputs (written, or += when accumulate != 0): dL_dmeans[N,3], dL_dlog_scales[N,3],
 * dL_dquats[N,4] (w.r.t. the un-normalised quaternion), dL_dsh[N,3,16]. */
int gs_backward_params(gs_ctx *ctx, int32_t N, const float *means, const float *log_scales,
                       const float *quats, const float *sh, const gs_camera *cam,
                       const int32_t *radii, const uint8_t *clamped, const float *dL_dcenters,
                       const float *dL_dconics, const float *dL_dcolors, int32_t accumulate,
                       float *dL_dmeans, float *dL_dlog_scales, float *dL_dquats, float *dL_dsh);

/* gs_blend_backward without any allocation.  NO counterpart in the reference: it exists for callers that
 * cannot call hipMalloc -- code under HIP graph capture, tight serving loops, harnesses that forbid it.
 * Same arguments, same results (to float-atomics rounding) as gs_blend_backward, but the two buffers that
 * call keeps in the ctx's grow-only arena (the packed 64-byte blend records and the 64-byte gradient rows)
 * live in one static device array of the library: 2 x 64 bytes x GS_NOALLOC_MAX_N = 8 MiB, held by every GPU
 * the library runs on until the process ends.  N above GS_NOALLOC_MAX_N is rejected (GS_ERR_ARG, "exceeds
 * the static scratch").  The call issues only kernel launches and one hipMemsetAsync on the ctx's stream:
 * no hipMalloc / hipFree / event creation, no host synchronisation.  Every call on a GPU shares that GPU's
 * array, whatever its ctx or stream: calls that overlap on one GPU race -- serialise them (one stream, or
 * events).  The per-gaussian arrays must be given (records set with gs_ctx_use_records are not used), and
 * the kernel is always the one-wave-per-tile kernel (the pixels_per_thread option is ignored). */
#define GS_NOALLOC_MAX_N 65536
int gs_blend_backward_noalloc(gs_ctx *ctx, int32_t N, const float *centers, const float *colors,
                              const float *opacities, const float *conics, const int32_t *vals,
                              const int32_t *ranges, int64_t D, const float *background_host3,
                              int32_t res_w, int32_t res_h, int32_t tile_size, float pixel_offset,
                              const int32_t *n_contrib, const float *t_final, const float *dL_dimage,
                              float *dL_dcenters, float *dL_dconics, float *dL_dopacities,
                              float *dL_dcolors);

/* Multi-view forms of the two backward entry points.  No counterpart in the reference, which
 * trains one view per iteration (train.py:18-43); they serve SURVEY section 8(e): a rank renders
 * its shard of the view batch, then converts all of its views' blend gradients to parameter
 * gradients in ONE pass over the gaussians before the all-reduce.
 *
 * gs_blend_backward_rows: gs_blend_backward, but the result stays in the kernel's native layout,
 * one 64-byte row per gaussian: grad_rows[N][16] = {d centre x,y (pixel units), d conic A,B,C,
 * d opacity, d colour r,g,b, 7 unused}.  The call zeroes the rows, then accumulates.
 *
 * gs_backward_params_batch: gs_backward_params over n_views views at once (launches of up to 8
 * views).  Parameters are read once, dL/dSigma is summed over the views before the
 * Sigma -> (log-scale, quaternion) chain, gradients are written once (or += when accumulate).
 * dL_dopacity[N] (may be NULL) receives the summed opacity gradient; when `opacity` is non-NULL
 * and opacity_is_logit != 0 it is chained through opacity = sigmoid(parameter)
 * (gaussian.py:50).  `views` is a HOST array; every view must share result_size. */
typedef struct gs_view_backward {
    const gs_camera *cam;       /* host */
    const int32_t *radii;       /* device [N]    from gs_preprocess of that view */
    const uint8_t *clamped;     /* device [N,3]  from gs_preprocess of that view */
    const float *grad_rows;     /* device [N,16] from gs_blend_backward_rows of that view */
} gs_view_backward;
int gs_blend_backward_rows(gs_ctx *ctx, int32_t N, const float *centers, const float *colors,
                           const float *opacities, const float *conics, const int32_t *vals,
                           const int32_t *ranges, int64_t D, const float *background_host3,
                           int32_t res_w, int32_t res_h, int32_t tile_size, float pixel_offset,
                           const int32_t *n_contrib, const float *t_final, const float *dL_dimage,
                           float *grad_rows);
int gs_backward_params_batch(gs_ctx *ctx, int32_t N, const float *means, const float *log_scales,
                             const float *quats, const float *sh, const float *opacity,
                             int32_t opacity_is_logit, int32_t n_views, const gs_view_backward *views,
                             int32_t accumulate, float *dL_dmeans, float *dL_dlog_scales,
                             float *dL_dquats, float *dL_dopacity, float *dL_dsh);

/* Workload statistics of one rendered view (no counterpart in the reference, which only prints per-stage
 * wall times, train.py:29-60, gaussian.py:45-51).  Computed by small reduction kernels from the arrays the
 * hot path produced: radii[N] (gs_preprocess), ranges[tiles,2] and D (gs_bin_fill*), n_contrib[W,H]
 * (gs_blend_forward); any of the three may be NULL (its fields are then -1).  Synchronises the ctx's stream.
 * `visited` is D* of SURVEY section 8(d): per 16x16 pixel block the deepest last-contributor, summed -- the
 * list entries the blend kernels walk before early-out; the bytes_* fields are the per-launch ALGORITHMIC
 * bytes of section 8(d) (fp32, degree-3 SH, split depth / tile sort) for these sizes. */
typedef struct gs_stats {
    int64_t n_gaussians, n_visible;          /* radii > 0 */
    int64_t duplicates;                      /* D: (gaussian, tile) pairs in the lists */
    int64_t visited;                         /* D* */
    int64_t max_tile_list, nonempty_tiles, tiles;
    int64_t pixels, pixels_broke;            /* pixels that left the loop through T < 1e-4 (rasterize.c:118) */
    int64_t bytes_preprocess, bytes_depth_sort, bytes_duplicate, bytes_tile_sort, bytes_ranges;
    int64_t bytes_blend_forward, bytes_blend_backward, bytes_param_backward;
} gs_stats;
int gs_view_stats(gs_ctx *ctx, int32_t N, const int32_t *radii, int64_t D, const int32_t *ranges,
                  int32_t res_w, int32_t res_h, int32_t tile_size, const int32_t *n_contrib,
                  gs_stats *out_host);

/* Training-loop side.
 * gs_image_loss replaces train.py:45-49 (an L1 "loss" on uint8 copies that wraps around, defect
 * B12, and no dL/dimage at all, defect B4): over n = W*H*3 floats, kind 0: loss = mean|image -
 * target|, dL_dimage = scale*sign(diff)/n; kind 1: loss = mean diff^2, dL_dimage = scale*2*diff/n.
 * loss_out[0] (device float) is written, or added to when accumulate != 0.
 * gs_adam_step replaces the parameter update of train.py:51-56.  mode 0: Adam with bias
 * correction for `step` (1-based), one learning rate per group in the order means, log_scales,
 * quats, opacity, sh (main.py:11-17: .0008, .025, .005, .25, .0125); grad_flat / m_flat / v_flat are
 * the flat buffers laid out in that order, each group (3N, 3N, 4N, N, 48N floats) starting at the
 * next multiple of 4 floats (N*59 floats in all when N % 4 == 0).  mode 1: the reference's intent,
 * param -= lr * grad * sgd_scale (sgd_scale = the L1 loss, train.py:52-56).  Non-finite gradients
 * count as 0 (np.nan_to_num, train.py:52-55). */
int gs_image_loss(gs_ctx *ctx, int64_t n, const float *image, const float *target, int32_t kind,
                  float scale, int32_t accumulate, float *dL_dimage, float *loss_out);
int gs_adam_step(gs_ctx *ctx, int32_t N, float *means, float *log_scales, float *quats, float *opacity,
                 float *sh, const float *grad_flat, float *m_flat, float *v_flat, const float *lr_host5,
                 float beta1, float beta2, float eps, int32_t step, int32_t mode, float sgd_scale);

/* Packed SH: a gaussian's 48 SH coefficients [3][16] as one 32-byte record, 192 -> 32 bytes (no counterpart in the
 * reference, which keeps them in full precision).  words[N][8] uint32, as four 64-bit little-endian numbers q0..q3:
 *   q0       half-precision bits of the constant terms (k = 0) of r, g, b at bits 0, 16, 32; scale bytes of r and g at
 *            bits 48 and 56
 *   q1..q3   channel r, g, b: the E2M1 code (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6) of
 *            coefficient k = 1..15 at bit 4 (k - 1); bits 60..63: the low half (r) and the high half (g) of the scale
 *            byte of b, 0 (b)
 * Coefficient k of a channel with scale byte s is its code's value times 2^(s - 127).  gs_sh_quantize takes for s the
 * exponent of the channel's largest magnitude (k >= 1) rounded to one mantissa bit, minus 2, within 0..252, and rounds to
 * the nearest code, ties to the even one, 6 scales at most; a channel with a NaN or an infinity among k >= 1 becomes NaN
 * (s = 255).  The constant terms are rounded to half precision (finite values saturate at 65504).
 * words must be 16-byte aligned, sh too.  gs_sh_dequantize writes the 48 floats a record stands for. */
int gs_sh_quantize(gs_ctx *ctx, int32_t N, const float *sh, uint32_t *words);
int gs_sh_dequantize(gs_ctx *ctx, int32_t N, const uint32_t *words, float *sh);

/* View-dependent colour from packed SH, for n_views cameras at once: the colour part of forward_pass (py_compute_color,
 * forward_pass.py:168-215) of EVERY gaussian (no culling).  cam_pos_host[n_views][3]: HOST doubles, camera_r^T @ camera_t
 * as forward_pass.py:47 forms them.  colors[n_views][N][3] = max(0, .5 + sum_k Y_k(d) c_k) with d the unit vector from
 * the camera position to the mean, clamped[n_views][N][3] = 1 where the sum was negative; coefficients above `degree` do
 * not take part; a gaussian at the camera's own position gets NaN (degree > 0).  Evaluated in fp64: where gs_preprocess
 * does not cull the gaussian, colour and flag are its results on the dequantised coefficients, up to the order of the fp64
 * sums. */
int gs_sh_color(gs_ctx *ctx, int32_t N, const uint32_t *words, const float *means, int32_t degree, int32_t n_views,
                const double *cam_pos_host, float *colors, uint8_t *clamped);
/* Its gradients, summed over the views (sh_backpass + kernel sh_grads, backward_pass.py:70-97, setup_gpu.py:256-303;
 * intent): dL_dsh[N][3][16] w.r.t. the coefficients the records stand for (a caller that trains the coefficients the
 * records were made from takes it for theirs: straight through the rounding), dL_dmeans[N][3] through the direction.
 * Clamped channels contribute nothing.  Written, or added to when accumulate != 0. */
int gs_sh_color_backward(gs_ctx *ctx, int32_t N, const uint32_t *words, const float *means, int32_t degree,
                         int32_t n_views, const double *cam_pos_host, const uint8_t *clamped, const float *dL_dcolors,
                         int32_t accumulate, float *dL_dsh, float *dL_dmeans);

/* Makes the parameter kernels read the SH coefficients from packed records: while words != NULL, gs_preprocess*,
 * gs_preprocess_batch*, gs_backward_params* and gs_backward_params_batch* on this ctx take the coefficients of their N
 * gaussians from words[N][8] and ignore their `sh` argument (which may be NULL); their outputs are those of the same call
 * on the dequantised coefficients, bit for bit (gradients to fp32 rounding).  N must be the N of those calls.
 * gs_ctx_use_packed_sh(ctx, 0, NULL) returns to the argument.  The records must stay unchanged while calls that use them
 * are in flight. */
int gs_ctx_use_packed_sh(gs_ctx *ctx, int32_t N, const uint32_t *words);

/* gs_preprocess_batch_records with opacities of its own per view: view v's records are built from
 * opacities[v * opacity_stride + i] (opacity_stride >= N, the layout gs_opacity_dropout writes; 0: one array for every
 * view). */
int gs_preprocess_batch_records_views(gs_ctx *ctx, int32_t N, const float *means, const float *log_scales,
                                      const float *quats, const float *sh, const float *opacities,
                                      int64_t opacity_stride, int32_t n_views, const gs_view_records *views);

/* gs_backward_params_batch for views that were blended with dropped-out opacities: the opacity gradient of view v is
 * multiplied by opacity_scale_host[v] (HOST, 1 / (1 - p); NULL: 1 for every view).  That is the whole backward pass of the
 * dropout: a gaussian that was left out has opacity 0, reaches alpha 1/255 nowhere, and its gradient row is zero.  (A NaN
 * logit has a NaN derivative here, as without dropout: 0 times it is NaN.) */
int gs_backward_params_batch_scaled(gs_ctx *ctx, int32_t N, const float *means, const float *log_scales,
                                    const float *quats, const float *sh, const float *opacity,
                                    int32_t opacity_is_logit, int32_t n_views, const gs_view_backward *views,
                                    const float *opacity_scale_host, int32_t accumulate, float *dL_dmeans,
                                    float *dL_dlog_scales, float *dL_dquats, float *dL_dopacity, float *dL_dsh);

/* Opacity dropout (no counterpart in the reference): per view, gaussian i is left out with probability p and the opacities
 * that stay are divided by 1 - p.  out[n_views][N] = keep ? o / (1 - p) : 0 with o = opacity[i], or its sigmoid when
 * opacity_is_logit != 0.  The mask is not stored: view s (view_ids_host, HOST, any 64-bit numbers) keeps gaussian i iff
 * word (s & 3) of Philox4x32-10 at the counter (i, 0, low and high 32 bits of s >> 2) under the key `seed` is at least
 * round(p 2^32), 0 <= p < 1.  gs_opacity_dropout_backward evaluates it again:
 * dL_dopacity[i] = do/dopacity / (1 - p) * sum over the views that keep i of dL_dout[view][i], written, or added to when
 * accumulate != 0; gradients of left-out gaussians are not read into the sum, NaN included, and a gaussian that every view
 * leaves out gets 0, whatever its opacity is. */
int gs_opacity_dropout(gs_ctx *ctx, int32_t N, const float *opacity, int32_t opacity_is_logit, double p, uint64_t seed,
                       int32_t n_views, const uint64_t *view_ids_host, float *out);
int gs_opacity_dropout_backward(gs_ctx *ctx, int32_t N, const float *opacity, int32_t opacity_is_logit, double p,
                                uint64_t seed, int32_t n_views, const uint64_t *view_ids_host, const float *dL_dout,
                                int32_t accumulate, float *dL_dopacity);

/* The reference's only native symbol (rasterize.c:27-28), kept as a compatibility shim with
 * HOST pointers and `double` conics (defect B7): blends one 16x16 tile on the device through the
 * same kernel as gs_blend_forward (pixel offset +0.5) and copies the chunk back.  Synchronous.
 * Returns 0 on success (the original always returns 0, rasterize.c:79), <0 on error. */
int rasterize_tile(double image_chunk[16][16][3], int last_contributors[16][16],
                   double centers[][2], double colors[][3], double opacities[],
                   double conics[][3], int gaus_stack[], double background_color[3],
                   int stack_size, int training, int tile_x, int tile_y, int result_x,
                   int result_y);

#ifdef __cplusplus
}
#endif
#endif /* GSPLAT_H */
