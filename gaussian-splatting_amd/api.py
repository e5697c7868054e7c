"""Host-side mirror of the reference's hot-path interface, backed by libgsplat_hip.so.

Same names, positional order, defaults and return tuples as the reference:

    setup_gpu()                                                   setup_gpu.py:3,370
    forward_pass(ctx, queue, program, camera, camera_r, camera_t, gaussians,
                 result_size, tile_size, training)                forward_pass.py:25,134,136
    match_gaus_to_tiles(ctx, queue, program, tiles_touched, radiis, depths,
                 result_size, tile_size)                          rasterization.py:6
    gpu_rasterize(ctx, queue, program, centers, colors, opacities, conics, mapped_keys,
                 training, result_size, tile_size, background_color)   rasterization.py:27,105-107
    c_rasterize(...) / rasterize(...)                             rasterization.py:109,155
    backward_pass(ctx, queue, program, camera, camera_r, camera_t, gaussians, radii, covs_2d,
                 covs_3d, ws, ms, ts, dirs, clampeds, d_colors, d_2d_centers, d_conics)
                                                                  backward_pass.py:19,68
    GaussianSet(centers, shs, scales, rots, opacities, degrees)   gaussian.py:31-37

Arrays may be NumPy (copied to the device; results come back as NumPy with the reference's dtypes)
or torch CUDA tensors (zero-copy; results are torch tensors that stay on the device).  There is no
CPU fallback: every function raises if the HIP library or a GPU is missing.

Extensions the reference lacks (all keyword-only, defaults keep the reference behaviour):
  gpu_rasterize(..., dL_dimage=None, pixel_offset=0.5)   explicit loss gradient (defect B4)
  backward_pass(..., result_size=[979,546], tile_size=16) needed because forward intermediates
                                                          are recomputed instead of re-read
"""
import ctypes
import math

import numpy as np
import torch

from . import _lib
from ._lib import GsCamera, GsError, check

TILE = 16
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


# --------------------------------------------------------------------------- context
class DeviceContext:
    """Replaces the (ctx, queue, program) triple of setup_gpu() (setup_gpu.py:3-6,370): device id
    + HIP stream + workspace arena owned by the native library."""

    def __init__(self, device=0):
        if not torch.cuda.is_available():
            raise GsError("no HIP device visible: the MI355X path has no CPU fallback")
        self.lib = _lib.load()
        self.device_index = int(device)
        self.device = torch.device("cuda", self.device_index)
        torch.cuda.set_device(self.device)
        torch.cuda.init()
        self._stream_id = int(torch.cuda.current_stream(self.device).cuda_stream)
        h = ctypes.c_void_p()
        check(self.lib.gs_ctx_create(self.device_index, ctypes.c_void_p(self._stream_id), ctypes.byref(h)),
              "gs_ctx_create")
        self.handle = h
        self.options = {}
        self._clones = []       # weak references: options set later reach the contexts cloned from this one

    def sync_stream(self):
        """Make the native ctx launch on torch's current stream for this device."""
        # (the handle alone where torch hands it out: 0.1 us of every call instead of 1.8 us for a Stream object)
        sid = _raw_stream(self.device_index) if _raw_stream else int(torch.cuda.current_stream(self.device).cuda_stream)
        if sid != self._stream_id:
            check(self.lib.gs_ctx_set_stream(self.handle, ctypes.c_void_p(sid)), "gs_ctx_set_stream")
            self._stream_id = sid

    # streams and sibling contexts are handed out by the context, so that everything above it (SplatPipeline,
    # train_step) names no device runtime: a context of another kind can stand in this slot
    def clone(self):
        """A second context (own workspace arena) on the same device, with this context's options; options set
        on this context later are applied to its clones too (a lane must blend the way its pipeline was told to)."""
        import weakref
        c = DeviceContext(self.device_index)
        for name, value in self.options.items():
            c.set_option(name, value)
        self._clones.append(weakref.ref(c))
        return c

    def new_stream(self):
        """A new stream of the default priority (the library refuses any other: gs_ctx_set_stream)."""
        return torch.cuda.Stream(self.device)

    def current_stream(self):
        return torch.cuda.current_stream(self.device)

    def use_stream(self, stream):
        """Context manager: `stream` is the current stream inside the block."""
        return torch.cuda.stream(stream)

    def synchronize(self):
        torch.cuda.synchronize(self.device)

    def set_option(self, name, value):
        check(self.lib.gs_ctx_set_option(self.handle, name.encode(), int(value)), "gs_ctx_set_option")
        self.options = dict(self.options, **{name: int(value)})
        alive = []
        for ref in self._clones:
            c = ref()
            if c is not None and c.handle:
                c.set_option(name, value)
                alive.append(ref)
        self._clones = alive

    def info(self, name):
        """gs_ctx_info: "workspace_bytes" or "allocations" of this context's arena."""
        v = int(self.lib.gs_ctx_info(self.handle, name.encode()))
        if v < 0:
            raise GsError(f"gs_ctx_info: unknown name '{name}'")
        return v

    def reserve(self, n_max, d_max, result_size, tile_size=16, arrays=False, batch_views=0):
        """gs_ctx_reserve: size this context's workspace once for up to n_max gaussians and d_max list entries per
        view (batch_views > 0: also for gs_bin_prepare_* batches of that many views), so that no later call regrows
        it in the middle of a step."""
        check(self.lib.gs_ctx_reserve(self.handle, int(n_max), int(d_max), int(result_size[0]), int(result_size[1]),
                                      int(tile_size), int(bool(arrays)), int(batch_views)), "gs_ctx_reserve")

    def profile(self, enable=True):
        """Bracket every kernel launch with HIP events (see read_profile)."""
        check(self.lib.gs_ctx_profile(self.handle, int(bool(enable))), "gs_ctx_profile")

    def read_profile(self):
        """{kernel name: (total ms, launches)} since the last read; synchronises the stream."""
        n = self.lib.gs_profile_kernel_count()
        ms = (ctypes.c_double * n)()
        cnt = (ctypes.c_int64 * n)()
        check(self.lib.gs_ctx_profile_read(self.handle, ms, cnt), "gs_ctx_profile_read")
        return {self.lib.gs_profile_kernel_name(i).decode(): (ms[i], cnt[i]) for i in range(n)}

    def close(self):
        if getattr(self, "handle", None):
            self.lib.gs_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KernelLibrary:
    """Stands in the `program` slot (the reference's built cl.Program); names the entry points."""

    def __init__(self, lib):
        self.lib = lib
        self.kernels = ("gs_preprocess", "gs_bin_count", "gs_bin_fill", "gs_blend_forward",
                        "gs_blend_backward", "gs_backward_params", "rasterize_tile")


_default_ctx = {}


def setup_gpu(device=None):
    """setup_gpu.py:3-6,370 -> (ctx, queue, program).  `queue` is the torch stream the kernels
    are launched on; `program` names the native entry points."""
    if device is None:
        device = torch.cuda.current_device() if torch.cuda.is_available() else 0
    ctx = DeviceContext(device)
    return ctx, torch.cuda.current_stream(ctx.device), KernelLibrary(ctx.lib)


def _ctx(ctx):
    if isinstance(ctx, DeviceContext):
        return ctx
    if ctx is None and _default_ctx:
        known = _default_ctx.get(torch.cuda.current_device())
        if known is not None:
            return known
    if ctx is not None:
        if all(hasattr(ctx, a) for a in ("lib", "handle", "device", "sync_stream", "clone", "new_stream")):
            return ctx            # a context of another kind with DeviceContext's interface
        raise TypeError("ctx must be the DeviceContext returned by setup_gpu() (or None)")
    dev = torch.cuda.current_device() if torch.cuda.is_available() else 0
    if dev not in _default_ctx:
        _default_ctx[dev] = DeviceContext(dev)
    return _default_ctx[dev]


# --------------------------------------------------------------------------- helpers
_NP = {torch.float32: np.float32, torch.int32: np.int32, torch.uint8: np.uint8, torch.int64: np.int64}


def _is_t(x):
    return isinstance(x, torch.Tensor)


def _dev(x, dtype, device, shape=None):
    """NumPy array / torch tensor -> contiguous device tensor of `dtype`."""
    if _is_t(x):
        t = x.to(device=device, dtype=dtype)
    else:
        t = torch.from_numpy(np.ascontiguousarray(np.asarray(x), dtype=_NP[dtype])).to(device)
    if shape is not None:
        t = t.reshape(shape)
    return t.contiguous()


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _np_out(t, dtype):
    return t.detach().cpu().numpy().astype(dtype)


CAM_APPLY_VIEW, CAM_DIAG_SCALE = 1, 2     # gs_camera.flags (include/gsplat.h)


def camera_flags(apply_view=False, diag_scale=False):
    """0 is the reference's live path bit for bit; the two switches select the 'sane' variant of quirk Q1
    (centres projected from view space) and Q4 (diagonal scale matrix).  No reference counterpart."""
    return (CAM_APPLY_VIEW if apply_view else 0) | (CAM_DIAG_SCALE if diag_scale else 0)


def make_camera(camera, camera_r, camera_t, result_size, tile_size, degrees, flags=0):
    c = GsCamera()
    r = np.asarray(camera_r.detach().cpu() if _is_t(camera_r) else camera_r, dtype=np.float64).reshape(3, 3)
    t = np.asarray(camera_t.detach().cpu() if _is_t(camera_t) else camera_t, dtype=np.float64).reshape(3)
    for i in range(9):
        c.R[i] = float(r.flat[i])
    for i in range(3):
        c.t[i] = float(t[i])
    c.fx = float(camera.params[0])
    c.fy = float(camera.params[1])
    c.cam_width = int(camera.width)
    c.cam_height = int(camera.height)
    c.res_w, c.res_h = int(result_size[0]), int(result_size[1])
    c.tile_size = int(tile_size)
    c.sh_degree = int(degrees)
    c.flags = int(flags)
    return c


class GaussianSet:
    """Parameter container with the field names of gaussian.py:31-37 (the live constructor).  spherical_harmonics may be a
    PackedSH (quantize_sh) wherever a GaussianSet is taken."""

    def __init__(self, centers, shs, scales, rots, opacities, degrees=3):
        self.center = centers
        self.spherical_harmonics = shs    # [N,3,16] (load_model.py:40 layout)
        self.scaling = scales             # log-scales
        self.rotation = rots              # (w,x,y,z)
        self.opacity = opacities
        self.degrees = degrees

    def rasterize(self, camera, source_image, ctx, queue, program, file_output=None, result_size=[979, 546]):
        """gaussian.py:39-52, the render entry of load_model.py: forward_pass -> match_gaus_to_tiles
        -> gpu_rasterize(sigmoid(opacity)) at tile_size 32, saved as <file_output>.jpg when a name
        is given.  Returns the image [W,H,3]."""
        from .io import quat_to_rotmat
        camera_r = quat_to_rotmat(source_image.qvec)                       # gaussian.py:41
        camera_t = np.asarray(source_image.tvec, dtype=np.float64)
        centers, depths, colors, conics, tiles_touched, radii = forward_pass(
            ctx, queue, program, camera, camera_r, camera_t, self, result_size=result_size, training=False,
            tile_size=32)
        key_mapper = match_gaus_to_tiles(ctx, queue, program, tiles_touched, radii, depths, result_size=result_size,
                                         tile_size=32)
        op = self.opacity
        op = torch.sigmoid(op) if _is_t(op) else 1.0 / (1.0 + np.exp(-np.asarray(op, dtype=np.float64)))   # functions.py:42
        image = gpu_rasterize(ctx, queue, program, centers, colors, op, conics, key_mapper, result_size=result_size,
                              training=False, tile_size=32)
        if file_output:
            from PIL import Image as PILImage
            arr = image.detach().cpu().numpy() if _is_t(image) else image
            PILImage.fromarray(np.swapaxes(np.uint8(np.clip(arr, 0, 1) * 255), 0, 1)).save(
                "{output}.jpg".format(output=file_output))
        return image


def _gaussian_tensors(g, device):
    N = len(g.center)
    means = _dev(g.center, torch.float32, device, (N, 3))
    scales = _dev(g.scaling, torch.float32, device, (N, 3))
    quats = _dev(g.rotation, torch.float32, device, (N, 4))
    sh = g.spherical_harmonics
    shape = tuple(sh.shape)
    if shape != (N, 3, 16):
        raise ValueError(f"spherical_harmonics must be [N,3,16] (forward_pass.py:172-204), got {shape}")
    sh = sh.to(device) if _is_packed(sh) else _dev(sh, torch.float32, device, (N, 3, 16))
    return N, means, scales, quats, sh


def _is_packed(sh):
    """A PackedSH (32-byte records) in the place of the [N,3,16] coefficients."""
    return hasattr(sh, "words")


class bound_sh:
    """The `sh` argument of the parameter kernels on ctx `c` for gaussians first..first+N: a pointer into the coefficients,
    or, for a PackedSH, NULL while its records are bound to the ctx (gs_ctx_use_packed_sh) -- unbound on the way out, also
    when the call inside raises."""

    def __init__(self, c, N, sh, first=0):
        self.c, self.N, self.sh, self.first = c, N, sh, first

    def __enter__(self):
        if not _is_packed(self.sh):
            return ctypes.c_void_p(self.sh.data_ptr() + self.first * 192)
        if self.N:
            check(self.c.lib.gs_ctx_use_packed_sh(self.c.handle, self.N,
                                                  ctypes.c_void_p(self.sh.words.data_ptr() + self.first * 32)),
                  "gs_ctx_use_packed_sh")
        return ctypes.c_void_p(0)

    def __exit__(self, *exc):
        if _is_packed(self.sh):
            self.c.lib.gs_ctx_use_packed_sh(self.c.handle, 0, None)
        return False


# --------------------------------------------------------------------------- forward_pass
def forward_pass(ctx, queue, program, camera, camera_r, camera_t, gaussians,
                 result_size=[979, 546], tile_size=16, training=True, apply_view=False, diag_scale=False):
    """forward_pass.py:25-136.  Returns the 13-tuple (training) or 6-tuple of the reference:
    centers, depths, colors, conics, [clamped,] tiles_touched, radii[, Ws, Ms, Ts, cov2d, cov3d,
    dirs].  apply_view / diag_scale: see camera_flags (default: the reference's behaviour)."""
    c = _ctx(ctx)
    c.sync_stream()
    dev = c.device
    numpy_mode = not _is_t(gaussians.center)
    N, means, scales, quats, sh = _gaussian_tensors(gaussians, dev)
    cam = make_camera(camera, camera_r, camera_t, result_size, tile_size, gaussians.degrees,
                      camera_flags(apply_view, diag_scale))
    f32, i32 = torch.float32, torch.int32
    centers = torch.empty((N, 2), dtype=f32, device=dev)
    depths = torch.empty((N,), dtype=i32, device=dev)
    colors = torch.empty((N, 3), dtype=f32, device=dev)
    conics = torch.empty((N, 3), dtype=f32, device=dev)
    clamped = torch.empty((N, 3), dtype=torch.uint8, device=dev)
    tiles_touched = torch.empty((N, 2, 2), dtype=i32, device=dev)
    radii = torch.empty((N,), dtype=i32, device=dev)
    extras = [None] * 6
    if training:
        extras = [torch.empty((N,) + s, dtype=f32, device=dev)
                  for s in ((6,), (3, 3), (3,), (3,), (6,), (3,))]
    with bound_sh(c, N, sh) as sh_ptr:
        check(c.lib.gs_preprocess(c.handle, N, _ptr(means), _ptr(scales), _ptr(quats), sh_ptr,
                                  ctypes.byref(cam), _ptr(centers), _ptr(depths), _ptr(colors), _ptr(conics),
                                  _ptr(clamped), _ptr(tiles_touched), _ptr(radii), *[_ptr(e) for e in extras]),
              "gs_preprocess")
    if numpy_mode:
        f64 = np.float64
        out = [_np_out(centers, f64), _np_out(depths, np.int32), _np_out(colors, f64), _np_out(conics, f64),
               _np_out(clamped, f64), _np_out(tiles_touched, np.int32), _np_out(radii, f64)]
        out += [_np_out(e, f64) for e in extras] if training else []
    else:
        out = [centers, depths, colors, conics, clamped, tiles_touched, radii] + (extras if training else [])
    if training:
        return tuple(out)
    return out[0], out[1], out[2], out[3], out[5], out[6]


# --------------------------------------------------------------------------- binning
class TileBinning:
    """What match_gaus_to_tiles returns in place of the reference's dense u64
    key_mapper[tiles_x, tiles_y, N] (rasterization.py:8): sorted (tile<<32|depth) keys, gaussian
    ids and per-tile [start,end), all device-resident."""

    def __init__(self, keys, vals, ranges, D, result_size, tile_size):
        self.keys, self.vals, self.ranges, self.D = keys, vals, ranges, int(D)
        self.result_size = [int(result_size[0]), int(result_size[1])]
        self.tile_size = int(tile_size)
        self.tiles_x = math.ceil(self.result_size[0] / self.tile_size)
        self.tiles_y = math.ceil(self.result_size[1] / self.tile_size)

    def gaus_stack(self, i, j):
        """The reference's per-tile sorted u64 gaus_stack ((g<<32)+depth, rasterization.py:66-71)."""
        s, e = (int(v) for v in self.ranges[i * self.tiles_y + j].tolist())
        k = self.keys[s:e].cpu().numpy().view(np.uint64) & np.uint64(0xFFFFFFFF)
        v = self.vals[s:e].cpu().numpy().astype(np.uint64)
        return (v << np.uint64(32)) + k

    def sorted_gaussians(self, i, j):
        s, e = (int(v) for v in self.ranges[i * self.tiles_y + j].tolist())
        return self.vals[s:e].cpu().numpy()

    def __getitem__(self, ij):
        return self.gaus_stack(*ij)


def match_gaus_to_tiles(ctx, queue, program, tiles_touched, radiis, depths,
                        result_size=[979, 546], tile_size=16, *, want_keys=True, cull=None):
    """rasterization.py:6-25 (+ the per-tile filter/sort of :66-71).  `radiis` is accepted for
    signature compatibility; like the reference's kernel (quirk Q11) it does not affect the keys.
    want_keys=False skips materialising the 64-bit (tile<<32|depth) keys (the blend kernels only
    need the gaussian ids and the tile ranges).  cull=(centers, colors, opacities, conics,
    pixel_offset) (float32 device tensors, the ones the blend calls will get) drops the pairs that
    cannot change a pixel of their tile (gs_bin_*_culled): same images and gradients, about half
    the list."""
    c = _ctx(ctx)
    c.sync_stream()
    dev = c.device
    N = len(depths)
    rect = _dev(tiles_touched, torch.int32, dev, (N, 4))
    dep = _dev(depths, torch.int32, dev, (N,))
    W, H, ts = int(result_size[0]), int(result_size[1]), int(tile_size)
    D = ctypes.c_int64(0)
    extra = ()
    if cull is not None:
        cen, col, opa, con, off = cull
        held = (_dev(cen, torch.float32, dev, (N, 2)), _dev(col, torch.float32, dev, (N, 3)),
                _dev(opa, torch.float32, dev, (N,)), _dev(con, torch.float32, dev, (N, 3)))   # alive until the end
        extra = tuple(_ptr(t) for t in held)
        check(c.lib.gs_bin_count_culled(c.handle, N, _ptr(rect), _ptr(dep), *extra, W, H, ts, float(off),
                                        ctypes.byref(D)), "gs_bin_count_culled")
    else:
        check(c.lib.gs_bin_count(c.handle, N, _ptr(rect), _ptr(dep), W, H, ts, ctypes.byref(D)), "gs_bin_count")
    tiles = math.ceil(W / ts) * math.ceil(H / ts)
    keys = torch.empty((max(D.value, 1),), dtype=torch.int64, device=dev) if want_keys else None
    vals = torch.empty((max(D.value, 1),), dtype=torch.int32, device=dev)
    ranges = torch.empty((tiles, 2), dtype=torch.int32, device=dev)
    if cull is not None:
        check(c.lib.gs_bin_fill_culled(c.handle, N, _ptr(rect), _ptr(dep), *extra, W, H, ts, float(cull[4]), D.value,
                                       _ptr(keys), _ptr(vals), _ptr(ranges)), "gs_bin_fill_culled")
    else:
        check(c.lib.gs_bin_fill(c.handle, N, _ptr(rect), _ptr(dep), W, H, ts, D.value, _ptr(keys), _ptr(vals),
                                _ptr(ranges)), "gs_bin_fill")
    return TileBinning(keys[:D.value] if want_keys else None, vals[:D.value], ranges, D.value, [W, H], ts)


def bin_culled_begin(ctx, tiles_touched, depths, result_size, tile_size, cull):
    """First half of match_gaus_to_tiles(..., cull=...) (gs_bin_count_culled_begin): launches the count on
    the ctx's stream and returns a token for bin_culled_finish; the host does not wait."""
    c = _ctx(ctx)
    c.sync_stream()
    dev = c.device
    N = len(depths)
    rect = _dev(tiles_touched, torch.int32, dev, (N, 4))
    dep = _dev(depths, torch.int32, dev, (N,))
    W, H, ts = int(result_size[0]), int(result_size[1]), int(tile_size)
    cen, col, opa, con, off = cull
    if cen is None:      # the ctx has been given records (gs_ctx_use_records): the four arrays are not read
        held, extra = (), (_ptr(None),) * 4
    else:
        held = (_dev(cen, torch.float32, dev, (N, 2)), _dev(col, torch.float32, dev, (N, 3)),
                _dev(opa, torch.float32, dev, (N,)), _dev(con, torch.float32, dev, (N, 3)))
        extra = tuple(_ptr(t) for t in held)
    check(c.lib.gs_bin_count_culled_begin(c.handle, N, _ptr(rect), _ptr(dep), *extra, W, H, ts, float(off)),
          "gs_bin_count_culled_begin")
    return dict(c=c, N=N, rect=rect, dep=dep, held=held, extra=extra, W=W, H=H, ts=ts, off=float(off))


def bin_exact_begin(ctx, tiles_touched, depths, result_size, tile_size):
    """First half of match_gaus_to_tiles on the reference's own lists (gs_bin_count_begin): launches the count
    and returns a token for bin_culled_finish; the host does not wait."""
    c = _ctx(ctx)
    c.sync_stream()
    dev = c.device
    N = len(depths)
    rect = _dev(tiles_touched, torch.int32, dev, (N, 4))
    dep = _dev(depths, torch.int32, dev, (N,))
    W, H, ts = int(result_size[0]), int(result_size[1]), int(tile_size)
    check(c.lib.gs_bin_count_begin(c.handle, N, _ptr(rect), _ptr(dep), W, H, ts), "gs_bin_count_begin")
    return dict(c=c, N=N, rect=rect, dep=dep, held=(), extra=None, W=W, H=H, ts=ts, off=0.0)


def bin_culled_finish(tok, want_keys=False):
    """Second half: waits for the count only (gs_bin_count_end), then sorts (gs_bin_fill_culled, or gs_bin_fill
    for a token of bin_exact_begin)."""
    c = tok["c"]
    c.sync_stream()
    dev = c.device
    D = ctypes.c_int64(0)
    check(c.lib.gs_bin_count_end(c.handle, ctypes.byref(D)), "gs_bin_count_end")
    W, H, ts, N = tok["W"], tok["H"], tok["ts"], tok["N"]
    tiles = math.ceil(W / ts) * math.ceil(H / ts)
    keys = torch.empty((max(D.value, 1),), dtype=torch.int64, device=dev) if want_keys else None
    vals = torch.empty((max(D.value, 1),), dtype=torch.int32, device=dev)
    ranges = torch.empty((tiles, 2), dtype=torch.int32, device=dev)
    if tok["extra"] is None:
        check(c.lib.gs_bin_fill(c.handle, N, _ptr(tok["rect"]), _ptr(tok["dep"]), W, H, ts, D.value, _ptr(keys),
                                _ptr(vals), _ptr(ranges)), "gs_bin_fill")
    else:
        check(c.lib.gs_bin_fill_culled(c.handle, N, _ptr(tok["rect"]), _ptr(tok["dep"]), *tok["extra"], W, H, ts,
                                       tok["off"], D.value, _ptr(keys), _ptr(vals), _ptr(ranges)),
              "gs_bin_fill_culled")
    return TileBinning(keys[:D.value] if want_keys else None, vals[:D.value], ranges, D.value, [W, H], ts)


def _prepare_views(pres, records):
    views = (_lib.GsViewPrepare * max(len(pres), 1))()
    for k, p in enumerate(pres):
        views[k].tiles_touched = p["rect"].data_ptr()
        views[k].depths = p["depths"].data_ptr()
        views[k].records = p["rec"].data_ptr() if records else None
        views[k].perm = p["perm"].data_ptr()
        views[k].offsets = p["offsets"].data_ptr()
    return views


def bin_prepare_begin(ctx, pres, result_size, tile_size, pixel_offset, culled):
    """gs_bin_prepare_begin for the views in `pres` (records of preprocess_batch, at most 8): launches their counts on
    the ctx's stream; every record gets "perm" and "offsets" device arrays.  Returns a token for bin_prepare_end."""
    c = _ctx(ctx)
    c.sync_stream()
    N = len(pres[0]["depths"]) if pres else 0
    # the records only receive their perm / offsets once the call has succeeded: a refused call must not replace
    # (and thereby free) arrays that an earlier, still pending batch is about to write
    fresh = [dict(p, perm=torch.empty((max(N, 1),), dtype=torch.int32, device=c.device),
                  offsets=torch.empty((max(N, 1),), dtype=torch.int32, device=c.device)) for p in pres]
    views = _prepare_views(fresh, culled)
    W, H, ts = int(result_size[0]), int(result_size[1]), int(tile_size)
    check(c.lib.gs_bin_prepare_begin(c.handle, N, len(pres), views, W, H, ts, float(pixel_offset)), "gs_bin_prepare_begin")
    for p, f in zip(pres, fresh):
        p["perm"], p["offsets"] = f["perm"], f["offsets"]
        p.pop("D", None)
        p.pop("prepared", None)
    return dict(c=c, N=N, pres=pres, views=views, W=W, H=H, ts=ts, off=float(pixel_offset), culled=bool(culled))


def bin_prepare_end(tok):
    """gs_bin_prepare_end: one host wait for the whole batch, then the depth sorts and scans of its views are
    launched; every record of the batch gets "D" (its number of pairs)."""
    c = tok["c"]
    c.sync_stream()
    n = len(tok["pres"])
    D = (ctypes.c_int64 * max(n, 1))()
    check(c.lib.gs_bin_prepare_end(c.handle, tok["N"], n, tok["views"], tok["W"], tok["H"], tok["ts"], D),
          "gs_bin_prepare_end")
    for k, p in enumerate(tok["pres"]):
        p["D"] = int(D[k])
        p["prepared"] = tok
    return [int(D[k]) for k in range(n)]


def bin_fill_prepared(ctx, pre, want_keys=False):
    """gs_bin_fill_prepared: emit + tile sort + ranges of one prepared view on `ctx` (its stream must be ordered
    behind the bin_prepare_end that produced pre["perm"] / pre["offsets"])."""
    c = _ctx(ctx)
    c.sync_stream()
    tok = pre["prepared"]
    W, H, ts, N, D = tok["W"], tok["H"], tok["ts"], tok["N"], pre["D"]
    tiles = math.ceil(W / ts) * math.ceil(H / ts)
    dev = c.device
    keys = torch.empty((max(D, 1),), dtype=torch.int64, device=dev) if want_keys else None
    vals = torch.empty((max(D, 1),), dtype=torch.int32, device=dev)
    ranges = torch.empty((tiles, 2), dtype=torch.int32, device=dev)
    check(c.lib.gs_bin_fill_prepared(c.handle, N, _ptr(pre["rect"]), _ptr(pre["depths"]),
                                     _ptr(pre["rec"]) if tok["culled"] else _ptr(None), _ptr(pre["perm"]),
                                     _ptr(pre["offsets"]), D, W, H, ts, tok["off"], _ptr(keys), _ptr(vals), _ptr(ranges)),
          "gs_bin_fill_prepared")
    return TileBinning(keys[:D] if want_keys else None, vals[:D], ranges, D, [W, H], ts)


class DeviceTileBinning(TileBinning):
    """Lists whose length never left the device (gs_bin_culled_batch): `vals` has the capacity the lists were
    built with, `D_dev` = (pairs in the list, pairs found) on the device.  `.D` handed to the blend calls is the
    capacity (ranges bound every read); true_D() copies the real length to the host (one synchronisation)."""

    def __init__(self, vals, ranges, D_dev, capacity, result_size, tile_size):
        super().__init__(None, vals, ranges, int(capacity), result_size, tile_size)
        self.D_dev = D_dev

    def true_D(self):
        kept, found = (int(v) for v in self.D_dev.tolist())
        if found > kept:
            raise GsError(f"gs_bin_culled_batch: {found} pairs found, capacity {kept}: the list was truncated")
        return kept


def bin_bounds_batch(ctx, pres, result_size, tile_size):
    """Per view of `pres` (records of preprocess_batch): (rect pairs, largest depth key), with one host wait."""
    c = _ctx(ctx)
    c.sync_stream()
    views = (_lib.GsViewBin * max(len(pres), 1))()
    for k, p in enumerate(pres):
        views[k].tiles_touched = p["rect"].data_ptr()
        views[k].depths = p["depths"].data_ptr()
    out = (ctypes.c_int64 * (2 * max(len(pres), 1)))()
    N = len(pres[0]["depths"]) if pres else 0
    check(c.lib.gs_bin_bounds_batch(c.handle, N, len(pres), views, int(result_size[0]), int(result_size[1]),
                                    int(tile_size), out), "gs_bin_bounds_batch")
    return [(int(out[2 * k]), int(out[2 * k + 1])) for k in range(len(pres))]


def bin_culled_batch(ctx, pres, result_size, tile_size, pixel_offset, depth_bits=32, capacity=None):
    """The culled lists of every view in `pres` (each with "rect", "depths" and the 64-byte records "rec") in
    one batch of launches and no host wait; returns one DeviceTileBinning per view.  capacity: size of every
    view's vals (default: the largest rect-pair count of the batch, from bin_bounds_batch -- one host wait)."""
    c = _ctx(ctx)
    c.sync_stream()
    dev = c.device
    W, H, ts = int(result_size[0]), int(result_size[1]), int(tile_size)
    if capacity is None:
        bounds = bin_bounds_batch(c, pres, result_size, tile_size)
        capacity = max([b[0] for b in bounds] + [1])
        depth_bits = max(max(b[1] for b in bounds).bit_length(), 1)
    tiles = math.ceil(W / ts) * math.ceil(H / ts)
    N = len(pres[0]["depths"])
    n = len(pres)
    vals = torch.empty((n, max(int(capacity), 1)), dtype=torch.int32, device=dev)
    ranges = torch.empty((n, tiles, 2), dtype=torch.int32, device=dev)
    D_dev = torch.empty((n, 2), dtype=torch.int64, device=dev)
    views = (_lib.GsViewBin * n)()
    for k, p in enumerate(pres):
        views[k].tiles_touched = p["rect"].data_ptr()
        views[k].depths = p["depths"].data_ptr()
        views[k].records = p["rec"].data_ptr()
        views[k].vals = vals[k].data_ptr()
        views[k].ranges = ranges[k].data_ptr()
        views[k].D_dev = D_dev[k].data_ptr()
    check(c.lib.gs_bin_culled_batch(c.handle, N, n, views, W, H, ts, float(pixel_offset), int(depth_bits),
                                    int(capacity)), "gs_bin_culled_batch")
    return [DeviceTileBinning(vals[k], ranges[k], D_dev[k], capacity, [W, H], ts) for k in range(n)]


def _binning_from_lists(mapped_keys, result_size, tile_size, device):
    """Accept the dict format the reference's c_rasterize/rasterize expect
    (mapped_keys[i][j] = {depth: gaussian}, rasterization.py:132,167)."""
    W, H = int(result_size[0]), int(result_size[1])
    tx_n, ty_n = math.ceil(W / tile_size), math.ceil(H / tile_size)
    vals, ranges = [], np.zeros((tx_n * ty_n, 2), dtype=np.int32)
    pos = 0
    for i in range(tx_n):
        for j in range(ty_n):
            items = sorted(mapped_keys[i][j].items())
            if items:
                ranges[i * ty_n + j] = (pos, pos + len(items))
                vals.extend(int(g) for _, g in items)
                pos += len(items)
    v = torch.tensor(vals if vals else [0], dtype=torch.int32, device=device)
    return TileBinning(None, v[:pos], torch.from_numpy(ranges).to(device), pos, [W, H], tile_size)


def _as_binning(mapped_keys, result_size, tile_size, device):
    if isinstance(mapped_keys, TileBinning):
        if mapped_keys.result_size != [int(result_size[0]), int(result_size[1])] or \
                mapped_keys.tile_size != int(tile_size):
            raise ValueError("mapped_keys was built for a different result_size/tile_size")
        return mapped_keys
    return _binning_from_lists(mapped_keys, result_size, tile_size, device)


# --------------------------------------------------------------------------- blend
def _bg3(background_color):
    b = background_color.detach().cpu().numpy() if _is_t(background_color) else np.asarray(background_color)
    b = b.astype(np.float64).reshape(3)
    return (ctypes.c_float * 3)(float(b[0]), float(b[1]), float(b[2]))


def blend_forward(c, centers, colors, opacities, conics, binning, bg, pixel_offset):
    """Device tensors in, (image[W,H,3], n_contrib[W,H], t_final[W,H]) out."""
    dev = c.device
    W, H = binning.result_size
    N = opacities.shape[0]
    image = torch.empty((W, H, 3), dtype=torch.float32, device=dev)
    n_contrib = torch.empty((W, H), dtype=torch.int32, device=dev)
    t_final = torch.empty((W, H), dtype=torch.float32, device=dev)
    check(c.lib.gs_blend_forward(c.handle, N, _ptr(centers), _ptr(colors), _ptr(opacities), _ptr(conics),
                                 _ptr(binning.vals), _ptr(binning.ranges), binning.D, ctypes.byref(bg), W, H,
                                 binning.tile_size, float(pixel_offset), _ptr(image), _ptr(n_contrib),
                                 _ptr(t_final)), "gs_blend_forward")
    return image, n_contrib, t_final


def blend_forward_loss(c, centers, colors, opacities, conics, binning, bg, pixel_offset, target, kind, scale, loss_out):
    """gs_blend_forward_loss: K6 with the loss and dL/dimage in its epilogue.  loss_out (1-element device tensor) is
    added to.  Returns (image, n_contrib, t_final, dL_dimage)."""
    dev = c.device
    W, H = binning.result_size
    N = opacities.shape[0]
    target = target.contiguous()
    if tuple(target.shape) != (W, H, 3) or target.dtype != torch.float32:
        raise ValueError("target must be a float32 tensor [W,H,3]")
    image = torch.empty((W, H, 3), dtype=torch.float32, device=dev)
    dL = torch.empty((W, H, 3), dtype=torch.float32, device=dev)
    n_contrib = torch.empty((W, H), dtype=torch.int32, device=dev)
    t_final = torch.empty((W, H), dtype=torch.float32, device=dev)
    check(c.lib.gs_blend_forward_loss(c.handle, N, _ptr(centers), _ptr(colors), _ptr(opacities), _ptr(conics),
                                      _ptr(binning.vals), _ptr(binning.ranges), binning.D, ctypes.byref(bg), W, H,
                                      binning.tile_size, float(pixel_offset), _ptr(image), _ptr(n_contrib),
                                      _ptr(t_final), _ptr(target), {"l1": 0, "l2": 1}[kind], float(scale), _ptr(dL),
                                      _ptr(loss_out)), "gs_blend_forward_loss")
    return image, n_contrib, t_final, dL


def blend_backward(c, centers, colors, opacities, conics, binning, bg, pixel_offset, n_contrib, t_final,
                   dL_dimage):
    dev = c.device
    W, H = binning.result_size
    N = centers.shape[0]
    f32 = torch.float32
    d_centers = torch.empty((N, 2), dtype=f32, device=dev)
    d_conics = torch.empty((N, 3), dtype=f32, device=dev)
    d_opac = torch.empty((N,), dtype=f32, device=dev)
    d_colors = torch.empty((N, 3), dtype=f32, device=dev)
    check(c.lib.gs_blend_backward(c.handle, N, _ptr(centers), _ptr(colors), _ptr(opacities), _ptr(conics),
                                  _ptr(binning.vals), _ptr(binning.ranges), binning.D, ctypes.byref(bg), W, H,
                                  binning.tile_size, float(pixel_offset), _ptr(n_contrib), _ptr(t_final),
                                  _ptr(dL_dimage), _ptr(d_centers), _ptr(d_conics), _ptr(d_opac),
                                  _ptr(d_colors)), "gs_blend_backward")
    return d_centers, d_conics, d_opac, d_colors


def view_stats(ctx, radii, binning, n_contrib):
    """gs_view_stats: N_visible, D, D* (visited), longest tile list and the algorithmic bytes per stage of one
    rendered view, computed by the library from device arrays (any of them may be None).  Returns a dict."""
    c = _ctx(ctx)
    c.sync_stream()
    st = _lib.GsStats()
    W, H = binning.result_size
    N = int(radii.shape[0]) if radii is not None else 0
    check(c.lib.gs_view_stats(c.handle, N, _ptr(radii), binning.D, _ptr(binning.ranges), W, H, binning.tile_size,
                              _ptr(n_contrib), ctypes.byref(st)), "gs_view_stats")
    return {name: int(getattr(st, name)) for name, _ in st._fields_}


def _blend_inputs(c, centers, colors, opacities, conics):
    dev = c.device
    N = len(centers)
    return (N, _dev(centers, torch.float32, dev, (N, 2)), _dev(colors, torch.float32, dev, (N, 3)),
            _dev(opacities, torch.float32, dev, (N,)), _dev(conics, torch.float32, dev, (N, 3)))


def gpu_rasterize(ctx, queue, program, centers, colors, opacities, conics, mapped_keys,
                  training=True, result_size=[979, 546], tile_size=16, background_color=np.zeros(3),
                  *, dL_dimage=None, pixel_offset=0.5, return_state=False):
    """rasterization.py:27-107.  Returns image[W,H,3], or (image, d_colors, d_centers, d_conics,
    d_opacity) when training.  d_centers is scaled by (.5*W, .5*H) as the reference's kernel does
    (setup_gpu.py:157-158).  dL_dimage=None reproduces the reference, which uses the rendered
    image itself as dL/dpixel (setup_gpu.py:112-114,139-140); pass the real loss gradient
    [W,H,3] to train.  pixel_offset=+0.5 is rasterize.c:103-104."""
    c = _ctx(ctx)
    c.sync_stream()
    numpy_mode = not _is_t(centers)
    N, cen, col, opa, con = _blend_inputs(c, centers, colors, opacities, conics)
    binning = _as_binning(mapped_keys, result_size, tile_size, c.device)
    bg = _bg3(background_color)
    image, n_contrib, t_final = blend_forward(c, cen, col, opa, con, binning, bg, pixel_offset)
    conv = (lambda t: _np_out(t, np.float64)) if numpy_mode else (lambda t: t)
    if not training:
        return (conv(image), n_contrib, t_final) if return_state else conv(image)
    W, H = binning.result_size
    dl = image if dL_dimage is None else _dev(dL_dimage, torch.float32, c.device, (W, H, 3))
    d_centers, d_conics, d_opac, d_colors = blend_backward(c, cen, col, opa, con, binning, bg, pixel_offset,
                                                           n_contrib, t_final, dl)
    d_centers = d_centers * torch.tensor([.5 * W, .5 * H], dtype=torch.float32, device=c.device)
    out = (conv(image), conv(d_colors), conv(d_centers), conv(d_conics), conv(d_opac))
    return out + (n_contrib, t_final) if return_state else out


def rasterize(centers, colors, opacities, conics, mapped_keys, training=True, result_size=[979, 546],
              tile_size=16, background_color=np.zeros(3), *, ctx=None):
    """rasterization.py:155-215 (pixel centre c - (x + .5), i.e. pixel_offset=-0.5); returns
    image[W,H,3]."""
    return gpu_rasterize(ctx, None, None, centers, colors, opacities, conics, mapped_keys, training=False,
                         result_size=result_size, tile_size=tile_size, background_color=background_color,
                         pixel_offset=-0.5)


def c_rasterize(centers, colors, opacities, conics, mapped_keys, training=True, result_size=[979, 546],
                tile_size=16, background_color=np.zeros(3, dtype=np.float64)):
    """rasterization.py:109-153: per-tile calls of the native symbol rasterize_tile through ctypes,
    exactly as the reference binds ./shared.so (host float64 arrays, pixel offset +0.5)."""
    if int(tile_size) != TILE:
        raise ValueError("rasterize_tile is compiled for TILE_SIZE 16 (rasterize.c:5)")
    lib = _lib.load()
    W, H = int(result_size[0]), int(result_size[1])
    cen = np.ascontiguousarray(centers, dtype=np.float64)
    col = np.ascontiguousarray(colors, dtype=np.float64)
    opa = np.ascontiguousarray(np.asarray(opacities, dtype=np.float64).reshape(-1))
    con = np.ascontiguousarray(conics, dtype=np.float64)
    bg = np.ascontiguousarray(background_color, dtype=np.float64)
    image = np.empty([W, H, 3])
    last_contributors = np.empty([W, H], dtype=np.int32)
    chunk = np.zeros([TILE, TILE, 3])
    lc = np.zeros([TILE, TILE], dtype=np.int32)
    for i in range(math.ceil(W / TILE)):
        for j in range(math.ceil(H / TILE)):
            if isinstance(mapped_keys, TileBinning):
                stack = np.ascontiguousarray(mapped_keys.sorted_gaussians(i, j), dtype=np.int32)
            else:
                items = sorted(mapped_keys[i][j].items())
                stack = np.asarray([g for _, g in items], dtype=np.int32)
            sp = stack if len(stack) else np.zeros(1, dtype=np.int32)
            p = lambda a: ctypes.c_void_p(a.ctypes.data)
            check(lib.rasterize_tile(p(chunk), p(lc), p(cen), p(col), p(opa), p(con), p(sp), p(bg),
                                     len(stack), int(bool(training)), i, j, W, H), "rasterize_tile")
            lx, ly = min((i + 1) * TILE, W), min((j + 1) * TILE, H)
            cx, cy = lx - i * TILE, ly - j * TILE
            image[i * TILE:lx, j * TILE:ly] = chunk[:cx, :cy]
            last_contributors[i * TILE:lx, j * TILE:ly] = lc[:cx, :cy]
    c_rasterize.last_contributors = last_contributors
    return image


# --------------------------------------------------------------------------- backward_pass
def backward_params(c, means, scales, quats, sh, cam, radii, clamped, d_centers_px, d_conics, d_colors,
                    out=None, accumulate=False):
    """Device tensors in; returns (dL_dmeans, dL_dlog_scales, dL_dquats, dL_dsh[N,3,16])."""
    dev = c.device
    N = means.shape[0]
    f32 = torch.float32
    if out is None:
        out = (torch.empty((N, 3), dtype=f32, device=dev), torch.empty((N, 3), dtype=f32, device=dev),
               torch.empty((N, 4), dtype=f32, device=dev), torch.empty((N, 3, 16), dtype=f32, device=dev))
    with bound_sh(c, N, sh) as sh_ptr:
        check(c.lib.gs_backward_params(c.handle, N, _ptr(means), _ptr(scales), _ptr(quats), sh_ptr,
                                       ctypes.byref(cam), _ptr(radii), _ptr(clamped), _ptr(d_centers_px),
                                       _ptr(d_conics), _ptr(d_colors), int(bool(accumulate)), _ptr(out[0]),
                                       _ptr(out[1]), _ptr(out[2]), _ptr(out[3])), "gs_backward_params")
    return out


def backward_pass(ctx, queue, program, camera, camera_r, camera_t, gaussians,
                  radii, covs_2d, covs_3d, ws, ms, ts, dirs, clampeds,
                  d_colors, d_2d_centers, d_conics, *, result_size=[979, 546], tile_size=16,
                  apply_view=False, diag_scale=False):
    """backward_pass.py:19-68 -> (d_colors, d_centers, d_shs, d_scales, d_rots).

    d_colors: the incoming colour gradient masked by the clamp flags (the intent of
    setup_gpu.py:279-281); d_centers[N,3]: dL/d(world mean); d_shs[N,16,3] (the reference's layout,
    backward_pass.py:73); d_scales[N,3]: dL/d(log-scale parameter) (defect B13: the reference
    mixes activated and log scales); d_rots[N,4]: dL/d(un-normalised quaternion).
    d_2d_centers uses gpu_rasterize's convention (scaled by .5*W, .5*H).  covs_2d, covs_3d, ws,
    ms, ts and dirs are accepted for signature compatibility; the kernel recomputes them."""
    c = _ctx(ctx)
    c.sync_stream()
    dev = c.device
    numpy_mode = not _is_t(gaussians.center)
    N, means, scales, quats, sh = _gaussian_tensors(gaussians, dev)
    for name, arr, tail in (("covs_2d", covs_2d, 3), ("covs_3d", covs_3d, 6), ("ws", ws, 6), ("ts", ts, 3),
                            ("dirs", dirs, 3)):
        if arr is not None and (len(arr) != N or int(np.prod(arr.shape[1:])) != tail):
            raise ValueError(f"{name} must be [N,{tail}]")
    if ms is not None and (len(ms) != N or int(np.prod(ms.shape[1:])) != 9):
        raise ValueError("ms must be [N,3,3]")
    cam = make_camera(camera, camera_r, camera_t, result_size, tile_size, gaussians.degrees,
                      camera_flags(apply_view, diag_scale))
    rad = _dev(radii, torch.int32, dev, (N,))
    cl = _dev(clampeds, torch.uint8, dev, (N, 3))
    W, H = int(result_size[0]), int(result_size[1])
    d2 = _dev(d_2d_centers, torch.float32, dev, (N, 2)) / torch.tensor([.5 * W, .5 * H], dtype=torch.float32,
                                                                       device=dev)
    dcon = _dev(d_conics, torch.float32, dev, (N, 3))
    dcol = _dev(d_colors, torch.float32, dev, (N, 3))
    g_means, g_scales, g_quats, g_sh = backward_params(c, means, scales, quats, sh, cam, rad, cl,
                                                       d2.contiguous(), dcon, dcol)
    d_colors_out = dcol * (cl == 0).to(torch.float32)
    d_shs = g_sh.permute(0, 2, 1).contiguous()     # [N,16,3]
    outs = (d_colors_out, g_means, d_shs, g_scales, g_quats)
    if numpy_mode:
        return tuple(_np_out(o, np.float64) for o in outs)
    return outs
