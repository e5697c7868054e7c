"""4-bit spherical harmonics: the SH coefficients of a scene as 32-byte records, and the view-dependent colour computed
from them (gs_sh_* in include/gsplat.h; no counterpart in the reference, which keeps 48 floats per gaussian).

    packed = quantize_sh(sh)                        [N,3,16] -> PackedSH (192 -> 32 bytes per gaussian)
    packed.dequantize()                             the [N,3,16] coefficients the records stand for
    colors, clamped = sh_color(packed, means, cam_pos)                      forward_pass.py:168-215
    d_sh, d_means = sh_color_backward(packed, means, cam_pos, clamped, d_colors)   backward_pass.py:70-97

Arrays may be NumPy (results come back as NumPy, float64) or torch tensors (results stay on the device).  Calls run on
torch's current stream of the context's device and do not synchronise; a PackedSH made on one stream and used on another
needs the event or wait_stream that any tensor needs."""
import ctypes

import numpy as np
import torch

from .api import _ctx, _dev, _is_t, _np_out, _ptr
from ._lib import check

WORDS = 8      # 32-bit words per record


class PackedSH:
    """The packed SH coefficients of N gaussians: `words` [N,8], int32 tensor or 32-bit NumPy array (layout:
    include/gsplat.h, "Packed SH"), moved to the context's device when one is given.  Stands in the spherical_harmonics
    slot of a GaussianSet.  Calls copy records that are not on their device there every time: move them once (to())."""

    def __init__(self, words, ctx=None):
        if not _is_t(words):
            words = np.asarray(words)
            if words.dtype not in (np.dtype(np.int32), np.dtype(np.uint32)):
                raise ValueError(f"packed SH records are 32-bit words, got {words.dtype}")
            words = torch.from_numpy(np.array(words, order="C").view(np.int32))
        if words.dtype != torch.int32 or words.dim() != 2 or words.shape[1] != WORDS:
            raise ValueError(f"packed SH records must be int32 [N,{WORDS}], got {words.dtype} {list(words.shape)}")
        if ctx is not None:
            words = words.to(_ctx(ctx).device)
        self.words = _aligned(words.contiguous())

    @property
    def shape(self):
        """The shape of the coefficients the records stand for."""
        return (len(self), 3, 16)

    @property
    def nbytes(self):
        return len(self) * WORDS * 4

    def __len__(self):
        return self.words.shape[0]

    def __getitem__(self, index):
        """The records of a slice, mask or list of gaussians."""
        words = self.words[index]
        if words.dim() != 2:
            raise IndexError("index a PackedSH with a slice, mask or list")
        return PackedSH(words)

    def to(self, device):
        return self if self.words.device == torch.device(device) else PackedSH(self.words.to(device))

    def numpy(self):
        """The records on the host, uint32 [N,8]."""
        return self.words.cpu().numpy().view(np.uint32)

    def dequantize(self, ctx=None):
        """[N,3,16] float32 tensor of the coefficients the records stand for (gs_sh_dequantize)."""
        c = _ctx(ctx)
        c.sync_stream()
        words = _words(self, c)
        sh = torch.empty(self.shape, dtype=torch.float32, device=c.device)
        check(c.lib.gs_sh_dequantize(c.handle, len(self), _ptr(words), _ptr(sh)), "gs_sh_dequantize")
        return sh


def _words(packed, c):
    if not isinstance(packed, PackedSH):
        raise TypeError("packed SH coefficients (quantize_sh) expected, got " + type(packed).__name__)
    return packed.words.to(c.device)


def _aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone()


def quantize_sh(sh, ctx=None):
    """SH coefficients [N,3,16] -> PackedSH (gs_sh_quantize).  Per (gaussian, channel) the 15 coefficients behind the
    constant term share a power-of-two scale and are rounded to 4 bits (E2M1); the constant term to half precision."""
    if isinstance(sh, PackedSH):
        raise TypeError("the coefficients are packed already")
    c = _ctx(ctx)
    c.sync_stream()
    shape = tuple(sh.shape)
    if len(shape) != 3 or shape[1:] != (3, 16):
        raise ValueError(f"spherical_harmonics must be [N,3,16] (forward_pass.py:172-204), got {shape}")
    sh = _aligned(_dev(sh, torch.float32, c.device))
    words = torch.empty((shape[0], WORDS), dtype=torch.int32, device=c.device)
    check(c.lib.gs_sh_quantize(c.handle, shape[0], _ptr(sh), _ptr(words)), "gs_sh_quantize")
    return PackedSH(words)


def camera_position(camera_r, camera_t):
    """forward_pass.py:47: camera_r^T @ camera_t, the position view directions start from, summed in the order the
    kernels use."""
    r = np.asarray(camera_r.detach().cpu() if _is_t(camera_r) else camera_r, dtype=np.float64).reshape(3, 3)
    t = np.asarray(camera_t.detach().cpu() if _is_t(camera_t) else camera_t, dtype=np.float64).reshape(3)
    return np.array([(float(r[0, k]) * float(t[0]) + float(r[1, k]) * float(t[1])) + float(r[2, k]) * float(t[2])
                     for k in range(3)])


def _positions(cam_pos):
    """([V][3] doubles on the host, V); a copy, so that the array passed in may be read-only or strided."""
    p = np.array(cam_pos.detach().cpu() if _is_t(cam_pos) else cam_pos, dtype=np.float64, order="C")
    if p.size == 0:
        return (ctypes.c_double * 1)(), 0
    if p.ndim not in (1, 2) or p.shape[-1] != 3:
        raise ValueError(f"cam_pos must be [V,3] (or [3] for one camera), got {list(p.shape)}")
    return (ctypes.c_double * p.size).from_buffer(p), p.size // 3


def _means(means, packed, c):
    if tuple(means.shape) != (len(packed), 3):
        raise ValueError(f"means must be [{len(packed)},3] for {len(packed)} records, got {list(means.shape)}")
    return _dev(means, torch.float32, c.device)


def sh_color(packed, means, cam_pos, degree=3, ctx=None):
    """Colours [V,N,3] and clamp flags [V,N,3] (uint8) of every gaussian seen from the V camera positions cam_pos [V,3]
    (host; camera_position), as forward_pass evaluates them for the gaussians it does not cull (gs_sh_color)."""
    c = _ctx(ctx)
    c.sync_stream()
    words = _words(packed, c)
    m = _means(means, packed, c)
    pos, V = _positions(cam_pos)
    N = len(packed)
    colors = torch.empty((V, N, 3), dtype=torch.float32, device=c.device)
    clamped = torch.empty((V, N, 3), dtype=torch.uint8, device=c.device)
    check(c.lib.gs_sh_color(c.handle, N, _ptr(words), _ptr(m), int(degree), V, pos, _ptr(colors), _ptr(clamped)),
          "gs_sh_color")
    if not _is_t(means):
        return _np_out(colors, np.float64), _np_out(clamped, np.uint8)
    return colors, clamped


def sh_color_backward(packed, means, cam_pos, clamped, d_colors, degree=3, ctx=None, out=None, accumulate=False):
    """Gradients of sh_color, summed over the views: (d_sh [N,3,16], d_means [N,3]) (gs_sh_color_backward).  `clamped` and
    d_colors are [V,N,3].  d_sh is the gradient with respect to the coefficients the records stand for; training the
    coefficients they were made from takes it as theirs.  out=(d_sh, d_means) receives the result, added to what is there
    when accumulate."""
    c = _ctx(ctx)
    c.sync_stream()
    words = _words(packed, c)
    m = _means(means, packed, c)
    pos, V = _positions(cam_pos)
    N = len(packed)
    for name, t in (("clamped", clamped), ("d_colors", d_colors)):
        if tuple(t.shape) != (V, N, 3) and not (V == 1 and tuple(t.shape) == (N, 3)):
            raise ValueError(f"{name} must be [{V},{N},3], got {list(t.shape)}")
    cl = _dev(clamped, torch.uint8, c.device)
    dc = _dev(d_colors, torch.float32, c.device)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out=(d_sh, d_means)")
        out = (torch.empty((N, 3, 16), dtype=torch.float32, device=c.device),
               torch.empty((N, 3), dtype=torch.float32, device=c.device))
    for name, t, shape in (("d_sh", out[0], (N, 3, 16)), ("d_means", out[1], (N, 3))):
        if not _is_t(t) or t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or \
                t.device != c.device:
            raise ValueError(f"out: {name} must be a contiguous float32 {list(shape)} tensor on {c.device}")
    check(c.lib.gs_sh_color_backward(c.handle, N, _ptr(words), _ptr(m), int(degree), V, pos, _ptr(cl), _ptr(dc),
                                     int(bool(accumulate)), _ptr(out[0]), _ptr(out[1])), "gs_sh_color_backward")
    if not _is_t(means):
        return _np_out(out[0], np.float64), _np_out(out[1], np.float64)
    return out
