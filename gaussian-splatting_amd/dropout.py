"""Opacity dropout (gs_opacity_dropout* in include/gsplat.h; no counterpart in the reference): while a scene is trained from
few views, each view leaves out every gaussian with probability p and divides the opacities that stay by 1 - p, so that no
gaussian can rely on the ones in front of it.  The mask is a function of (seed, gaussian, view number) and is never stored:
the backward pass evaluates it again, and every rank and device gets the same one.

    op = dropout_opacity(opacity, p, seed, views)             [N] -> [V,N], in front of gpu_rasterize
    d_opacity = dropout_opacity_backward(d_op, opacity, p, seed, views)
    train_step(pipe, views, targets, grads, dropout=OpacityDropout(p, seed, first_view=step * len(views)))

Arrays may be NumPy (results come back as NumPy, float64) or torch tensors (results stay on the device).  Calls run on
torch's current stream of the context's device and do not synchronise.  Seed and view numbers are read when the call is
made: a captured graph replays the masks it was captured with."""
import ctypes

import numpy as np
import torch

from .api import _ctx, _dev, _is_t, _np_out, _ptr
from ._lib import check


def _view_ids(views):
    ids = [int(v) for v in views]
    if ids and (min(ids) < 0 or max(ids) >= 2 ** 64):
        raise ValueError("view numbers must be in 0 .. 2^64 - 1")
    return (ctypes.c_uint64 * max(len(ids), 1))(*ids), len(ids)


def _seed(seed):
    seed = int(seed)
    if not 0 <= seed < 2 ** 64:
        raise ValueError(f"seed {seed} must be in 0 .. 2^64 - 1")
    return seed


def _opacity(opacity, c):
    shape = tuple(opacity.shape)
    if len(shape) not in (1, 2) or (len(shape) == 2 and shape[1] != 1):
        raise ValueError(f"opacity must be [N] or [N,1], got {list(shape)}")
    return shape[0], _dev(opacity, torch.float32, c.device, (shape[0],))


class OpacityDropout:
    """Dropout of one training step: probability p, seed, and the number of the step's first view; the step's view k (its
    position in the whole batch, whichever rank renders it) is number first_view + k.  A training gives every step numbers
    of its own: step * views_per_step."""

    def __init__(self, p, seed=0, first_view=0):
        if not 0.0 <= float(p) < 1.0:
            raise ValueError(f"dropout probability {p} not in [0, 1)")
        self.p, self.seed, self.first_view = float(p), _seed(seed), int(first_view)

    @property
    def scale(self):
        """What the opacities that stay are multiplied by, and the gradient of a view's opacities with them."""
        return 1.0 / (1.0 - self.p)

    def opacities(self, opacity, numbers, is_logit, ctx=None):
        """[V,N] opacities of the step's views `numbers`."""
        return dropout_opacity(opacity, self.p, self.seed, [self.first_view + int(k) for k in numbers], is_logit, ctx)


def dropout_opacity(opacity, p, seed, views, is_logit=False, ctx=None):
    """The opacities [V,N] that the V views numbered `views` see: keep(seed, i, view) ? o_i / (1 - p) : 0, with o the
    opacities [N] (their sigmoid when is_logit), 0 <= p < 1 (gs_opacity_dropout)."""
    c = _ctx(ctx)
    c.sync_stream()
    N, op = _opacity(opacity, c)
    ids, V = _view_ids(views)
    out = torch.empty((V, N), dtype=torch.float32, device=c.device)
    check(c.lib.gs_opacity_dropout(c.handle, N, _ptr(op), int(bool(is_logit)), float(p), _seed(seed), V, ids, _ptr(out)),
          "gs_opacity_dropout")
    return out if _is_t(opacity) else _np_out(out, np.float64)


def dropout_opacity_backward(d_opacities, opacity, p, seed, views, is_logit=False, ctx=None, out=None, accumulate=False):
    """Gradient [N] with respect to `opacity` of a loss whose gradients with respect to dropout_opacity's result are
    d_opacities [V,N] (gs_opacity_dropout_backward).  out [N] receives the result, added to what is there when
    accumulate."""
    c = _ctx(ctx)
    c.sync_stream()
    N, op = _opacity(opacity, c)
    ids, V = _view_ids(views)
    shape = tuple(d_opacities.shape)
    if shape != (V, N) and not (V == 1 and shape == (N,)):
        raise ValueError(f"d_opacities must be [{V},{N}], got {list(shape)}")
    d = _dev(d_opacities, torch.float32, c.device)
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty((N,), dtype=torch.float32, device=c.device)
    elif not _is_t(out) or out.dtype != torch.float32 or tuple(out.shape) != (N,) or not out.is_contiguous() or \
            out.device != c.device:
        raise ValueError(f"out must be a contiguous float32 [{N}] tensor on {c.device}")
    check(c.lib.gs_opacity_dropout_backward(c.handle, N, _ptr(op), int(bool(is_logit)), float(p), _seed(seed), V, ids, _ptr(d),
                                            int(bool(accumulate)), _ptr(out)), "gs_opacity_dropout_backward")
    return out if _is_t(opacity) else _np_out(out, np.float64)
