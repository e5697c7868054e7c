"""CPU: the packed SH that a view was rendered from stays with the view.  Through the stand-in library of
test_distributed_packed_cpu.py, whose records here also say which packing they come from."""
import ctypes

import numpy as np
import pytest
import torch

from test_distributed_cpu import FakeCtx, FakeStream, N, _scene, _views_targets
from test_distributed_packed_cpu import PackedLib


class CountingLib(PackedLib):
    """Word 1 of every record is the number of the packing; the parameter backward logs which packing it reads."""

    def __init__(self):
        super().__init__()
        self.packings = 0
        self.read = []                   # per K8 launch: (packing, views, accumulate)

    def _words(self, address, n):
        return np.ctypeslib.as_array((ctypes.c_uint32 * (8 * n)).from_address(address)).reshape(n, 8)

    def gs_sh_quantize(self, h, n, sh, words):
        self.packings += 1
        self._words(words.value, n)[:, 1] = self.packings
        return super().gs_sh_quantize(h, n, sh, words)

    def gs_backward_params_batch(self, h, n, means, ls, quats, sh, opacity, is_logit, n_views, views, accumulate, *tail):
        have, address = self.packed[h]
        assert have == n and not sh.value
        (packing,) = set(self._words(address, n)[:, 1].tolist())
        self.read.append((packing, n_views, int(accumulate)))
        return super().gs_backward_params_batch(h, n, means, ls, quats, sh, opacity, is_logit, n_views, views, accumulate, *tail)


class Ctx(FakeCtx):
    """Streams that note what they wait for."""

    def __init__(self, lib):
        super().__init__(lib)
        self.stream = Stream()

    def current_stream(self):
        return self.stream


class Stream(FakeStream):
    def __init__(self):
        self.waited, self.recorded = [], []

    def wait_event(self, event):
        self.waited.append(event)

    def record_event(self):
        self.recorded.append(object())
        return self.recorded[-1]


def _pipe():
    import gsplat_amd as gs
    lib = CountingLib()
    ctx = Ctx(lib)
    return gs, lib, ctx, gs.SplatPipeline(_scene(), [8, 6], ctx=ctx, sh_format="mxfp4")


def _render(pipe, view, **kw):
    image, state = pipe.forward(view, pre=pipe.preprocess_batch([view], **kw)[0])
    pipe.backward_rows(state, image)
    return state


def test_backward_reads_the_records_of_its_view():
    gs, lib, ctx, pipe = _pipe()
    views, _ = _views_targets(gs, 3)
    first = _render(pipe, views[0])
    pipe.sh.mul_(0.5)
    second = _render(pipe, views[1])                       # packed anew
    again = _render(pipe, views[2], repack=False)
    grads = gs.FlatGrads(N, torch.device("cpu"))
    pipe.backward_params([first], grads)
    pipe.backward_params([second, again], grads, accumulate=True)
    assert lib.read == [(1, 1, 0), (2, 2, 1)] and not lib.packed


def test_views_of_different_records_take_a_launch_each():
    gs, lib, ctx, pipe = _pipe()
    views, _ = _views_targets(gs, 4)
    states = [_render(pipe, v) for v in views[:2]] + [_render(pipe, v, repack=False) for v in views[2:]]
    for accumulate in (False, True):
        grads, want = (gs.FlatGrads(N, torch.device("cpu")) for _ in range(2))
        for g in (grads, want):
            g.flat.fill_(7.0)
        lib.read.clear()
        pipe.backward_params(states, grads, accumulate=accumulate)
        assert lib.read == [(1, 1, int(accumulate)), (2, 3, 1)]
        for k, st in enumerate(states):
            pipe.backward_params([st], want, accumulate=accumulate or k > 0)
        torch.testing.assert_close(grads.flat, want.flat, rtol=1e-6, atol=0)


def test_another_stream_waits_for_the_packing():
    gs, lib, ctx, pipe = _pipe()
    views, _ = _views_targets(gs, 2)
    packing_stream = ctx.stream
    first = _render(pipe, views[0])
    (packed,) = packing_stream.recorded
    grads = gs.FlatGrads(N, torch.device("cpu"))
    pipe.backward_params([first], grads)
    assert packing_stream.waited == []                     # in order already
    ctx.stream = Stream()
    second = _render(pipe, views[1])                       # its own packing, on its own stream
    assert ctx.stream.waited == []
    pipe.backward_params([second], grads)
    assert ctx.stream.waited == []
    pipe.backward_params([first], grads, g_range=(0, 400))
    assert ctx.stream.waited == [packed]
    ctx.stream = Stream()
    pipe.preprocess_batch(views, repack=False)             # K1 from the last packing
    assert len(ctx.stream.waited) == 1 and ctx.stream.waited != [packed]


def test_a_view_of_a_scene_that_has_grown_is_refused():
    gs, lib, ctx, pipe = _pipe()
    views, _ = _views_targets(gs, 1)
    state = _render(pipe, views[0])
    for name in ("means", "log_scales", "quats", "opacity", "sh"):
        t = getattr(pipe, name)
        setattr(pipe, name, torch.cat([t, t[:7]]))
    pipe.N = N + 7
    with pytest.raises(ValueError, match=f"rendered with {N} gaussians"):
        pipe.backward_params([state], gs.FlatGrads(N + 7, torch.device("cpu")))
    assert lib.read == []


def test_records_given_as_parameters_stay_the_callers():
    gs, lib, ctx, pipe = _pipe()
    g = _scene()
    g.spherical_harmonics = gs.quantize_sh(torch.from_numpy(g.spherical_harmonics), ctx=ctx)
    pipe = gs.SplatPipeline(g, [8, 6], ctx=ctx)
    views, _ = _views_targets(gs, 1)
    ctx.stream = Stream()
    state = _render(pipe, views[0])
    pipe.backward_params([state], gs.FlatGrads(N, torch.device("cpu")))
    assert lib.packings == 1 and lib.read == [(1, 1, 0)] and ctx.stream.waited == [] and ctx.stream.recorded == []


def test_a_pipeline_set_back_to_its_coefficients_reads_them():
    gs, lib, ctx, pipe = _pipe()
    views, _ = _views_targets(gs, 1)
    _render(pipe, views[0])
    pipe.sh_format = "fp32"
    pre = pipe.preprocess_batch(views, repack=False)[0]
    assert pre["packed"] is None and pipe._kept_sh(ctx) is pipe.sh
