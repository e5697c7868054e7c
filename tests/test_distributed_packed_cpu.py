"""CPU, world_size 1 and 2 (gloo): train_step with packed SH and opacity dropout through the stand-in library of
test_distributed_cpu.py.  Every view must get the opacities of its own number (its place in the whole batch, whichever rank
renders it), K8 the records of its range of gaussians and the scale of the dropout, and nothing may stay bound."""
import ctypes
import os
import sys

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from conftest import ROOT
from test_distributed_cpu import FakeCtx, FakeLib, N, _check, _f32, _free_port, _scene, _views_targets

P_DROP, SEED, FIRST = 0.25, 99, 1000


class PackedLib(FakeLib):
    """Record i starts with the word i; the opacities of view number s are s + 1 / 1024 everywhere."""

    def __init__(self):
        super().__init__()
        self.packed = {}                 # ctx handle -> (N, address) while bound
        self.numbers = []                # (camera's view id, view number its opacities carry)

    def gs_sh_quantize(self, h, n, sh, words):
        np.ctypeslib.as_array((ctypes.c_uint32 * (8 * n)).from_address(words.value)).reshape(n, 8)[:, 0] = np.arange(n)
        self.log.append(("pack", n))
        return 0

    def gs_ctx_use_packed_sh(self, h, n, words):
        if words is None:
            del self.packed[h]
        else:
            self.packed[h] = (n, words.value)
        return 0

    def _first_record(self, h, n):
        have, addr = self.packed[h]
        assert have == n
        return int(ctypes.c_uint32.from_address(addr).value)

    def gs_opacity_dropout(self, h, n, opacity, is_logit, p, seed, n_views, ids, out):
        assert p == P_DROP and seed == SEED and is_logit == 1
        o = _f32(out, n_views * n).reshape(n_views, n) if n_views else None
        for k in range(n_views):
            o[k] = ids[k] + 1 / 1024
        return 0

    def gs_preprocess_batch_records_views(self, h, n, means, ls, quats, sh, opac, stride, n_views, arr):
        assert not sh.value and self._first_record(h, n) == 0 and stride == n
        o = _f32(opac, n_views * n).reshape(n_views, n) if n_views else None      # a rank may have no view
        for k in range(n_views):
            assert (o[k] == o[k, 0]).all()
            self.numbers.append((int(arr[k].cam.contents.fx), int(o[k, 0])))
        return self.gs_preprocess_batch_records(h, n, means, ls, quats, sh, opac, n_views, arr)

    def gs_backward_params_batch_scaled(self, h, n, means, ls, quats, sh, opacity, is_logit, n_views, views, scale, *tail):
        assert not sh.value
        if n:
            r = _f32(views[0].grad_rows, n * 16).reshape(n, 16)
            assert self._first_record(h, n) == int(r[0, 1])         # rows carry the gaussian's global index
        assert all(abs(scale[k] - 1 / (1 - P_DROP)) < 1e-7 for k in range(n_views))
        return self.gs_backward_params_batch(h, n, means, ls, quats, sh, opacity, is_logit, n_views, views, *tail)


def _run(n_views, lanes, **step_args):
    import gsplat_amd as gs
    lib = PackedLib()
    pipe = gs.SplatPipeline(_scene(), [8, 6], ctx=FakeCtx(lib), sh_format="mxfp4")
    grads = gs.FlatGrads(N, torch.device("cpu"))
    grads.flat.fill_(123.0)
    views, targets = _views_targets(gs, n_views)
    gs.train_step(pipe, views, targets, grads, concurrent_views=lanes,
                  dropout=gs.OpacityDropout(P_DROP, SEED, first_view=FIRST), **step_args)
    assert not lib.packed, "records stayed bound"
    return lib, grads


@pytest.mark.parametrize("n_views,lanes,args", [(8, 4, {}), (5, 4, {}), (1, 1, {}), (3, 1, {}), (8, 2, {"prepared": True}),
                                                (6, 3, {"batch_binning": True, "bin_group": 2})])
def test_one_rank(n_views, lanes, args):
    lib, grads = _run(n_views, lanes, **args)
    _check(grads, n_views, str(args))
    assert sorted(lib.numbers) == [(v, FIRST + v) for v in range(n_views)]
    assert [e for e in lib.log if e[0] == "pack"] == [("pack", N)]              # once per step


def _worker(rank, world, port, n_views, out):
    sys.path.insert(0, ROOT)
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    import datetime
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
    lib, grads = _run(n_views, 4)
    torch.save({"flat": grads.flat.clone(), "numbers": lib.numbers}, os.path.join(out, f"rank{rank}.pt"))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("n_views", [8, 5, 1])
def test_two_ranks_number_the_views_of_the_whole_batch(tmp_path, n_views):
    import gsplat_amd as gs
    mp.spawn(_worker, args=(2, _free_port(), n_views, str(tmp_path)), nprocs=2, join=True)
    r = [torch.load(os.path.join(tmp_path, f"rank{k}.pt")) for k in range(2)]
    assert torch.equal(r[0]["flat"], r[1]["flat"])
    full = gs.FlatGrads(N, torch.device("cpu"))
    full.flat.copy_(r[0]["flat"])
    _check(full, n_views, "2 ranks")
    for k in range(2):
        assert sorted(r[k]["numbers"]) == [(v, FIRST + v) for v in range(n_views) if v % 2 == k]


def test_records_are_packed_again_when_the_scene_has_grown():
    """K8 reads N records: those of a smaller scene are never taken."""
    import gsplat_amd as gs
    lib = PackedLib()
    pipe = gs.SplatPipeline(_scene(), [8, 6], ctx=FakeCtx(lib), sh_format="mxfp4")
    pipe.pack_sh()
    for name in ("means", "log_scales", "quats", "opacity", "sh"):
        t = getattr(pipe, name)
        setattr(pipe, name, torch.cat([t, t[:7]]))
    pipe.N = N + 7
    assert len(pipe._kept_sh(pipe.ctx)) == N + 7 and len(pipe.packed) == N + 7


def test_pipelines_without_coefficients_are_not_trained():
    import types
    import gsplat_amd as gs
    g = _scene()
    g.spherical_harmonics = gs.PackedSH(torch.zeros((N, 8), dtype=torch.int32))
    pipe = gs.SplatPipeline(g, [8, 6], ctx=FakeCtx(PackedLib()))
    assert pipe.sh is None and pipe.sh_format == "mxfp4" and len(pipe.pack_sh()) == N
    with pytest.raises(ValueError, match="packed SH only"):
        gs.Optimizer(pipe)
    with pytest.raises(ValueError, match="packed SH only"):
        gs.Densifier(pipe)
    with pytest.raises(ValueError, match="sh_format"):
        gs.SplatPipeline(g, [8, 6], ctx=FakeCtx(PackedLib()), sh_format="fp32")
    with pytest.raises(ValueError, match="sh_format"):
        gs.SplatPipeline(_scene(), [8, 6], ctx=FakeCtx(PackedLib()), sh_format="int4")
    with pytest.raises(ValueError, match="dropout probability"):
        gs.OpacityDropout(1.0)
    with pytest.raises(ValueError, match="seed"):
        gs.OpacityDropout(.1, seed=-3)
    pipe = gs.SplatPipeline(_scene(), [8, 6], ctx=FakeCtx(PackedLib()))
    view = gs.View(types.SimpleNamespace(params=[1., 1.], width=8, height=6), np.eye(3), np.zeros(3))
    with pytest.raises(ValueError, match="view numbers"):
        pipe.preprocess_batch([view, view], dropout=gs.OpacityDropout(P_DROP, SEED), numbers=[0])


def test_packed_checkpoint_round_trip(tmp_path):
    import gsplat_amd as gs
    words = np.random.default_rng(0).integers(0, 2 ** 32, (11, 8), dtype=np.uint32)
    g = gs.GaussianSet(np.ones((11, 3)), gs.PackedSH(words), np.zeros((11, 3)), np.ones((11, 4)), np.full(11, .5), 2)
    gs.save_gaussians(str(tmp_path / "small"), g)
    back = gs.load_gaussians(str(tmp_path / "small"), degrees=2)
    np.testing.assert_array_equal(back.spherical_harmonics.numpy(), words)
    np.testing.assert_array_equal(back.center, g.center)
    with np.load(tmp_path / "small.npz") as d:
        np.testing.assert_array_equal(d["arr_1"], words.view(np.float16)[:, :3].astype(np.float64))
    bad = gs.GaussianSet(np.ones((10, 3)), gs.PackedSH(words), np.zeros((10, 3)), np.ones((10, 4)), np.full(10, .5), 2)
    gs.save_gaussians(str(tmp_path / "bad"), bad)
    with pytest.raises(ValueError, match="packed SH records"):
        gs.load_gaussians(str(tmp_path / "bad"))
