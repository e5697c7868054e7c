"""GPU: packed SH and opacity dropout inside the hot path -- the array API, SplatPipeline, train_step, train_model -- against
the same path on the dequantised coefficients and on opacities that were dropped out by hand."""
import collections
import types
from importlib import import_module

import numpy as np
import pytest

from conftest import synth_scene
from oracle import packed_ref

pytestmark = pytest.mark.gpu


def _scene(n=1501, W=208, H=128, seed=5):
    cam, R, t, g, rs = synth_scene(n, W, H, seed=seed, fx=150.0, log_scale=(2.0, 3.2))
    g.opacity = np.random.default_rng(seed).normal(size=n).astype(np.float32)        # logits
    return cam, g, rs


def _views(gs, cam, n):
    out = []
    for k in range(n):
        a = .03 * (k - n / 2)
        R = np.array([[np.cos(a), 0, np.sin(a)], [0, 1, 0], [-np.sin(a), 0, np.cos(a)]])
        out.append(gs.View(cam, R, np.array([.05 * k, -.02 * k, .1])))
    return out


def _targets(ctx, rs, n):
    import torch
    gen = torch.Generator().manual_seed(4)
    return [torch.rand((rs[0], rs[1], 3), generator=gen).to(ctx.device) for _ in range(n)]


def _with(g, **kw):
    return types.SimpleNamespace(**{**g.__dict__, **kw})


@pytest.fixture()
def det_ctx(gpu_ctx):
    """A context whose blend backward adds in a fixed order, so that gradients can be compared bit for bit."""
    c = gpu_ctx.clone()
    c.set_option("deterministic_backward", 1)
    yield c
    c.close()


@pytest.mark.parametrize("cull", [True, False])
@pytest.mark.parametrize("general", [False, True])
def test_views_from_records_equal_views_from_their_coefficients(det_ctx, cull, general, monkeypatch):
    """K1 (both forms, 10 views: two launches), lists, image; K8 (both forms) to the rounding of its fp32 sums."""
    import torch
    import gsplat_amd as gs
    if general:
        monkeypatch.setenv("GS_K1_GENERAL", "1")
        monkeypatch.setenv("GS_K8_GENERAL", "1")
    cam, g, rs = _scene()
    packed = gs.quantize_sh(g.spherical_harmonics, ctx=det_ctx)
    a = gs.SplatPipeline(_with(g, spherical_harmonics=packed), rs, ctx=det_ctx, cull_tiles=cull)
    b = gs.SplatPipeline(_with(g, spherical_harmonics=packed.dequantize(det_ctx).cpu().numpy()), rs, ctx=det_ctx, cull_tiles=cull)
    views = _views(gs, cam, 10)
    for records in (True, False):
        pa, pb = (p.preprocess_batch(views, records=records) for p in (a, b))
        for x, y in zip(pa, pb):
            for key in ("rec", "depths", "clamped", "rect", "radii", "colors", "centers", "conics"):
                if x.get(key) is not None:
                    assert torch.equal(x[key], y[key]), key
    pa, pb = (p.preprocess_batch(views) for p in (a, b))
    grads = []
    for p, pres in ((a, pa), (b, pb)):
        states = []
        for v, pre in zip(views, pres):
            img, st = p.forward(v, pre=pre)
            p.backward_rows(st, img.contiguous())
            states.append((img, st))
        gr = gs.FlatGrads(p.N, det_ctx.device)
        p.backward_params([st for _, st in states], gr, g_range=None)
        grads.append((states, gr))
    for (ia, sa), (ib, sb) in zip(grads[0][0], grads[1][0]):
        assert torch.equal(ia, ib) and torch.equal(sa["rows"], sb["rows"])
    ga, gb = grads[0][1].flat, grads[1][1].flat
    scale = float(gb.abs().max())
    assert float((ga - gb).abs().max()) <= 2 ** -20 * scale and scale > 0
    # a range of gaussians reads its own records
    part = gs.FlatGrads(a.N, det_ctx.device)
    a.backward_params([s for _, s in grads[0][0]], part, g_range=(0, 700))
    a.backward_params([s for _, s in grads[0][0]], part, g_range=(700, a.N))
    assert torch.equal(part.flat, ga)
    # single view without preprocess_batch
    ia, _ = a.forward(views[0])
    assert torch.equal(ia, grads[0][0][0][0])


def test_array_api_takes_records(gpu_ctx):
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(900)
    packed = gs.quantize_sh(g.spherical_harmonics, ctx=gpu_ctx)
    dense = gs.GaussianSet(g.center, packed.dequantize(gpu_ctx).cpu().numpy(), g.scaling, g.rotation, g.opacity)
    small = gs.GaussianSet(g.center, packed.to("cpu"), g.scaling, g.rotation, g.opacity)
    R, t = np.eye(3), np.array([.1, 0, .2])
    fa, fb = (gs.forward_pass(gpu_ctx, None, None, cam, R, t, s, result_size=rs) for s in (small, dense))
    for x, y in zip(fa, fb):
        np.testing.assert_array_equal(x, y)
    rng = np.random.default_rng(0)
    up = [rng.normal(size=s) for s in ((900, 3), (900, 2), (900, 3))]
    back = []
    for s, f in ((small, fa), (dense, fb)):
        centers, depths, colors, conics, clamped, tt, radii, ws, ms, ts, c2, c3, dirs = f
        back.append(gs.backward_pass(gpu_ctx, None, None, cam, R, t, s, radii, c2, c3, ws, ms, ts, dirs, clamped, *up,
                                     result_size=rs))
    for x, y in zip(*back):
        np.testing.assert_allclose(x, y, rtol=0, atol=2 ** -20 * max(np.abs(y).max(), 1e-30))
    src = types.SimpleNamespace(qvec=np.array([1.0, 0, 0, 0]), tvec=np.zeros(3))
    ia, ib = (s.rasterize(cam, src, gpu_ctx, None, None, result_size=rs) for s in (small, dense))
    np.testing.assert_array_equal(ia, ib)
    # nothing stays bound: the next call reads its own coefficients
    fc = gs.forward_pass(gpu_ctx, None, None, cam, R, t, dense, result_size=rs)
    np.testing.assert_array_equal(fc[2], fb[2])


def test_records_of_another_scene_are_refused(gpu_ctx):
    import ctypes
    import gsplat_amd as gs
    cam, g, rs = _scene(300)
    packed = gs.quantize_sh(g.spherical_harmonics, ctx=gpu_ctx)
    pipe = gs.SplatPipeline(g, rs, ctx=gpu_ctx)
    view = _views(gs, cam, 1)[0]
    lib, h = gpu_ctx.lib, gpu_ctx.handle
    try:
        assert lib.gs_ctx_use_packed_sh(h, 299, ctypes.c_void_p(packed.words.data_ptr())) == 0
        with pytest.raises(gs.GsError, match="N=299"):
            pipe.forward(view)
        with pytest.raises(gs.GsError, match="N=299"):
            pipe.preprocess_batch([view])
        assert lib.gs_ctx_use_packed_sh(h, 300, ctypes.c_void_p(packed.words.data_ptr() + 4)) < 0      # alignment
    finally:
        assert lib.gs_ctx_use_packed_sh(h, 0, None) == 0
    pipe.forward(view)
    null, ptr = ctypes.c_void_p(0), ctypes.c_void_p(pipe.sh.data_ptr())
    check = import_module("gaussian-splatting_amd._lib").check
    with pytest.raises(gs.GsError, match="no packed records"):                       # neither coefficients nor records
        check(lib.gs_preprocess_batch_records(h, 300, ptr, ptr, ptr, null, ptr, 1,
                                              (import_module("gaussian-splatting_amd._lib").GsViewRecords * 1)()), "K1")
    with pytest.raises(gs.GsError, match="no packed records"):
        check(lib.gs_backward_params_batch(h, 300, ptr, ptr, ptr, null, ptr, 0, 0, None, 0, ptr, ptr, ptr, ptr, ptr), "K8")
    with pytest.raises(gs.GsError, match="opacity_stride"):
        import_module("gaussian-splatting_amd._lib").check(lib.gs_preprocess_batch_records_views(h, 300, *([ctypes.c_void_p(pipe.sh.data_ptr())] * 5), 299, 1,
                                                            (import_module("gaussian-splatting_amd._lib").GsViewRecords * 1)()), "views")


@pytest.mark.parametrize("lanes,args", [(1, {}), (3, {}), (4, {}), (4, {"prepared": True}), (2, {"batch_binning": True}),
                                        (2, {"fused_loss": True})])
def test_step_with_dropout_equals_views_dropped_by_hand(det_ctx, lanes, args):
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene()
    views, targets = _views(gs, cam, 5), _targets(det_ctx, rs, 5)
    drop = gs.OpacityDropout(.3, 77, first_view=2 ** 33 + 2)
    pipe = gs.SplatPipeline(g, rs, ctx=det_ctx, sh_format="mxfp4")
    grads = gs.FlatGrads(pipe.N, det_ctx.device)
    loss, _ = gs.train_step(pipe, views, targets, grads, concurrent_views=lanes, dropout=drop, **args)
    torch.cuda.synchronize()
    # by hand: the opacities of each view as raw opacities of a pipeline of its own
    keep = packed_ref.keep_mask(pipe.N, .3, 77, [2 ** 33 + 2 + v for v in range(5)])
    x = g.opacity.astype(np.float64)
    o = 1 / (1 + np.exp(-x))
    dropped = gs.dropout_opacity(pipe.opacity, .3, 77, [2 ** 33 + 2 + v for v in range(5)], is_logit=True, ctx=det_ctx)
    want = np.zeros((pipe.N, 59))
    want_loss, dsh = 0.0, packed_ref.dequantize(packed_ref.quantize(g.spherical_harmonics)).astype(np.float32)
    for v in range(5):
        by_hand = gs.SplatPipeline(_with(g, opacity=dropped[v], spherical_harmonics=dsh),
                                   rs, opacity_is_logit=False, ctx=det_ctx)
        gv = gs.FlatGrads(pipe.N, det_ctx.device)
        lv, _ = gs.train_step(by_hand, [views[v]], [targets[v]], gv, concurrent_views=1)
        want_loss += float(lv)
        parts = [gv.means, gv.log_scales, gv.quats, gv.opacity[:, None] * torch.from_numpy((o * (1 - o) * keep[v] / .7)[:, None]).to(det_ctx.device),
                 gv.sh.reshape(-1, 48)]
        want += torch.cat([p.double().reshape(pipe.N, -1) for p in parts], dim=1).cpu().numpy()
        # gradients of left-out gaussians are zero, all of them
        out = torch.from_numpy(~keep[v]).to(det_ctx.device)
        for p in (gv.means, gv.log_scales, gv.quats, gv.opacity, gv.sh):
            assert (p[out] == 0).all()
    got = torch.cat([p.double().reshape(pipe.N, -1) for p in (grads.means, grads.log_scales, grads.quats, grads.opacity, grads.sh)],
                    dim=1).cpu().numpy()
    # the same images and rows; K8's sums over 5 views are fp32 in another order (5 x 48 terms at most), and the sigmoid's
    # derivative is K8's own __expf: 2^-16 of the largest gradient of each parameter group
    for sl in (slice(0, 3), slice(3, 6), slice(6, 10), slice(10, 11), slice(11, 59)):
        assert np.abs(got[:, sl] - want[:, sl]).max() <= 2 ** -16 * np.abs(want[:, sl]).max()
    assert abs(float(loss) - want_loss) <= 1e-6 * want_loss
    # without dropout the step is another one
    plain = gs.FlatGrads(pipe.N, det_ctx.device)
    gs.train_step(pipe, views, targets, plain, concurrent_views=lanes, **args)
    assert not torch.equal(plain.flat, grads.flat)


def test_step_repeats_with_its_numbers_and_changes_with_them(det_ctx):
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(700)
    views, targets = _views(gs, cam, 4), _targets(det_ctx, rs, 4)
    pipe = gs.SplatPipeline(g, rs, ctx=det_ctx)

    def step(**kw):
        gr = gs.FlatGrads(pipe.N, det_ctx.device)
        gs.train_step(pipe, views, targets, gr, concurrent_views=4, dropout=gs.OpacityDropout(**kw))
        torch.cuda.synchronize()
        return gr.flat
    a = step(p=.2, seed=1, first_view=8)
    assert torch.equal(a, step(p=.2, seed=1, first_view=8))
    assert not torch.equal(a, step(p=.2, seed=2, first_view=8)) and not torch.equal(a, step(p=.2, seed=1, first_view=12))


def test_dropout_in_front_of_the_array_api(gpu_ctx):
    """dropout_opacity -> gpu_rasterize -> dropout_opacity_backward: the gradient of the opacities against differences."""
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(400, 96, 64)
    d = gpu_ctx.device
    gt = gs.GaussianSet(*(torch.from_numpy(np.ascontiguousarray(a)).to(d) for a in
                          (g.center, g.spherical_harmonics, g.scaling, g.rotation, g.opacity)))
    R, t = np.eye(3), np.zeros(3)
    centers, depths, colors, conics, _, tt, radii = gs.forward_pass(gpu_ctx, None, None, cam, R, t, gt, result_size=rs)[:7]
    b = gs.match_gaus_to_tiles(gpu_ctx, None, None, tt, radii, depths, result_size=rs)
    gen = torch.Generator().manual_seed(0)
    up = torch.rand((rs[0], rs[1], 3), generator=gen).to(d)

    def loss(x, training=False):
        op = gs.dropout_opacity(x, .4, 3, [17], is_logit=True, ctx=gpu_ctx)[0]
        out = gs.gpu_rasterize(gpu_ctx, None, None, centers, colors, op, conics, b, training=training, result_size=rs, dL_dimage=up)
        return out if training else float((out.double() * up).sum())
    d_op = loss(gt.opacity, training=True)[4]
    got = gs.dropout_opacity_backward(d_op, gt.opacity, .4, 3, [17], is_logit=True, ctx=gpu_ctx).cpu().numpy()
    keep = packed_ref.keep_mask(400, .4, 3, [17])[0]
    assert (got[~keep] == 0).all() and np.abs(got[keep]).max() > 0
    # along the gradient of the kept gaussians.  The contour where a gaussian is cut off (alpha 1/255) moves with its opacity
    # o, which the gradient leaves out: 1 / (255 o) of its share, 4 % at o = .1; the curvature over .02 is below 1 %
    h = 0.02
    step = torch.from_numpy(got / np.linalg.norm(got)).to(d).float()
    diff = (loss(gt.opacity + h * step) - loss(gt.opacity - h * step)) / (2 * h)
    assert abs(diff - np.linalg.norm(got)) <= 0.05 * np.linalg.norm(got)


def _colmap(cam, W, H):
    Camera = collections.namedtuple("Camera", ["id", "model", "width", "height", "params"])
    Image = collections.namedtuple("Image", ["id", "qvec", "tvec", "camera_id", "name"])
    cameras = {1: Camera(1, "PINHOLE", W, H, np.array(cam.params))}
    images = {k + 1: Image(k + 1, np.array([np.cos(.02 * k), 0.0, np.sin(.02 * k), 0.0]), np.array([.02 * k, 0, .1]), 1, f"{k}.jpg")
              for k in range(6)}
    return cameras, images


@pytest.mark.parametrize("drop_rate", [0.15, lambda i: 0.0 if i == 0 else 0.05 * i])
def test_train_model_with_both(gpu_ctx, tmp_path, drop_rate):
    """Runs, grows by densification, writes packed checkpoints that render what the trained pipeline renders."""
    import torch
    import gsplat_amd as gs
    W, H = 96, 64
    cam, _, _, g, rs = synth_scene(500, W, H, seed=3, fx=70.0, log_scale=(2.0, 3.0), degree=3)
    cameras, images = _colmap(cam, W, H)
    target = np.random.default_rng(0).uniform(size=(W, H, 3)).astype(np.float32)
    logs = []
    out, hist = gs.train_model(cameras, images, None, gs.REFERENCE_LEARNING_RATES, gpu_ctx, iters=6, result_size=rs,
                               views_per_step=3, image_loader=lambda src: target, output_dir=str(tmp_path), subset_fraction=.9,
                               seed=5, gaussians=g, save_images_every=0, checkpoint_every=3, concurrent_views=2, log=logs.append,
                               densify_every=2, densify_from=1, densify_options={"grad_threshold": 1e-7}, drop_rate=drop_rate,
                               sh_format="mxfp4")
    assert len(hist) == 7 and np.all(np.isfinite(hist)) and len(out.center) > 500
    for name in ("center", "scaling", "rotation", "opacity", "spherical_harmonics"):
        assert np.all(np.isfinite(getattr(out, name)))
    packed = gs.load_gaussians(str(tmp_path / "iter_6_packed"))
    dense = gs.load_gaussians(str(tmp_path / "iter_6_gaus"))
    np.testing.assert_array_equal(packed.spherical_harmonics.numpy(), packed_ref.quantize(dense.spherical_harmonics))
    view = gs.View(cameras[1], np.eye(3), np.zeros(3))
    ia, _ = gs.SplatPipeline(packed, rs, opacity_is_logit=False, ctx=gpu_ctx).forward(view)
    trained = gs.SplatPipeline(dense, rs, opacity_is_logit=False, ctx=gpu_ctx, sh_format="mxfp4")
    ib, _ = trained.forward(view)
    assert torch.equal(ia, ib)
    small, big = ((tmp_path / f"iter_6_{k}.npz").stat().st_size for k in ("packed", "gaus"))
    assert small < big / 2
    # export: coefficients, records, and both ways from records alone
    assert gs.SplatPipeline(packed, rs, ctx=gpu_ctx).export(packed=False).spherical_harmonics.shape == (len(out.center), 3, 16)
    np.testing.assert_array_equal(trained.export(packed=True).spherical_harmonics.numpy(), packed.spherical_harmonics.numpy())
    gs.save_ply(str(tmp_path / "p.ply"), packed)
    np.testing.assert_array_equal(gs.load_data(str(tmp_path / "p.ply")).spherical_harmonics,
                                  packed.spherical_harmonics.dequantize(gpu_ctx).cpu().numpy())


def test_changed_coefficients_are_packed_again(gpu_ctx):
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(300)
    pipe = gs.SplatPipeline(g, rs, ctx=gpu_ctx, sh_format="mxfp4")
    view = _views(gs, cam, 1)[0]
    a, _ = pipe.forward(view)
    pipe.sh.mul_(0.5)                                   # behind the pipeline's back
    b, _ = pipe.forward(view)
    c, _ = pipe.forward(view, pre=pipe.preprocess_batch([view])[0])
    assert not torch.equal(a, b) and torch.equal(b, c)


def test_densifier_does_not_count_left_out_views(gpu_ctx):
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(400)
    g.opacity = np.abs(g.opacity)
    pipe = gs.SplatPipeline(g, rs, ctx=gpu_ctx)
    den = gs.Densifier(pipe)
    views, targets = _views(gs, cam, 4), _targets(gpu_ctx, rs, 4)
    radii = [st["radii"] for st in pipe.preprocess_batch(views)]
    gs.train_step(pipe, views, targets, gs.FlatGrads(pipe.N, gpu_ctx.device), concurrent_views=2, states_hook=den.accumulate,
                  dropout=gs.OpacityDropout(.5, 3, first_view=40))
    keep = torch.from_numpy(packed_ref.keep_mask(pipe.N, .5, 3, range(40, 44))).to(gpu_ctx.device)
    want = sum(((r > 0) & k).float() for r, k in zip(radii, keep))
    assert torch.equal(den.denom, want) and 0 < float(want.sum()) < sum(int((r > 0).sum()) for r in radii)


@pytest.mark.parametrize("lanes", [1, 4])
@pytest.mark.parametrize("ordered", [False, True])
def test_step_in_which_every_gaussian_is_left_out(gpu_ctx, det_ctx, lanes, ordered):
    """Empty lists, and exact lists whose entries do nothing, with both reductions of the blend backward: the background, no
    gradient, a finite loss."""
    gpu_ctx = det_ctx if ordered else gpu_ctx
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(200, 96, 64)
    assert not packed_ref.keep_mask(200, .9999999, 1, range(4)).any()
    for cull in (True, False):
        pipe = gs.SplatPipeline(g, rs, ctx=gpu_ctx, cull_tiles=cull, sh_format="mxfp4", background=(.2, .3, .4))
        views, targets = _views(gs, cam, 4), _targets(gpu_ctx, rs, 4)
        drop = gs.OpacityDropout(.9999999, 1)
        grads = gs.FlatGrads(pipe.N, gpu_ctx.device)
        grads.flat.fill_(3.0)
        loss, _ = gs.train_step(pipe, views, targets, grads, concurrent_views=lanes, dropout=drop)
        bg = torch.tensor([.2, .3, .4], device=gpu_ctx.device)
        want = sum(((bg - t) ** 2).mean() for t in targets)
        assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
        for part in (grads.means, grads.log_scales, grads.quats, grads.opacity, grads.sh):
            assert (part == 0).all()
        image, _ = pipe.forward(views[0], pre=pipe.preprocess_batch(views[:1], dropout=drop)[0])
        assert torch.equal(image, bg.expand_as(image))
