"""GPU: views rendered from packed SH on several streams and behind changed coefficients, against the same views one by one."""
import numpy as np
import pytest

from test_gpu_packed_train import _scene, _targets, _views, det_ctx   # noqa: F401

pytestmark = pytest.mark.gpu


def test_forwards_on_two_lanes_before_their_backwards(det_ctx):      # noqa: F811
    """Every forward packs on its own stream; the coefficients change in between; the backwards come last, on a third."""
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(3001)
    views, targets = _views(gs, cam, 4), _targets(det_ctx, rs, 4)
    pipe = gs.SplatPipeline(g, rs, ctx=det_ctx, sh_format="mxfp4")
    main = det_ctx.current_stream()
    scale = [1.0, 0.5, -1.0, 0.25]

    def run(k, ctx):
        image, st = pipe.forward(views[k], ctx=ctx)
        dL, _ = pipe.image_loss(image, targets[k], "l2", ctx=ctx)
        pipe.backward_rows(st, dL)
        return st

    want = gs.FlatGrads(pipe.N, det_ctx.device)
    sh = pipe.sh.clone()
    for k in range(4):
        pipe.sh.copy_(scale[k] * sh)
        pipe.backward_params([run(k, det_ctx)], want, accumulate=k > 0)
    torch.cuda.synchronize()
    pipe.sh.copy_(sh)
    lanes = pipe.lanes(2)
    states = []
    for k in range(4):
        ctx, stream = lanes[k % 2]
        for _, other in lanes:                          # the coefficients change when every lane has packed its own
            main.wait_stream(other)
        pipe.sh.copy_(scale[k] * sh)
        stream.wait_stream(main)
        with det_ctx.use_stream(stream):
            states.append(run(k, ctx))
    third = det_ctx.new_stream()
    for _, stream in lanes:
        third.wait_stream(stream)
    got = gs.FlatGrads(pipe.N, det_ctx.device)
    third.wait_stream(main)
    with det_ctx.use_stream(third):
        pipe.backward_params(states, got)               # four packings: four launches, in the order of the views
    main.wait_stream(third)
    torch.cuda.synchronize()
    assert torch.equal(got.flat, want.flat) and float(want.flat.abs().max()) > 0
    # the packings really differ: with the records of one view for all, another gradient
    same = gs.FlatGrads(pipe.N, det_ctx.device)
    pipe.backward_params([dict(st, packed=states[0]["packed"]) for st in states], same)
    assert not torch.equal(same.flat, got.flat)


@pytest.mark.parametrize("degree,switches", [(0, {}), (1, {}), (2, {}), (3, dict(apply_view=True)), (3, dict(diag_scale=True)),
                                             (1, dict(apply_view=True, diag_scale=True))])
@pytest.mark.parametrize("dropout", [False, True])
def test_records_in_every_form_of_the_parameter_kernels(det_ctx, degree, switches, dropout):      # noqa: F811
    """Lower degrees and the camera switches, 9 views (two K1 launches): from records as from their coefficients."""
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(1003)
    g.degrees = degree
    packed = gs.quantize_sh(g.spherical_harmonics, ctx=det_ctx)
    views, targets = _views(gs, cam, 9), _targets(det_ctx, rs, 9)
    drop = gs.OpacityDropout(.25, 5, first_view=6) if dropout else None
    out = []
    for sh in (packed, packed.dequantize(det_ctx)):
        scene = gs.GaussianSet(*(torch.as_tensor(a).to(det_ctx.device) for a in (g.center,)), sh,
                               *(torch.as_tensor(a).to(det_ctx.device) for a in (g.scaling, g.rotation, g.opacity)), degree)
        pipe = gs.SplatPipeline(scene, rs, ctx=det_ctx, **switches)
        pres = pipe.preprocess_batch(views, dropout=drop)
        grads = gs.FlatGrads(pipe.N, det_ctx.device)
        loss, _ = gs.train_step(pipe, views, targets, grads, concurrent_views=2, dropout=drop)
        torch.cuda.synchronize()
        out.append((pres, grads, float(loss)))
    (pa, ga, la), (pb, gb, lb) = out
    for x, y in zip(pa, pb):
        for key in ("rec", "depths", "clamped", "rect", "radii"):
            assert torch.equal(x[key], y[key]), key
    assert la == lb
    for name in ("means", "log_scales", "quats", "opacity", "sh"):
        a, b = getattr(ga, name), getattr(gb, name)
        # the same rows; the two instances of K8 may contract other products: fp32 sums of a few dozen terms
        assert float((a - b).abs().max()) <= 2 ** -20 * float(b.abs().max()) and float(b.abs().max()) > 0, name
    assert (ga.sh[:, :, (degree + 1) ** 2:] == 0).all()


@pytest.mark.parametrize("lanes", [1, 4])
def test_dropout_on_the_exact_lists(det_ctx, lanes):      # noqa: F811
    """Left-out gaussians keep their place in the exact lists and do nothing there: the step of the culled lists."""
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene()
    views, targets = _views(gs, cam, 5), _targets(det_ctx, rs, 5)
    drop = gs.OpacityDropout(.3, 77, first_view=2 ** 33 + 2)
    got = []
    for cull in (True, False):
        pipe = gs.SplatPipeline(g, rs, ctx=det_ctx, sh_format="mxfp4", cull_tiles=cull)
        grads = gs.FlatGrads(pipe.N, det_ctx.device)
        loss, _ = gs.train_step(pipe, views, targets, grads, concurrent_views=lanes, dropout=drop)
        image, _ = pipe.forward(views[1], pre=pipe.preprocess_batch(views[:2], dropout=drop)[1])
        torch.cuda.synchronize()
        got.append((grads, float(loss), image))
    (a, la, ia), (b, lb, ib) = got
    assert torch.equal(ia, ib) and la == lb
    for name in ("means", "log_scales", "quats", "opacity", "sh"):
        x, y = getattr(a, name), getattr(b, name)
        # the rows' sums in another order: 2^-18 of the largest gradient (fp32 sums over a few thousand pixels)
        assert float((x - y).abs().max()) <= 2 ** -18 * float(y.abs().max()) and float(y.abs().max()) > 0, name
    # and by hand, on the exact lists themselves: the opacities of each view as those of a pipeline of its own
    dropped = gs.dropout_opacity(torch.as_tensor(g.opacity).to(det_ctx.device), .3, 77, [2 ** 33 + 2 + v for v in range(5)],
                                 is_logit=True, ctx=det_ctx)
    want = 0.0
    for v in range(5):
        scene = gs.GaussianSet(g.center, gs.quantize_sh(g.spherical_harmonics, ctx=det_ctx), g.scaling, g.rotation, dropped[v])
        by_hand = gs.SplatPipeline(scene, rs, ctx=det_ctx, opacity_is_logit=False, cull_tiles=False)
        gv = gs.FlatGrads(by_hand.N, det_ctx.device)
        gs.train_step(by_hand, [views[v]], [targets[v]], gv, concurrent_views=1)
        assert (gv.means[dropped[v] == 0] == 0).all() and (gv.sh[dropped[v] == 0] == 0).all()
        want = want + gv.sh.double()
    assert float((b.sh.double() - want).abs().max()) <= 2 ** -18 * float(want.abs().max())


def test_captured_between_eager_launches(det_ctx):      # noqa: F811
    """K1 with its packing, and K8 of views that were rendered before, in a graph on another stream: each replay reads the
    coefficients and rows as they are then, and eager launches go on around it."""
    import torch
    import gsplat_amd as gs
    cam, g, rs = _scene(1003)
    views, targets = _views(gs, cam, 3), _targets(det_ctx, rs, 3)
    pipe = gs.SplatPipeline(g, rs, ctx=det_ctx, sh_format="mxfp4")

    def rendered():
        states = []
        for k, pre in enumerate(pipe.preprocess_batch(views)):
            image, st = pipe.forward(views[k], pre=pre)
            pipe.backward_rows(st, pipe.image_loss(image, targets[k], "l2")[0])
            states.append(st)
        return states

    states = rendered()
    out = gs.FlatGrads(pipe.N, det_ctx.device)
    side = det_ctx.new_stream()
    side.wait_stream(det_ctx.current_stream())
    with det_ctx.use_stream(side):
        pipe.backward_params(states, out)
        pipe.preprocess_batch(views)
    det_ctx.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pres = pipe.preprocess_batch(views)
        pipe.backward_params(states, out)
    captured = pres[0]["packed"]
    assert captured is not states[0]["packed"]
    sh = pipe.sh.clone()
    for scale in (1.0, 0.5, -2.0):
        pipe.sh.copy_(scale * sh)
        for st in states:
            st["rows"].mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        want = gs.FlatGrads(pipe.N, det_ctx.device)
        pipe.backward_params(states, want)
        for a, b in zip(pres, pipe.preprocess_batch(views)):
            assert torch.equal(a["rec"], b["rec"]) and torch.equal(a["clamped"], b["clamped"])
        assert torch.equal(out.flat, want.flat) and float(want.flat.abs().max()) > 0
        torch.cuda.synchronize()
    # the records packed inside the graph serve an eager launch too
    same = gs.FlatGrads(pipe.N, det_ctx.device)
    pipe.backward_params([dict(st, packed=captured) for st in states], same)
    fresh = [dict(st, packed=pre["packed"]) for st, pre in zip(states, pipe.preprocess_batch(views))]
    want = gs.FlatGrads(pipe.N, det_ctx.device)
    pipe.backward_params(fresh, want)
    torch.cuda.synchronize()
    assert torch.equal(same.flat, want.flat)
