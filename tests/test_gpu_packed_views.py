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
