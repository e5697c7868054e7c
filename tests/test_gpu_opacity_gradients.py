"""GPU: gradients with respect to opacity logits far from 0, where the opacity is 1 or 0 to fp32 and its derivative is not.
u = 2^-24 is half a step of fp32."""
import numpy as np
import pytest

from oracle import packed_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
FAR = [12.0, 16.0, 16.7, 17.4, 20.0, 33.0, 60.0, 80.0]


@pytest.mark.parametrize("n", [257, (1 << 19) + 3])          # one gaussian per thread; four
@pytest.mark.parametrize("p,views", [(0.0, [5]), (0.25, [0, 1, 2, 3, 9])])
def test_dropout_gradient_of_confident_gaussians(gpu_ctx, n, p, views):
    import torch
    import gsplat_amd as gs
    rng = np.random.default_rng(n)
    x = (rng.normal(size=n) * 6).astype(np.float32)
    x[:2 * len(FAR)] = FAR + [-v for v in FAR]
    x[-len(FAR):] = FAR
    g = rng.normal(size=(len(views), n)).astype(np.float32)
    keep = np.ones((len(views), n), bool)
    if p:
        ones = gs.dropout_opacity(torch.ones(n, device=gpu_ctx.device), p, 3, views, ctx=gpu_ctx)
        keep = (ones != 0).cpu().numpy()
        np.testing.assert_array_equal(keep[:, :300], packed_ref.keep_mask(min(n, 300), p, 3, views))
    got = gs.dropout_opacity_backward(torch.from_numpy(g).to(gpu_ctx.device), torch.from_numpy(x).to(gpu_ctx.device), p, 3, views,
                                      is_logit=True, ctx=gpu_ctx).cpu().numpy()
    e = np.exp(-np.abs(x.astype(np.float64)))
    act = e / (1 + e) ** 2
    s = np.where(keep, g.astype(np.float64), 0)
    # exp to one step (2 u, at most as much in the quotient), 1 + e twice, its square, the quotient: 6 u; the two products and
    # the scale's rounding: 3 u; the sum
    tol = np.abs(s).sum(axis=0) * act / (1 - p) * (9 + len(views)) * U
    assert (np.abs(got - s.sum(axis=0) * act / (1 - p)) <= tol).all()
    assert (got[:2 * len(FAR)][keep.all(axis=0)[:2 * len(FAR)]] != 0).all()


@pytest.mark.parametrize("general", [False, True])
def test_parameter_backward_of_confident_gaussians(gpu_ctx, general, monkeypatch):
    """K8 on logits against K8 on the opacities they stand for: the same images and rows, times the derivative."""
    import torch
    import gsplat_amd as gs
    from test_gpu_packed_train import _scene, _targets, _views, _with
    if general:
        monkeypatch.setenv("GS_K8_GENERAL", "1")
    c = gpu_ctx.clone()
    c.set_option("deterministic_backward", 1)
    cam, g, rs = _scene(1501)
    x = np.random.default_rng(2).choice([2.0, 7.5] + FAR, size=1501).astype(np.float32)
    views, targets = _views(gs, cam, 3), _targets(c, rs, 3)
    logits = gs.SplatPipeline(_with(g, opacity=x), rs, ctx=c)
    raw = gs.SplatPipeline(_with(g, opacity=torch.sigmoid(logits.opacity)), rs, ctx=c, opacity_is_logit=False)
    grads = []
    for pipe in (logits, raw):
        gr = gs.FlatGrads(pipe.N, c.device)
        gs.train_step(pipe, views, targets, gr, concurrent_views=1)
        torch.cuda.synchronize()
        grads.append(gr)
    assert torch.equal(grads[0].means, grads[1].means)
    got, by_opacity = (gr.opacity.double().cpu().numpy() for gr in grads)
    e = np.exp(-np.abs(x.astype(np.float64)))
    want = by_opacity * e / (1 + e) ** 2
    # exp as 2^(x log2 e): the product and its constant are each off by u, which x turns into 2 |x| u of the result, and one
    # step (2 u) of the hardware's exp2; then four roundings of 1 + e, the square and the quotient, and the product.  The
    # products at x = 80 (1.8e-35 times gradients down to 1e-12) leave fp32's normal numbers: there the last rounding is off
    # by half of their spacing 2^-149 whatever the value, which is 2^-150
    assert (np.abs(got - want) <= (2 * np.abs(x) + 8) * U * np.abs(want) + 2.0 ** -150).all()
    far = (x >= 17) & (np.abs(want) >= 2.0 ** -126)
    assert far.sum() > 100 and (got[far] != 0).all()
    c.close()


@pytest.mark.parametrize("n", [180, (1 << 19) + 90])
@pytest.mark.parametrize("is_logit", [False, True])
def test_dropout_gradient_of_gaussians_left_out_of_every_view(gpu_ctx, n, is_logit):
    """0 whatever the opacity is, as their opacities are in the forward pass; the others get the formula's value."""
    import torch
    import gsplat_amd as gs
    d = gpu_ctx.device
    some = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e30, -1e30, 0.0, -0.0, 200.0, -200.0], device=d)
    x = some.repeat((n + 8) // 9)[:n].contiguous()
    for views in ([4], [0, 1, 2], [3, 8, 13, 18], list(range(0, 5 * 40, 5)), []):       # 40 blocks: two launches
        p = .5 if len(views) < 10 else .97
        keep = gs.dropout_opacity(torch.ones_like(x), p, 7, views, ctx=gpu_ctx) != 0
        some_view = keep.any(dim=0) if views else torch.zeros(n, dtype=torch.bool, device=d)
        assert not views or 0 < int(some_view.sum()) < n
        got = gs.dropout_opacity_backward(torch.ones((len(views), n), device=d), x, p, 7, views, is_logit=is_logit, ctx=gpu_ctx)
        assert (got[~some_view] == 0).all()
        act = torch.ones(n, dtype=torch.float64, device=d)
        if is_logit:
            act = torch.where(x == 0, .25, 0.0).double()
            act[x.isnan()] = float("nan")
        want = (keep.sum(dim=0) * act / (1 - p))[some_view]
        # counts and 1/4 are exact: the scale's rounding and the product, per launch, and the launches' sum
        torch.testing.assert_close(got[some_view].double(), want, rtol=6 * U, atol=0, equal_nan=True)
        out = torch.full((n,), 2.0, device=d)
        gs.dropout_opacity_backward(torch.ones((len(views), n), device=d), x, p, 7, views, is_logit=is_logit, ctx=gpu_ctx,
                                    out=out, accumulate=True)
        assert (out[~some_view] == 2).all()
