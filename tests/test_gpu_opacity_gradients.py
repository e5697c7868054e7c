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
