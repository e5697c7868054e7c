"""GPU: packed SH (records, colour, gradients) and opacity dropout against fp64 restatements.  u = 2^-24 is half a step of
fp32; every tolerance counts roundings of that size on sums of magnitudes."""
import numpy as np
import pytest

from conftest import synth_scene
from oracle import packed_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _sh(n, seed=0):
    rng = np.random.default_rng(seed)
    sh = rng.normal(size=(n, 3, 16)) * np.exp(rng.normal(0, 1, (n, 3, 1)))
    sh[:, :, 0] = rng.uniform(-1.8, 1.8, (n, 3))
    return sh.astype(np.float32)


def _means(n, seed=1):
    rng = np.random.default_rng(seed)
    return (rng.normal(size=(n, 3)) * [3, 3, 8] + [0, 0, 15]).astype(np.float32)


def _edge_sh():
    """Blocks whose rounding can go wrong: ties of every code, both signs, scale borders, denormals, the largest floats,
    zeros, infinities and NaN in every place."""
    blocks = []
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    near = [np.nextafter(np.float32(t), np.float32(d)) for t in ties for d in (0, 10)]
    for e in (-140, -127, -126, -30, 0, 60, 120, 124, 125):
        with np.errstate(over="ignore", under="ignore"):
            for vals in (ties + [4.0] * 8, near + [4.0], [6.0] + ties + near[:7], [7.0, 6.99, 5.5, -0.0] + ties + [1, 2, 3, 4],
                         [np.nextafter(np.float32(7), np.float32(0)), 6.5, 0.3] + ties + [0.1] * 5, [0.2] * 15, [-7.9] + [0.0] * 14):
                v = np.array(vals, dtype=np.float64) * 2.0 ** e
                v = np.clip(v, -np.finfo(np.float32).max, np.finfo(np.float32).max)
                blocks += [v, -v]
    f = np.finfo(np.float32)
    blocks += [np.full(15, f.max), np.full(15, f.tiny), np.full(15, 2.0 ** -149), np.zeros(15), np.full(15, -0.0),
               np.array([f.max] + [1e-30] * 14), np.array([2.0 ** -149] + [0] * 14)]
    for bad in (np.nan, np.inf, -np.inf):
        for k in (0, 7, 8, 14):
            v = np.linspace(-1, 1, 15)
            v[k] = bad
            blocks.append(v)
    while len(blocks) % 3:
        blocks.append(np.linspace(-3, 2, 15))
    sh = np.zeros((len(blocks) // 3, 3, 16), dtype=np.float32)
    sh[:, :, 1:] = np.array(blocks).reshape(-1, 3, 15)
    dc = [0, -0.0, 1e-8, 6e-8, 5.9e-5, 65504, 65519.9, 65520, 1e30, -1e30, np.inf, -np.inf, np.nan, 2049, 2051, 1 + 2 ** -11,
          1 + 3 * 2 ** -11, -0.3333333]
    sh[:, :, 0] = np.resize(np.array(dc, dtype=np.float32), sh.shape[:2])
    return sh


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 255, 256, 257, 1021])
def test_quantize_bit_for_bit(gpu_ctx, n):
    import torch
    import gsplat_amd as gs
    sh = _sh(n, n)
    packed = gs.quantize_sh(torch.from_numpy(sh).to(gpu_ctx.device), ctx=gpu_ctx)
    want = packed_ref.quantize(sh)
    np.testing.assert_array_equal(packed.numpy(), want)
    np.testing.assert_array_equal(packed.dequantize(gpu_ctx).cpu().numpy(), packed_ref.dequantize(want).astype(np.float32))


def test_quantize_edges_bit_for_bit(gpu_ctx):
    import gsplat_amd as gs
    sh = _edge_sh()
    got = gs.quantize_sh(sh, ctx=gpu_ctx).numpy()
    want = packed_ref.quantize(sh)
    # a NaN constant term is some half-precision NaN: compare that one by value
    g, w = (np.ascontiguousarray(a).view(np.uint16).reshape(len(sh), 16).copy() for a in (got, want))
    for c in range(3):
        gn, wn = (np.isnan(a[:, c].copy().view(np.float16)) for a in (g, w))
        np.testing.assert_array_equal(gn, wn)
        g[gn, c] = w[wn, c] = 0
    np.testing.assert_array_equal(g, w)
    # what the records stand for, through the device
    np.testing.assert_array_equal(gs.PackedSH(got, ctx=gpu_ctx).dequantize(gpu_ctx).cpu().numpy(),
                                  packed_ref.dequantize(got).astype(np.float32))


def test_dequantize_every_scale_and_code(gpu_ctx):
    """All 256 scale bytes (253 and 254 are never written but may be read) with all 16 codes."""
    import gsplat_amd as gs
    q = np.zeros((256, 4), dtype=np.uint64)
    s = np.arange(256, dtype=np.uint64)
    code = sum((k + 1) << (4 * k) for k in range(15))
    q[:, 0] = (s << np.uint64(48)) | (s[::-1] << np.uint64(56))
    q[:, 1] = np.uint64(code) | ((s & np.uint64(15)) << np.uint64(60))
    q[:, 2] = np.uint64(code >> 4) | ((s >> np.uint64(4)) << np.uint64(60))
    q[:, 3] = np.uint64(0x0123456789abcde)
    words = q.view(np.uint32).reshape(256, 8)
    got = gs.PackedSH(words, ctx=gpu_ctx).dequantize(gpu_ctx).cpu().numpy()
    with np.errstate(over="ignore"):
        want = packed_ref.dequantize(words).astype(np.float32)
    np.testing.assert_array_equal(got, want)


def test_quantize_inputs_that_are_not_plain_tensors(gpu_ctx):
    """NumPy float64, strided, misaligned and empty inputs."""
    import torch
    import gsplat_amd as gs
    sh = _sh(130, 5)
    want = packed_ref.quantize(sh)
    np.testing.assert_array_equal(gs.quantize_sh(sh.astype(np.float64), ctx=gpu_ctx).numpy(), want)
    t = torch.from_numpy(sh).to(gpu_ctx.device)
    strided = t.permute(0, 2, 1).contiguous().permute(0, 2, 1)
    np.testing.assert_array_equal(gs.quantize_sh(strided, ctx=gpu_ctx).numpy(), want)
    flat = torch.empty(130 * 48 + 1, device=gpu_ctx.device)
    flat[1:] = t.reshape(-1)
    np.testing.assert_array_equal(gs.quantize_sh(flat[1:].view(130, 3, 16), ctx=gpu_ctx).numpy(), want)
    empty = gs.quantize_sh(t[:0], ctx=gpu_ctx)
    assert len(empty) == 0 and empty.dequantize(gpu_ctx).shape == (0, 3, 16)
    part = gs.quantize_sh(t, ctx=gpu_ctx)[torch.arange(0, 130, 3, device=gpu_ctx.device)]
    np.testing.assert_array_equal(part.numpy(), want[::3])


def _exact_color(words, means, cams, degree):
    coef = packed_ref.dequantize(words)
    size = 3.0 * np.abs(coef).sum(axis=2).max()           # every |Y_k| evaluated term by term is below 3
    return packed_ref.color(coef, means, cams, degree), size


@pytest.mark.parametrize("degree", [0, 1, 2, 3])
@pytest.mark.parametrize("n,V", [(1, 1), (63, 2), (257, 1), (1000, 8), (130, 33)])
def test_color(gpu_ctx, n, V, degree):
    import torch
    import gsplat_amd as gs
    words, means = packed_ref.quantize(_sh(n, n + V)), _means(n)
    cams = np.random.default_rng(3).uniform(-1, 1, (V, 3))
    col, cl = gs.sh_color(gs.PackedSH(words, ctx=gpu_ctx), torch.from_numpy(means).to(gpu_ctx.device), cams, degree, ctx=gpu_ctx)
    assert col.shape == (V, n, 3) and cl.dtype == torch.uint8
    r, size = _exact_color(words, means, cams, degree)
    err = np.abs(col.cpu().numpy() - np.maximum(r, 0))
    assert (err <= U * np.abs(r) + 1e-14 * size).all()       # fp64 sums, one rounding to fp32
    sure = np.abs(r) > 1e-13 * size
    np.testing.assert_array_equal(cl.cpu().numpy()[sure], (r < 0)[sure])
    assert (r < 0).any() or n < 10


def test_color_matches_forward_pass(gpu_ctx):
    """On the dequantised coefficients, for every gaussian forward_pass does not cull: both round one fp64 sum of 16 terms
    to fp32, so they differ by that rounding at most, and rarely."""
    import torch
    import gsplat_amd as gs
    cam, R, t, g, rs = synth_scene(3000, 320, 240, seed=2, fx=200.0, log_scale=(2.0, 3.0))
    t = np.array([.3, -.2, .1])
    a = .2
    R = np.array([[np.cos(a), 0, np.sin(a)], [0, 1, 0], [-np.sin(a), 0, np.cos(a)]])
    packed = gs.quantize_sh(g.spherical_harmonics, ctx=gpu_ctx)
    g.spherical_harmonics = packed.dequantize(gpu_ctx)
    for name in ("center", "scaling", "rotation", "opacity"):
        setattr(g, name, torch.from_numpy(getattr(g, name)).to(gpu_ctx.device))
    _, _, colors, _, clamped, _, radii = gs.forward_pass(gpu_ctx, None, None, cam, R, t, g, result_size=rs)[:7]
    col, cl = gs.sh_color(packed, g.center, gs.camera_position(R, t), ctx=gpu_ctx)
    seen = radii > 0
    assert int(seen.sum()) > 1000
    a, b = col[0][seen].double(), colors[seen].double()
    assert ((a - b).abs() <= 2 * U * b.abs()).all() and int((a != b).sum()) <= 3
    assert torch.equal(cl[0][seen], clamped[seen])


def _exact_grad(words, means, cams, degree, cl, dc):
    """(d_sh, d_means) in fp64 by autograd, and the magnitudes their tolerances are counted on."""
    import torch
    coef = torch.from_numpy(packed_ref.dequantize(words)).requires_grad_()
    pos = torch.from_numpy(means.astype(np.float64)).requires_grad_()
    total = torch.zeros((), dtype=torch.float64)
    g = torch.from_numpy(np.where(cl != 0, 0.0, dc).astype(np.float64))
    dist = []
    for v, p in enumerate(cams):
        d = pos - torch.from_numpy(p)
        n = d.norm(dim=1, keepdim=True)
        dist.append(n.detach())
        x, y, z = (d / n).unbind(dim=1)
        b = [0.28209479177387814 + 0 * x, -0.4886025119029199 * y, 0.4886025119029199 * z, -0.4886025119029199 * x,
             1.0925484305920792 * x * y, -1.0925484305920792 * y * z, 0.31539156525252005 * (2 * z * z - x * x - y * y),
             -1.0925484305920792 * x * z, 0.5462742152960396 * (x * x - y * y),
             -0.5900435899266435 * y * (3 * x * x - y * y), 2.890611442640554 * x * y * z,
             -0.4570457994644658 * y * (4 * z * z - x * x - y * y), 0.3731763325901154 * z * (2 * z * z - 3 * x * x - 3 * y * y),
             -0.4570457994644658 * x * (4 * z * z - x * x - y * y), 1.445305721320277 * z * (x * x - y * y),
             -0.5900435899266435 * x * (x * x - 3 * y * y)][:(degree + 1) ** 2]
        r = (torch.stack(b, dim=1)[:, None, :] * coef[:, :, :len(b)]).sum(dim=2)
        total = total + (r * g[v]).sum()
    total.backward()
    dist = torch.stack(dist).numpy()[:, :, 0]
    ag, ac = np.abs(g.numpy()), np.abs(coef.detach().numpy())
    w = (ag[:, :, :, None] * ac[None]).sum(axis=(2, 3))                    # [V,N]
    return coef.grad.numpy(), pos.grad.numpy(), ag.sum(axis=0), (w / dist).sum(axis=0)


@pytest.mark.parametrize("degree", [0, 1, 2, 3])
@pytest.mark.parametrize("n,V", [(1, 1), (63, 2), (257, 1), (1000, 8), (130, 33)])
def test_color_backward(gpu_ctx, n, V, degree):
    import torch
    import gsplat_amd as gs
    rng = np.random.default_rng(n + degree)
    words, means = packed_ref.quantize(_sh(n, n)), _means(n)
    cams = rng.uniform(-1, 1, (V, 3))
    dc = rng.normal(size=(V, n, 3)).astype(np.float32)
    cl = (rng.uniform(size=(V, n, 3)) < .2).astype(np.uint8)
    dc[cl != 0] = np.nan                                    # never read into a sum
    d = gpu_ctx.device
    args = (gs.PackedSH(words, ctx=gpu_ctx), torch.from_numpy(means).to(d), cams, torch.from_numpy(cl).to(d),
            torch.from_numpy(dc).to(d), degree)
    d_sh, d_means = gs.sh_color_backward(*args, ctx=gpu_ctx)
    want_sh, want_means, g_sum, w_sum = _exact_grad(words, means, cams, degree, cl, np.nan_to_num(dc))
    # basis: at most 3 term by term, 10 roundings (three of the direction, its products, the polynomial); one per view's
    # addition, one more when a second launch adds to the first
    tol = 3 * (10 + V + 2) * U * g_sum[:, :, None]
    assert (np.abs(d_sh.cpu().numpy() - want_sh) <= tol).all()
    assert (d_sh.cpu().numpy()[:, :, (degree + 1) ** 2:] == 0).all()
    # each derivative: at most 12 term by term (2.89 x 3 and less), 16 + 3 + 10 roundings; the projection at most doubles;
    # two roundings of the result
    tol = 2 * 12 * 29 * U * w_sum[:, None] + 2 * U * np.abs(want_means)
    assert (np.abs(d_means.cpu().numpy() - want_means) <= tol).all()
    if degree == 0:
        assert (d_means == 0).all()
    # added to what is there
    out = (d_sh.clone(), d_means.clone())
    got = gs.sh_color_backward(*args, ctx=gpu_ctx, out=out, accumulate=True)
    assert got[0] is out[0]
    np.testing.assert_allclose(out[0].cpu().numpy(), 2 * d_sh.cpu().numpy(), rtol=4 * U, atol=3 * 2 * U * float(g_sum.max()))
    np.testing.assert_allclose(out[1].cpu().numpy(), 2 * d_means.cpu().numpy(), rtol=4 * U, atol=2 * U * float(w_sum.max()))


def test_color_gradients_against_differences(gpu_ctx):
    """The gradient of a position against central differences of the fp64 colour."""
    import torch
    import gsplat_amd as gs
    n = 40
    words, means = packed_ref.quantize(_sh(n, 9)), _means(n, 9)
    cams = np.array([[.1, .2, -.3], [-.5, 0, .4]])
    dc = np.random.default_rng(1).normal(size=(2, n, 3)).astype(np.float32)
    coef = packed_ref.dequantize(words)
    cl = (packed_ref.color(coef, means, cams, 3) < 0).astype(np.uint8)
    d = gpu_ctx.device
    _, got = gs.sh_color_backward(gs.PackedSH(words, ctx=gpu_ctx), torch.from_numpy(means).to(d), cams,
                                  torch.from_numpy(cl).to(d), torch.from_numpy(dc).to(d), ctx=gpu_ctx)
    h = 1e-4
    for k in range(3):
        step = np.zeros(3)
        step[k] = h
        f = lambda m: (np.where(cl != 0, 0, packed_ref.color(coef, m, cams, 3)) * dc).sum(axis=(0, 2))
        diff = (f(means + step) - f(means - step)) / (2 * h)
        # h^2 / 6 of third derivatives of size |c| |Y'''| / dist^3, and the fp32 gradient's own error
        np.testing.assert_allclose(got.cpu().numpy()[:, k], diff, rtol=1e-5, atol=2e-5)


def test_color_of_no_views_and_no_gaussians(gpu_ctx):
    import torch
    import gsplat_amd as gs
    d = gpu_ctx.device
    packed, means = gs.PackedSH(packed_ref.quantize(_sh(5)), ctx=gpu_ctx), torch.from_numpy(_means(5)).to(d)
    col, cl = gs.sh_color(packed, means, np.zeros((0, 3)), ctx=gpu_ctx)
    assert col.shape == (0, 5, 3) and cl.shape == (0, 5, 3)
    none = torch.zeros((0, 5, 3), device=d)
    d_sh, d_means = gs.sh_color_backward(packed, means, np.zeros((0, 3)), none, none, ctx=gpu_ctx)
    assert (d_sh == 0).all() and (d_means == 0).all()
    col, _ = gs.sh_color(packed[:0], means[:0], np.zeros((2, 3)), ctx=gpu_ctx)
    assert col.shape == (2, 0, 3)
    with pytest.raises(gs.GsError, match="degree"):
        gs.sh_color(packed, means, np.zeros((1, 3)), degree=4, ctx=gpu_ctx)


@pytest.mark.parametrize("is_logit", [False, True])
@pytest.mark.parametrize("n,views,p", [(1, [0], .5), (65, [3, 2, 1, 0], .3), (257, [7, 7, 2 ** 64 - 1, 2 ** 34 + 1], .1),
                                       (1001, [4, 5, 6, 7, 8], 0.0), (130, [5 * v for v in range(65)], .9)])
def test_dropout(gpu_ctx, n, views, p, is_logit):
    import torch
    import gsplat_amd as gs
    rng = np.random.default_rng(n)
    x = (rng.normal(size=n) * 4 if is_logit else rng.uniform(size=n)).astype(np.float32)
    seed = 0xfedcba9876543210
    keep = packed_ref.keep_mask(n, p, seed, views)
    x64 = x.astype(np.float64)
    o = 1 / (1 + np.exp(-x64)) if is_logit else x64
    xt = torch.from_numpy(x).to(gpu_ctx.device)
    got = gs.dropout_opacity(xt, p, seed, views, is_logit=is_logit, ctx=gpu_ctx).cpu().numpy()
    assert got.shape == (len(views), n)
    np.testing.assert_array_equal(got != 0, keep & (o > 0))
    # exp to one step, an addition, a division, the scale's rounding and the product
    np.testing.assert_allclose(got, np.where(keep, o / (1 - p), 0), rtol=6 * U, atol=0)
    g = rng.normal(size=(len(views), n)).astype(np.float32)
    g[~keep] = np.nan                                        # gradients of left-out gaussians stay out
    gt = torch.from_numpy(g).to(gpu_ctx.device)
    got = gs.dropout_opacity_backward(gt, xt, p, seed, views, is_logit=is_logit, ctx=gpu_ctx)
    s = np.where(keep, np.nan_to_num(g).astype(np.float64), 0)
    act = o * (1 - o) if is_logit else np.ones(n)
    want = s.sum(axis=0) * act / (1 - p)
    # the sum's roundings and the factors'; 1 - o is off by the rounding of o
    tol = np.abs(s).sum(axis=0) / (1 - p) * ((len(views) + 6) * U * act + (6 * U * o if is_logit else 0))
    assert (np.abs(got.cpu().numpy() - want) <= tol).all()
    twice = gs.dropout_opacity_backward(gt, xt, p, seed, views, is_logit=is_logit, ctx=gpu_ctx, out=got.clone(), accumulate=True)
    np.testing.assert_allclose(twice.cpu().numpy(), 2 * got.cpu().numpy(), rtol=2 * U, atol=(len(views) + 2) * U * np.abs(s).sum(axis=0).max() / (1 - p))


@pytest.mark.parametrize("n", [(1 << 19) - 1, 1 << 19, (1 << 19) + 1, (1 << 19) + 1022])
def test_dropout_with_four_gaussians_per_thread(gpu_ctx, n):
    """Around the size from which a thread takes four, whole and ragged last blocks: the same masks and sums as on parts."""
    import torch
    import gsplat_amd as gs
    d, views = gpu_ctx.device, [3, 2, 9, 9, 40]
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(d)
    out = gs.dropout_opacity(x, .4, 11, views, is_logit=True, ctx=gpu_ctx)
    small = gs.dropout_opacity(x[:1000], .4, 11, views, is_logit=True, ctx=gpu_ctx)
    assert torch.equal(out[:, :1000], small)
    for i in (n - 1, n - 2, n - 1023, n // 2):
        keep = [packed_ref.philox((i, 0, v >> 2, 0), (11, 0))[v & 3] >= int(np.floor(.4 * 2 ** 32 + .5)) for v in views]
        assert (out[:, i] != 0).tolist() == keep
    kept = out[out != 0]
    assert abs(kept.numel() / out.numel() - .6) < 6 * np.sqrt(.24 / (4 * n))             # four different views
    g = torch.randn((5, n), generator=torch.Generator().manual_seed(1)).to(d)
    got = gs.dropout_opacity_backward(g, x, .4, 11, views, is_logit=True, ctx=gpu_ctx)
    s = torch.sigmoid(x.double())
    want = (torch.where(out != 0, g, torch.zeros_like(g)).double().sum(dim=0) / .6) * s * (1 - s)
    tol = g.double().abs().sum(dim=0) / .6 * (11 * U * s * (1 - s) + 6 * U * s)
    assert ((got.double() - want).abs() <= tol).all()
    again = gs.dropout_opacity_backward(g, x, .4, 11, views, is_logit=True, ctx=gpu_ctx, out=got.clone(), accumulate=True)
    assert ((again.double() - 2 * got.double()).abs() <= 2 * U * got.double().abs() + tol).all()


def test_dropout_edges(gpu_ctx):
    import torch
    import gsplat_amd as gs
    d = gpu_ctx.device
    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e30, -1e30, 0.0, -0.0, 200.0, -200.0] * 20, device=d)
    views = list(range(9))
    keep = torch.from_numpy(packed_ref.keep_mask(len(x), .5, 7, views)).to(d)
    out = gs.dropout_opacity(x, .5, 7, views, ctx=gpu_ctx)
    assert (out[~keep] == 0).all()                           # whatever the opacity is
    want = (2 * x).expand(9, -1)
    assert torch.equal(torch.nan_to_num(out[keep], nan=5.0), torch.nan_to_num(want[keep], nan=5.0))
    logit = gs.dropout_opacity(x, 0.0, 7, [0], is_logit=True, ctx=gpu_ctx)[0]
    np.testing.assert_allclose(logit[1:9].cpu().numpy(), [1, 0, 1, 0, .5, .5, 1, 0], rtol=0, atol=2 * U)
    # [N,1] opacities, NumPy in and out, no gaussians, no views
    got = gs.dropout_opacity(np.full((6, 1), .25), .2, 3, [11], ctx=gpu_ctx)
    np.testing.assert_allclose(got, np.where(packed_ref.keep_mask(6, .2, 3, [11]), .3125, 0), rtol=4 * U)
    assert gs.dropout_opacity(x[:0], .2, 3, [1, 2], ctx=gpu_ctx).shape == (2, 0)
    assert gs.dropout_opacity(x, .2, 3, [], ctx=gpu_ctx).shape == (0, 180)
    none = gs.dropout_opacity_backward(torch.zeros((0, 180), device=d), x, .2, 3, [], ctx=gpu_ctx)
    assert (none == 0).all()
    for bad in (-.1, 1.0, 1 - 1e-11, float("nan")):
        with pytest.raises(gs.GsError, match=r"not in \[0, 1\)"):
            gs.dropout_opacity(x, bad, 3, [0], ctx=gpu_ctx)
        with pytest.raises(gs.GsError, match=r"not in \[0, 1\)"):
            gs.dropout_opacity_backward(out[:1], x, bad, 3, [0], ctx=gpu_ctx)


def test_captured_and_replayed(gpu_ctx):
    """All calls in one graph, replayed on new contents with eager work and synchronisation in between."""
    import torch
    import gsplat_amd as gs
    d, n, V = gpu_ctx.device, 700, 3
    cams = np.random.default_rng(0).uniform(-1, 1, (V, 3))
    sh, means, x = (torch.zeros(s, device=d) for s in ((n, 3, 16), (n, 3), (n,)))
    g, gc = torch.zeros((V, n), device=d), torch.zeros((V, n, 3), device=d)

    def fill(seed):
        gen = torch.Generator().manual_seed(seed)
        for t in (sh, means, x, g, gc):
            t.copy_(torch.randn(t.shape, generator=gen))
        means[:, 2] += 12

    def calls():
        packed = gs.quantize_sh(sh, ctx=gpu_ctx)
        col, cl = gs.sh_color(packed, means, cams, ctx=gpu_ctx)
        d_sh, d_means = gs.sh_color_backward(packed, means, cams, cl, gc, ctx=gpu_ctx)
        op = gs.dropout_opacity(x, .3, 5, range(V), is_logit=True, ctx=gpu_ctx)
        d_x = gs.dropout_opacity_backward(g, x, .3, 5, range(V), is_logit=True, ctx=gpu_ctx)
        return packed.words, packed.dequantize(gpu_ctx), col, cl, d_sh, d_means, op, d_x

    fill(0)
    side = torch.cuda.Stream(d)
    side.wait_stream(torch.cuda.current_stream(d))
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream(d).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for seed in (1, 2, 3):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize(d)
        want = calls()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_on_another_stream(gpu_ctx):
    """Launched on torch's current stream, behind that stream's own work."""
    import torch
    import gsplat_amd as gs
    d = gpu_ctx.device
    sh = torch.from_numpy(_sh(5000, 3)).to(d)
    want = packed_ref.quantize((_sh(5000, 3)[:200]))
    side = torch.cuda.Stream(d)
    side.wait_stream(torch.cuda.current_stream(d))
    with torch.cuda.stream(side):
        buf = torch.zeros_like(sh)
        for _ in range(20):
            buf = buf + 0 * sh                               # work in front of the copy on the same stream
        buf.copy_(sh)
        packed = gs.quantize_sh(buf, ctx=gpu_ctx)
    torch.cuda.current_stream(d).wait_stream(side)
    np.testing.assert_array_equal(packed.numpy()[:200], want)


def test_offsets_past_32_bits(gpu_ctx):
    """More than 4 GiB of coefficients, colours and opacities: the last rows are those of a call on them alone."""
    import torch
    import gsplat_amd as gs
    d, n, tail = gpu_ctx.device, 23_000_001, 777
    sh = torch.rand((n, 3, 16), device=d) - 0.5                       # 4.4 GB
    packed = gs.quantize_sh(sh, ctx=gpu_ctx)
    last = gs.quantize_sh(sh[-tail:], ctx=gpu_ctx)
    assert torch.equal(packed.words[-tail:], last.words)
    del sh
    dense = packed.dequantize(gpu_ctx)
    assert torch.equal(dense[-tail:], last.dequantize(gpu_ctx))
    del dense
    means = torch.rand((n, 3), device=d) + torch.tensor([0., 0., 5.], device=d)
    V = 17
    cams = np.random.default_rng(0).uniform(-1, 1, (V, 3))
    col, cl = gs.sh_color(packed, means, cams, ctx=gpu_ctx)           # 4.7 GB
    c1, f1 = gs.sh_color(last, means[-tail:], cams, ctx=gpu_ctx)
    assert torch.equal(col[:, -tail:], c1) and torch.equal(cl[:, -tail:], f1)
    d_sh, d_means = gs.sh_color_backward(packed, means, cams, cl, col, ctx=gpu_ctx)
    e_sh, e_means = gs.sh_color_backward(last, means[-tail:], cams, f1, c1, ctx=gpu_ctx)
    assert torch.equal(d_sh[-tail:], e_sh) and torch.equal(d_means[-tail:], e_means)
    del col, cl, d_sh
    x, views = torch.ones(n, device=d), list(range(100, 148))
    out = gs.dropout_opacity(x, .5, 9, views, ctx=gpu_ctx)             # 4.4 GB
    for i in (0, n // 2, n - 2, n - 1):
        keep = [packed_ref.philox((i, 0, v >> 2, 0), (9, 0))[v & 3] >= 2 ** 31 for v in views]
        assert (out[:, i] != 0).tolist() == keep
    back = gs.dropout_opacity_backward(out, x, .5, 9, views, ctx=gpu_ctx)
    assert float(back[-1]) == 4.0 * sum(keep) and float(back[0]) == 2.0 * float(out[:, 0].sum())


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_misaligned_inputs(gpu_ctx, offset):
    """Gradients, flags, positions and opacities that start at any float or byte."""
    import torch
    import gsplat_amd as gs
    d, n, V = gpu_ctx.device, 301, 3

    def shifted(t):
        flat = torch.zeros(t.numel() + offset, dtype=t.dtype, device=d)
        flat[offset:] = t.reshape(-1)
        return flat[offset:].view(t.shape)
    gen = torch.Generator().manual_seed(offset)
    packed = gs.quantize_sh(torch.randn((n, 3, 16), generator=gen).to(d), ctx=gpu_ctx)
    means = (torch.randn((n, 3), generator=gen) + torch.tensor([0., 0., 9.])).to(d)
    cams = np.random.default_rng(1).uniform(-1, 1, (2 * V, 3))[::2]                  # strided on the host
    col, cl = gs.sh_color(packed, means, cams, ctx=gpu_ctx)
    g = torch.randn((V, n, 3), generator=gen).to(d)
    want = gs.sh_color_backward(packed, means, cams, cl, g, ctx=gpu_ctx)
    got = gs.sh_color_backward(packed, shifted(means), cams, shifted(cl), shifted(g), ctx=gpu_ctx)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(gs.sh_color(packed, shifted(means), cams, ctx=gpu_ctx)[0], col)
    strided = g.permute(2, 1, 0).contiguous().permute(2, 1, 0)
    got = gs.sh_color_backward(packed, means, cams, cl, strided, ctx=gpu_ctx)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    part = gs.PackedSH(packed.words[1:])                                              # records from the second on
    assert torch.equal(gs.sh_color(part, means[1:], cams, ctx=gpu_ctx)[0], col[:, 1:])
    x, gx = torch.randn(n, generator=gen).to(d), torch.randn((V, n), generator=gen).to(d)
    assert torch.equal(gs.dropout_opacity(shifted(x), .3, 2, range(V), True, ctx=gpu_ctx),
                       gs.dropout_opacity(x, .3, 2, range(V), True, ctx=gpu_ctx))
    assert torch.equal(gs.dropout_opacity_backward(shifted(gx), shifted(x), .3, 2, range(V), True, ctx=gpu_ctx),
                       gs.dropout_opacity_backward(gx, x, .3, 2, range(V), True, ctx=gpu_ctx))


def test_numpy_in_numpy_out(gpu_ctx):
    import gsplat_amd as gs
    words, means = packed_ref.quantize(_sh(20)), _means(20).astype(np.float64)
    cam = np.array([.1, .2, .3])                                                       # one camera, [3]
    cam.setflags(write=False)
    col, cl = gs.sh_color(gs.PackedSH(words), means, cam, ctx=gpu_ctx)                 # records on the host
    assert col.dtype == np.float64 and cl.dtype == np.uint8 and col.shape == (1, 20, 3)
    want = packed_ref.color(packed_ref.dequantize(words), means.astype(np.float32), cam, 3)
    np.testing.assert_allclose(col, np.maximum(want, 0), rtol=2 * U, atol=1e-12)
    d_sh, d_means = gs.sh_color_backward(gs.PackedSH(words), means, cam, cl[0], np.ones((20, 3)), ctx=gpu_ctx)
    assert d_sh.shape == (20, 3, 16) and d_means.dtype == np.float64
    g = gs.dropout_opacity_backward(np.ones(20), np.full(20, .5), .25, 1, [6], ctx=gpu_ctx)
    np.testing.assert_allclose(g, np.where(packed_ref.keep_mask(20, .25, 1, [6])[0], 4 / 3, 0), rtol=4 * U)


def test_nothing_outside_the_outputs_is_written(gpu_ctx):
    """Guard words around every output buffer that the caller owns."""
    import torch
    import gsplat_amd as gs
    d, n, V = gpu_ctx.device, 131, 2
    packed = gs.quantize_sh(torch.from_numpy(_sh(n)).to(d), ctx=gpu_ctx)
    means = torch.from_numpy(_means(n)).to(d)
    cams = np.zeros((V, 3))

    def guarded(shape):
        k = int(np.prod(shape))
        buf = torch.full((k + 128,), 7.5, device=d)
        return buf, buf[64:64 + k].view(shape)
    b1, d_sh = guarded((n, 3, 16))
    b2, d_means = guarded((n, 3))
    b3, d_op = guarded((n,))
    col, cl = gs.sh_color(packed, means, cams, ctx=gpu_ctx)
    gs.sh_color_backward(packed, means, cams, cl, col, ctx=gpu_ctx, out=(d_sh, d_means))
    gs.dropout_opacity_backward(torch.ones((V, n), device=d), torch.ones(n, device=d), .1, 0, [0, 1], ctx=gpu_ctx, out=d_op)
    for b in (b1, b2, b3):
        assert (b[:64] == 7.5).all() and (b[-64:] == 7.5).all()
    want = gs.sh_color_backward(packed, means, cams, cl, col, ctx=gpu_ctx)
    assert torch.equal(d_sh, want[0]) and torch.equal(d_means, want[1])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float64"])
def test_other_float_types_are_taken_as_their_float32_values(gpu_ctx, dtype):
    import torch
    import gsplat_amd as gs
    d, t = gpu_ctx.device, getattr(torch, dtype)
    sh, means = torch.from_numpy(_sh(70)).to(d).to(t), torch.from_numpy(_means(70)).to(d).to(t)
    packed = gs.quantize_sh(sh, ctx=gpu_ctx)
    np.testing.assert_array_equal(packed.numpy(), packed_ref.quantize(sh.float().cpu().numpy()))
    cam = np.array([[.3, .2, .1]])
    col, cl = gs.sh_color(packed, means, cam, ctx=gpu_ctx)
    assert torch.equal(col, gs.sh_color(packed, means.float(), cam, ctx=gpu_ctx)[0])
    g = torch.randn((1, 70, 3), generator=torch.Generator().manual_seed(0)).to(d).to(t)
    a, b = (gs.sh_color_backward(packed, means.to(k), cam, cl.bool() if k is t else cl, g.to(k), ctx=gpu_ctx)
            for k in (t, torch.float32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    x = torch.randn(70, generator=torch.Generator().manual_seed(1)).to(d).to(t)
    assert torch.equal(gs.dropout_opacity(x, .2, 1, [5], True, ctx=gpu_ctx), gs.dropout_opacity(x.float(), .2, 1, [5], True, ctx=gpu_ctx))


def test_color_at_the_camera_and_far_away(gpu_ctx):
    """A gaussian at the camera has no direction; one 1e18 away has."""
    import torch
    import gsplat_amd as gs
    d = gpu_ctx.device
    packed = gs.quantize_sh(torch.from_numpy(_sh(3)).to(d), ctx=gpu_ctx)
    means = torch.tensor([[1., 2., 3.], [1e18, -2e18, 1e17], [1., 2., 3.0001]], device=d)
    cam = np.array([[1., 2., 3.]])
    col, cl = gs.sh_color(packed, means, cam, ctx=gpu_ctx)
    assert torch.isnan(col[0, 0]).all() and (cl[0, 0] == 0).all()
    want = packed_ref.color(packed_ref.dequantize(packed.numpy()[1:]), means.cpu().numpy()[1:], cam, 3)
    np.testing.assert_allclose(col[0, 1:].cpu().numpy(), np.maximum(want[0], 0), rtol=2 * U, atol=1e-12)
    _, d_means = gs.sh_color_backward(packed, means, cam, cl, torch.ones_like(col), ctx=gpu_ctx)
    assert torch.isnan(d_means[0]).all() and torch.isfinite(d_means[1:]).all() and float(d_means[1].abs().max()) < 1e-16
    assert torch.isfinite(gs.sh_color(packed, means, cam, degree=0, ctx=gpu_ctx)[0]).all()
