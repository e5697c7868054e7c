"""Measured cases of two families of operators on the parameters of a gaussian scene.

4-bit spherical harmonics.  A gaussian's 48 SH coefficients [3 channels][16] become a record of 32 bytes: the three
constant terms (k = 0) in half precision, and per channel the 15 others as E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and
a sign) that share one power-of-two scale.
    "quantize"    coefficients -> records -> the coefficients that the records stand for
    "color"       records times the SH basis in the directions of V cameras -> colours [V,N,3], and the flags of the
                  channels that were clamped at 0
    "color_grad"  gradients of that product: coefficients [N,3,16] and positions [N,3]

Opacity dropout.  Gaussian i is left out of view s with probability p, decided by a counter-based generator from
(seed, i, s); the opacities that stay are divided by 1 - p.  No mask is stored.
    "drop"        opacity logits [N] -> the opacities of V views [V,N]
    "drop_grad"   gradients of those [V,N] -> gradient of the logits [N]

`run` makes the package's calls where `own` is true and is the plain form, in elementary torch operations, where it is
false; `exact` evaluates the definitions in 64 bits."""
import math

import numpy as np
import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
CHUNK = 1 << 18          # gaussians that exact() takes at a time
MAX_N = 10_000_000


def listed():
    return [
        # a first look at a scene of 3 000 gaussians: bound by the latency of the launches
        {"name": "quantize_3k", "op": "quantize", "N": 3000},
        # a scene that has grown by densification (odd count), packed for a checkpoint and unpacked for editing
        {"name": "quantize_5m", "op": "quantize", "N": 5_000_001},
        # the 10 k-gaussian scene seen by one camera
        {"name": "color_10k_1view", "op": "color", "N": 10_000, "V": 1, "degree": 3},
        # the 8 views of a training step at 1 M gaussians
        {"name": "color_1m_8views", "op": "color", "N": 1_000_000, "V": 8, "degree": 3},
        # serving: one camera on the 10 M-gaussian scene
        {"name": "color_10m_1view", "op": "color", "N": 10_000_000, "V": 1, "degree": 3},
        # early training: few gaussians, the SH degree not yet raised to 3
        {"name": "color_grad_2501_2views", "op": "color_grad", "N": 2501, "V": 2, "degree": 1},
        # the backward pass of a training step at 1 M gaussians
        {"name": "color_grad_1m_8views", "op": "color_grad", "N": 1_000_000, "V": 8, "degree": 3},
        # the backward pass of a 4-view step on a scene of 3 M gaussians (odd count)
        {"name": "color_grad_3m_4views", "op": "color_grad", "N": 3_000_001, "V": 4, "degree": 3},
        # dropout for one view of the 10 k-gaussian scene
        {"name": "drop_10k_1view", "op": "drop", "N": 10_000, "V": 1, "p": 0.2},
        # dropout for the 8 views of a training step at 1 M gaussians
        {"name": "drop_1m_8views", "op": "drop", "N": 1_000_000, "V": 8, "p": 0.1},
        # its gradient in a small step (odd count)
        {"name": "drop_grad_10k_8views", "op": "drop_grad", "N": 10_001, "V": 8, "p": 0.1},
        # its gradient in a 4-view step on the 10 M-gaussian scene
        {"name": "drop_grad_10m_4views", "op": "drop_grad", "N": 10_000_000, "V": 4, "p": 0.05},
    ]


def draw(rng):
    op = rng.choice(["quantize", "color", "color_grad", "drop", "drop_grad"])
    V = 1 if op == "quantize" else rng.randint(1, 12)
    # the largest listed case of each operator bounds the drawn ones
    most = {"quantize": 5_000_001, "color": 10_000_000, "color_grad": 3_000_001, "drop": 8_000_000,
            "drop_grad": MAX_N}[op]
    if op != "quantize":
        most = min(most, {"color": 10_000_000, "color_grad": 12_000_004, "drop": 8_000_000,
                          "drop_grad": 40_000_000}[op] // V)
    N = max(1, int(math.exp(rng.uniform(0.0, math.log(most)))))
    case = {"op": op, "N": N}
    if op != "quantize":
        case["V"] = V
    if op in ("color", "color_grad"):
        case["degree"] = rng.randint(0, 3)
    if op in ("drop", "drop_grad"):
        case["p"] = rng.choice([0.0, 0.05, 0.1, 0.2, 0.5, 0.9])
    return case


def work(case):
    N, V = case["N"], case.get("V", 1)
    op = case["op"]
    if op == "quantize":                     # coefficients in, coefficients out
        return {"bytes": N * (192 + 192), "flops": N * 45 * 3}
    if op == "color":                        # record, position; colour and flags per view
        return {"bytes": N * (32 + 12) + V * N * (12 + 3), "flops": V * N * (2 * 48 + 60)}
    if op == "color_grad":                   # record, position, colour gradients and flags; two gradients
        return {"bytes": N * (32 + 12) + V * N * (12 + 3) + N * (192 + 12), "flops": V * N * (2 * 48 * 2 + 2 * 45 + 120)}
    if op == "drop":
        return {"bytes": N * 4 + V * N * 4, "flops": N * 10 + V * N * 2}
    return {"bytes": N * 4 + V * N * 4 + N * 4, "flops": N * 12 + V * N * 2}


# ------------------------------------------------------------------------------------------------- inputs
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _coefficients(N, gen, dev):
    """Constant terms of colours in 0..1; the others of a magnitude that differs from gaussian to gaussian and falls
    with the degree; one gaussian in twenty still has none (as point-cloud initialisation leaves them)."""
    sh = torch.randn((N, 3, 16), generator=gen, device=dev)
    sh[:, :, 0] = (torch.rand((N, 3), generator=gen, device=dev) - 0.5) / 0.28209479177387814
    size = 0.15 * torch.exp(0.7 * torch.randn((N, 1, 1), generator=gen, device=dev))
    size *= (torch.rand((N, 1, 1), generator=gen, device=dev) >= 0.05)
    band = torch.tensor([1.0] * 3 + [0.6] * 5 + [0.35] * 7, device=dev)
    sh[:, :, 1:] *= size * band
    return sh


def _cameras(V, rng):
    """Camera positions around the origin, in front of the scene."""
    return rng.uniform(-1.0, 1.0, (V, 3))


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    N, V, op = case["N"], case.get("V", 1), case["op"]
    state = {"op": op}
    if own:
        import gsplat_amd
        state["gs"] = gsplat_amd
    if op == "quantize":
        state["sh"] = _coefficients(N, gen, dev)
        return state
    if op in ("color", "color_grad"):
        # a scene is packed once (_pack) and then kept; positions as in the benchmark's scene
        words = _pack(_coefficients(N, gen, dev))
        z = 3.0 + 27.0 * torch.rand(N, generator=gen, device=dev)
        xy = (2.0 * torch.rand((N, 2), generator=gen, device=dev) - 1.0) * z[:, None] * torch.tensor([0.87, 0.49], device=dev)
        state.update(words=words, means=torch.cat([xy, z[:, None]], dim=1).contiguous(), cameras=_cameras(V, rng),
                     degree=case["degree"])
        if own:
            state["packed"] = state["gs"].PackedSH(words)
        if op == "color_grad":
            state["d_colors"] = torch.randn((V, N, 3), generator=gen, device=dev) * 1e-3
            state["clamped"] = (torch.rand((V, N, 3), generator=gen, device=dev) < 0.1).to(torch.uint8)
        return state
    state["opacity"] = 1.5 * torch.randn(N, generator=gen, device=dev)
    state["p"], state["seed"] = case["p"], int(rng.integers(0, 2 ** 63))
    state["views"] = [8 * int(rng.integers(0, 2 ** 33)) + v for v in range(V)]      # view numbers of a running training
    if op == "drop_grad":
        state["grad"] = torch.randn((V, N), generator=gen, device=dev) * 1e-3
    return state


def run(state):
    op = state["op"]
    if own:
        gs = state["gs"]
        if op == "quantize":
            return gs.quantize_sh(state["sh"]).dequantize()
        if op == "color":
            return gs.sh_color(state["packed"], state["means"], state["cameras"], degree=state["degree"])
        if op == "color_grad":
            return gs.sh_color_backward(state["packed"], state["means"], state["cameras"], state["clamped"],
                                        state["d_colors"], degree=state["degree"])
        if op == "drop":
            return gs.dropout_opacity(state["opacity"], state["p"], state["seed"], state["views"], is_logit=True)
        return gs.dropout_opacity_backward(state["grad"], state["opacity"], state["p"], state["seed"], state["views"],
                                           is_logit=True)
    if op == "quantize":
        return _quantize_plain(state["sh"])
    if op == "color":
        return _color_plain(state["words"], state["means"], state["cameras"], state["degree"])
    if op == "color_grad":
        return _color_grad_plain(state["words"], state["means"], state["cameras"], state["clamped"], state["d_colors"],
                                 state["degree"])
    if op == "drop":
        return _drop_plain(state["opacity"], state["p"], state["seed"], state["views"])
    return _drop_grad_plain(state["grad"], state["opacity"], state["p"], state["seed"], state["views"])


# ------------------------------------------------------------------------------------------------- plain forms
def _scale_bytes(ac):
    """E8M0 byte of the shared scale: exponent of the largest magnitude, rounded to one mantissa bit, minus 2."""
    amax = ac.abs().amax(dim=2)
    return (((amax.view(torch.int32) + 0x200000) >> 23) - 2).clamp(0, 252)


def _power_of_two(exponent_field):
    return (exponent_field << 23).to(torch.int32).view(torch.float32)


def _codes(ac, scale):
    """Magnitude code 0..7 of every coefficient, to nearest, ties to the even code."""
    x = ac.abs() * _power_of_two(254 - scale)[:, :, None]
    code = (x > 0.25).to(torch.int32)
    for threshold, inclusive in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (x >= threshold) if inclusive else (x > threshold)
    return code


def _values(code, negative, scale):
    table = torch.tensor(E2M1, dtype=torch.float32, device=code.device)
    # 2^(scale - 127) in two factors, so that neither is a denormal number
    half = scale >> 1
    mag = table[code.long()] * _power_of_two(half + 64)[:, :, None] * _power_of_two(scale - half + 63)[:, :, None]
    return torch.where(negative, -mag, mag)


def _quantize_plain(sh):
    dc, ac = sh[:, :, :1], sh[:, :, 1:]
    scale = _scale_bytes(ac)
    return torch.cat([dc.clamp(-65504.0, 65504.0).half().float(), _values(_codes(ac, scale), ac < 0, scale)], dim=2)


def _pack(sh):
    """Records [N,8] int32 (four 64-bit words, low half first): word 0 holds the three half-precision constants and
    two scales, words 1..3 the 15 codes of a channel; the third scale is in the top four bits of words 1 and 2."""
    dc, ac = sh[:, :, 0], sh[:, :, 1:]
    scale = _scale_bytes(ac)
    code = _codes(ac, scale) | ((ac < 0).to(torch.int32) << 3)
    bits = dc.half().view(torch.int16).to(torch.int64) & 0xffff
    s = scale.to(torch.int64)
    q = torch.zeros((sh.shape[0], 4), dtype=torch.int64, device=sh.device)
    q[:, 0] = bits[:, 0] | (bits[:, 1] << 16) | (bits[:, 2] << 32) | (s[:, 0] << 48) | (s[:, 1] << 56)
    for k in range(15):
        q[:, 1:] |= code[:, :, k].to(torch.int64) << (4 * k)
    q[:, 1] |= (s[:, 2] & 15) << 60
    q[:, 2] |= (s[:, 2] >> 4) << 60
    return q.view(torch.int32).contiguous()


def _unpack(words):
    q = words.view(torch.int64)
    dc = torch.stack([(q[:, 0] >> s) & 0xffff for s in (0, 16, 32)], dim=1).to(torch.int16).view(torch.float16).float()
    scale = torch.stack([(q[:, 0] >> 48) & 255, (q[:, 0] >> 56) & 255,
                         ((q[:, 1] >> 60) & 15) | (((q[:, 2] >> 60) & 15) << 4)], dim=1).to(torch.int32)
    code = torch.stack([(q[:, 1:] >> (4 * k)) & 15 for k in range(15)], dim=2).to(torch.int32)
    return torch.cat([dc[:, :, None], _values(code & 7, code >= 8, scale)], dim=2)


def _basis(d, degree):
    x, y, z = d.unbind(dim=1)
    b = [torch.full_like(x, 0.28209479177387814)]
    if degree > 0:
        b += [-0.4886025119029199 * y, 0.4886025119029199 * z, -0.4886025119029199 * x]
    if degree > 1:
        b += [1.0925484305920792 * x * y, -1.0925484305920792 * y * z, 0.31539156525252005 * (2 * z * z - x * x - y * y),
              -1.0925484305920792 * x * z, 0.5462742152960396 * (x * x - y * y)]
    if degree > 2:
        b += [-0.5900435899266435 * y * (3 * x * x - y * y), 2.890611442640554 * x * y * z,
              -0.4570457994644658 * y * (4 * z * z - x * x - y * y),
              0.3731763325901154 * z * (2 * z * z - 3 * x * x - 3 * y * y),
              -0.4570457994644658 * x * (4 * z * z - x * x - y * y), 1.445305721320277 * z * (x * x - y * y),
              -0.5900435899266435 * x * (x * x - 3 * y * y)]
    return torch.stack(b, dim=1)


def _basis_grad(d, degree):
    """Partial derivatives of the basis polynomials, [N,3,(degree+1)^2]."""
    x, y, z = d.unbind(dim=1)
    o = torch.zeros_like(x)
    gx, gy, gz = [o], [o], [o]
    if degree > 0:
        c = torch.full_like(x, 0.4886025119029199)
        gx += [o, o, -c]
        gy += [-c, o, o]
        gz += [o, c, o]
    if degree > 1:
        a, b, c = 1.0925484305920792, 0.31539156525252005, 0.5462742152960396
        gx += [a * y, o, -2 * b * x, -a * z, 2 * c * x]
        gy += [a * x, -a * z, -2 * b * y, o, -2 * c * y]
        gz += [o, -a * y, 4 * b * z, -a * x, o]
    if degree > 2:
        a, b, c, e, f = -0.5900435899266435, 2.890611442640554, -0.4570457994644658, 0.3731763325901154, 1.445305721320277
        xx, yy, zz = x * x, y * y, z * z
        gx += [6 * a * x * y, b * y * z, -2 * c * x * y, -6 * e * x * z, c * (4 * zz - 3 * xx - yy), 2 * f * x * z,
               3 * a * (xx - yy)]
        gy += [3 * a * (xx - yy), b * x * z, c * (4 * zz - xx - 3 * yy), -6 * e * y * z, -2 * c * x * y, -2 * f * y * z,
               -6 * a * x * y]
        gz += [o, b * x * y, 8 * c * y * z, 3 * e * (2 * zz - xx - yy), 8 * c * x * z, f * (xx - yy), o]
    return torch.stack([torch.stack(g, dim=1) for g in (gx, gy, gz)], dim=1)


def _direction(means, camera):
    """Unit vectors from the camera to the gaussians, in 64 bits: the positions may be far off and nearly equal."""
    v = means.double() - torch.tensor(camera, dtype=torch.float64, device=means.device)
    n = (v * v).sum(dim=1, keepdim=True).sqrt()
    return v / n, n


def _color_plain(words, means, cameras, degree):
    coef = _unpack(words)[:, :, :(degree + 1) ** 2].double()
    colors = torch.empty((len(cameras),) + tuple(means.shape), dtype=torch.float32, device=means.device)
    clamped = torch.empty(colors.shape, dtype=torch.uint8, device=means.device)
    for v, camera in enumerate(cameras):
        # in 64 bits: the flag is the sign of the sum
        r = (coef * _basis(_direction(means, camera)[0], degree)[:, None, :]).sum(dim=2) + 0.5
        clamped[v] = r < 0
        colors[v] = r.clamp(min=0.0)
    return colors, clamped


def _color_grad_plain(words, means, cameras, clamped, d_colors, degree):
    nb = (degree + 1) ** 2
    coef = _unpack(words)[:, :, :nb]
    d_sh = torch.zeros((means.shape[0], 3, 16), dtype=torch.float32, device=means.device)
    d_means = torch.zeros(means.shape, dtype=torch.float64, device=means.device)
    for v, camera in enumerate(cameras):
        d, n = _direction(means, camera)
        g = torch.where(clamped[v] != 0, torch.zeros_like(d_colors[v]), d_colors[v])
        d32 = d.float()
        d_sh[:, :, :nb] += g[:, :, None] * _basis(d32, degree)[:, None, :]
        w = (g[:, :, None] * coef).sum(dim=1)
        dd = (_basis_grad(d32, degree) * w[:, None, :]).sum(dim=2).double()
        d_means += (dd - d * (d * dd).sum(dim=1, keepdim=True)) / n
    return d_sh, d_means.float()


def _mul_hi_lo(a, b):
    """High and low halves of the product of 32-bit unsigned numbers held in int64 (b a constant)."""
    low = a * (b & 0xffff)
    high = a * (b >> 16) + (low >> 16)
    return high >> 16, ((high & 0xffff) << 16) | (low & 0xffff)


def _philox(index, block, seed):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw 2011) of the counter (index, 0, block) under the 64-bit key."""
    c = [index, torch.zeros_like(index), torch.full_like(index, block & 0xffffffff),
         torch.full_like(index, (block >> 32) & 0xffffffff)]
    k0, k1 = seed & 0xffffffff, (seed >> 32) & 0xffffffff
    for _ in range(10):
        h0, l0 = _mul_hi_lo(c[0], 0xD2511F53)
        h1, l1 = _mul_hi_lo(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    return c


def _kept(N, p, seed, views, device):
    """One mask [N] per view: word (view & 3) of the generator's block (view >> 2) is at least p 2^32."""
    index = torch.arange(N, dtype=torch.int64, device=device)
    limit = int(math.floor(p * 4294967296.0 + 0.5))
    block, words = None, None
    for view in views:
        if view >> 2 != block:
            block = view >> 2
            words = _philox(index, block, seed)
        yield words[view & 3] >= limit


def _drop_plain(opacity, p, seed, views):
    act = 1.0 / (1.0 + torch.exp(-opacity))
    act = act * (1.0 / (1.0 - p))
    return torch.stack([torch.where(keep, act, torch.zeros_like(act))
                        for keep in _kept(opacity.shape[0], p, seed, views, opacity.device)])


def _drop_grad_plain(grad, opacity, p, seed, views):
    total = torch.zeros_like(opacity)
    for v, keep in enumerate(_kept(opacity.shape[0], p, seed, views, opacity.device)):
        total += torch.where(keep, grad[v], torch.zeros_like(total))
    act = 1.0 / (1.0 + torch.exp(-opacity))
    return total * (act * (1.0 - act)) * (1.0 / (1.0 - p))


# ------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    op = state["op"]
    if op == "quantize":
        return torch.cat([_quantize_exact(part) for part in state["sh"].split(CHUNK)])
    if op == "color":
        parts = [_color_exact(w, m, state["cameras"], state["degree"])
                 for w, m in zip(state["words"].split(CHUNK), state["means"].split(CHUNK))]
        r = torch.cat(parts, dim=1)
        return r.clamp(min=0.0), (r < 0).to(torch.uint8)
    if op == "color_grad":
        parts = [_color_grad_exact(*part, state["cameras"], state["degree"]) for part in
                 zip(state["words"].split(CHUNK), state["means"].split(CHUNK), state["clamped"].split(CHUNK, dim=1),
                     state["d_colors"].split(CHUNK, dim=1))]
        return torch.cat([a for a, _ in parts]), torch.cat([b for _, b in parts])
    x = state["opacity"].double()
    act = torch.sigmoid(x)
    keep = _kept_exact(case["N"], state["p"], state["seed"], state["views"]).to(x.device)
    if op == "drop":
        return keep * (act / (1.0 - state["p"]))
    return (keep * state["grad"].double()).sum(dim=0) * act * torch.sigmoid(-x) / (1.0 - state["p"])


def _quantize_exact(sh):
    """Every coefficient to the nearest multiple of its spacing (half a power of two, at least half the scale)."""
    dc, ac = sh[:, :, :1], sh[:, :, 1:].double()
    m, e = torch.frexp(ac.abs().amax(dim=2, keepdim=True))        # amax = m 2^e, m in [.5, 1)
    e = torch.where(m >= 0.875, e + 1, e) - 1 - 2                   # amax rounds up to 2^e from seven eighths on
    e = torch.where(m == 0, torch.full_like(e, -127), e).clamp(-127, 125)
    x = ac.abs() * torch.pow(2.0, -e.double())
    step = torch.where(x < 2.0, 0.5, torch.where(x < 4.0, 1.0, 2.0)).double()
    q = (torch.round(x / step) * step).clamp(max=6.0) * torch.pow(2.0, e.double())
    return torch.cat([dc.half().double(), torch.copysign(q, ac)], dim=2)


def _coefficients_exact(words):
    """Coefficients from the records' bytes."""
    b = words.view(torch.uint8).reshape(-1, 32)
    dc = b[:, :6].contiguous().view(torch.float16).double()
    nib = torch.stack([b & 15, b >> 4], dim=2).reshape(-1, 64)[:, 16:].reshape(-1, 3, 16).long()
    scale = torch.stack([b[:, 6].double(), b[:, 7].double(), (nib[:, 0, 15] + 16 * nib[:, 1, 15]).double()], dim=1)
    code = nib[:, :, :15]
    exponent, mantissa = (code & 7) >> 1, (code & 1).double()
    mag = torch.where(exponent == 0, mantissa * 0.5, (1.0 + 0.5 * mantissa) * torch.pow(2.0, exponent.double() - 1.0))
    sign = 1.0 - 2.0 * (code >> 3).double()
    return torch.cat([dc[:, :, None], sign * mag * torch.pow(2.0, scale - 127.0)[:, :, None]], dim=2)


def _harmonics_exact(v, degree):
    """Real spherical harmonics with the Condon-Shortley phase in the direction of v, from the derivatives of the
    Legendre polynomials and the real and imaginary parts of (x + i y)^m."""
    x, y, z = (v / torch.linalg.vector_norm(v, dim=-1, keepdim=True)).unbind(dim=-1)
    one = torch.ones_like(z)
    legendre = {(0, 0): one, (1, 0): z, (1, 1): one, (2, 0): (3 * z ** 2 - 1) / 2, (2, 1): 3 * z, (2, 2): 3 * one,
                (3, 0): (5 * z ** 3 - 3 * z) / 2, (3, 1): (15 * z ** 2 - 3) / 2, (3, 2): 15 * z, (3, 3): 15 * one}
    re, im = [one], [torch.zeros_like(z)]
    for _ in range(3):
        re, im = re + [re[-1] * x - im[-1] * y], im + [re[-1] * y + im[-1] * x]
    out = []
    for l in range(degree + 1):
        for m in range(-l, l + 1):
            a = abs(m)
            norm = math.sqrt((2 * l + 1) / (4 * math.pi) * math.factorial(l - a) / math.factorial(l + a))
            norm *= (-1) ** a * (math.sqrt(2.0) if a else 1.0)
            out.append(norm * legendre[(l, a)] * (im[a] if m < 0 else re[a]))
    return torch.stack(out, dim=-1)


def _color_exact(words, means, cameras, degree):
    coef = _coefficients_exact(words)[:, :, :(degree + 1) ** 2]
    cam = torch.tensor(cameras, dtype=torch.float64, device=means.device)
    return torch.stack([(_harmonics_exact(means.double() - c, degree)[:, None, :] * coef).sum(dim=2) + 0.5 for c in cam])


def _color_grad_exact(words, means, clamped, d_colors, cameras, degree):
    nb = (degree + 1) ** 2
    coef = _coefficients_exact(words).requires_grad_()
    pos = means.double().requires_grad_()
    cam = torch.tensor(cameras, dtype=torch.float64, device=means.device)
    total = 0.0
    for v in range(len(cameras)):
        r = (_harmonics_exact(pos - cam[v], degree)[:, None, :] * coef[:, :, :nb]).sum(dim=2)
        total = total + (r * d_colors[v].double() * (clamped[v] == 0)).sum()
    total.backward()
    return coef.grad, torch.zeros_like(pos) if pos.grad is None else pos.grad


def _kept_exact(N, p, seed, views):
    """The masks [V,N] with the generator in unsigned 64-bit integers."""
    u, mask = np.uint64, np.uint64(0xffffffff)
    limit, out, blocks = u(int(math.floor(p * 4294967296.0 + 0.5))), [], {}
    for view in views:
        if view >> 2 not in blocks:
            b = view >> 2
            c = [np.arange(N, dtype=u), np.zeros(N, dtype=u), np.full(N, b & 0xffffffff, dtype=u),
                 np.full(N, b >> 32, dtype=u)]
            for r in range(10):
                k0 = u(((seed & 0xffffffff) + r * 0x9E3779B9) & 0xffffffff)
                k1 = u(((seed >> 32) + r * 0xBB67AE85) & 0xffffffff)
                a, e = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
                c = [(e >> u(32)) ^ c[1] ^ k0, e & mask, (a >> u(32)) ^ c[3] ^ k1, a & mask]
            blocks = {b: c}
        out.append(torch.from_numpy(blocks[view >> 2][view & 3] >= limit))
    return torch.stack(out)
