"""NumPy fp64 restatement of packed SH (records, colour, gradients) and opacity dropout, written from include/gsplat.h."""
import numpy as np

E2M1 = np.array([0., .5, 1., 1.5, 2., 3., 4., 6.])


def quantize(sh):
    """[N,3,16] -> records [N,8] uint32."""
    sh = np.asarray(sh, dtype=np.float32)
    n = len(sh)
    q = np.zeros((n, 4), dtype=np.uint64)
    with np.errstate(over="ignore", invalid="ignore"):
        dc = np.where(np.isfinite(sh[:, :, 0]), np.clip(sh[:, :, 0], -65504, 65504), sh[:, :, 0])
        half = dc.astype(np.float16).view(np.uint16).astype(np.uint64)
    for c in range(3):
        q[:, 0] |= half[:, c] << np.uint64(16 * c)
    scale = np.zeros((n, 3), dtype=np.int64)
    for i in range(n):
        for c in range(3):
            v = sh[i, c, 1:].astype(np.float64)
            if not np.all(np.isfinite(v)):
                scale[i, c] = 255
                continue
            amax = np.abs(v).max()
            if amax > 0:
                m, e = np.frexp(amax)                     # amax = m 2^e, .5 <= m < 1
                e = e - 1 + (1 if m >= 0.875 else 0)      # exponent after rounding to one mantissa bit (tie upwards)
                scale[i, c] = min(max(e - 2 + 127, 0), 252)
            s = 2.0 ** (int(scale[i, c]) - 127)
            for k in range(15):
                dist = np.abs(E2M1 - abs(v[k]) / s)
                best = np.flatnonzero(dist == dist.min())
                code = int(best[0] if len(best) == 1 or best[0] % 2 == 0 else best[1])      # ties: the even code
                code |= 8 if np.signbit(v[k]) else 0
                q[i, 1 + c] |= np.uint64(code << (4 * k))
    u = scale.astype(np.uint64)
    q[:, 0] |= u[:, 0] << np.uint64(48) | u[:, 1] << np.uint64(56)
    q[:, 1] |= (u[:, 2] & np.uint64(15)) << np.uint64(60)
    q[:, 2] |= (u[:, 2] >> np.uint64(4)) << np.uint64(60)
    return q.view(np.uint32).reshape(n, 8)


def dequantize(words):
    """records -> [N,3,16] float64."""
    q = np.ascontiguousarray(words).view(np.uint64).reshape(-1, 4)
    out = np.zeros((len(q), 3, 16))
    u = np.uint64
    for c in range(3):
        out[:, c, 0] = ((q[:, 0] >> u(16 * c)) & u(0xffff)).astype(np.uint16).view(np.float16)
        s = [(q[:, 0] >> u(48)) & u(255), q[:, 0] >> u(56), (q[:, 1] >> u(60)) | ((q[:, 2] >> u(60)) << u(4))][c]
        f = np.where(s == 255, np.nan, 2.0 ** (s.astype(np.float64) - 127))
        for k in range(15):
            code = ((q[:, 1 + c] >> u(4 * k)) & u(15)).astype(np.int64)
            out[:, c, 1 + k] = np.where(code >= 8, -1.0, 1.0) * E2M1[code & 7] * f
    return out


def basis(d, degree):
    """SH basis [N,16] at the unit directions d [N,3]; zero above `degree`."""
    x, y, z = d[:, 0], d[:, 1], d[:, 2]
    b = np.zeros((len(d), 16))
    b[:, 0] = 0.28209479177387814
    if degree > 0:
        b[:, 1], b[:, 2], b[:, 3] = -0.4886025119029199 * y, 0.4886025119029199 * z, -0.4886025119029199 * x
    if degree > 1:
        b[:, 4], b[:, 5] = 1.0925484305920792 * x * y, -1.0925484305920792 * y * z
        b[:, 6] = 0.31539156525252005 * (2 * z * z - x * x - y * y)
        b[:, 7], b[:, 8] = -1.0925484305920792 * x * z, 0.5462742152960396 * (x * x - y * y)
    if degree > 2:
        b[:, 9], b[:, 10] = -0.5900435899266435 * y * (3 * x * x - y * y), 2.890611442640554 * x * y * z
        b[:, 11] = -0.4570457994644658 * y * (4 * z * z - x * x - y * y)
        b[:, 12] = 0.3731763325901154 * z * (2 * z * z - 3 * x * x - 3 * y * y)
        b[:, 13] = -0.4570457994644658 * x * (4 * z * z - x * x - y * y)
        b[:, 14], b[:, 15] = 1.445305721320277 * z * (x * x - y * y), -0.5900435899266435 * x * (x * x - 3 * y * y)
    return b


def color(coef, means, cam_pos, degree):
    """(.5 + sum Y_k c_k) [V,N,3], not clamped."""
    out = []
    for p in np.asarray(cam_pos, dtype=np.float64).reshape(-1, 3):
        v = np.asarray(means, dtype=np.float64) - p
        b = basis(v / np.linalg.norm(v, axis=1, keepdims=True), degree)
        out.append(.5 + np.einsum("nk,nck->nc", b, coef))
    return np.array(out).reshape(-1, len(means), 3)


def philox(counter, key):
    """Philox4x32-10: four 32-bit words from four counter and two key words (Salmon et al. 2011)."""
    c, k = [int(v) for v in counter], [int(v) for v in key]
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


def keep_mask(n, p, seed, views):
    """[V,N] bool."""
    limit = int(np.floor(p * 4294967296.0 + .5))
    key = (seed & 0xffffffff, seed >> 32)
    return np.array([[philox((i, 0, (v >> 2) & 0xffffffff, v >> 34), key)[v & 3] >= limit for i in range(n)]
                     for v in views], dtype=bool).reshape(len(views), n)
