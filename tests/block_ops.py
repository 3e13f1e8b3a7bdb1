"""Plain numpy statements of layer norm, dropout, 8-bit rows and their product, and bounds on how far a correct float32 or
float64 computation may be from them. Used by the tests of both machines."""
import numpy as np

U = {"f4": 2.0 ** -24, "f8": 2.0 ** -53}     # half a step of the type: what one rounding is off, relative to the value
WIDE = {"f4": np.float64, "f8": np.longdouble}


def norm(x, gain, bias, eps):
    """(y, xh, rstd) in a wider type."""
    w = WIDE[x.dtype.str[1:]]
    x, gain, bias = x.astype(w), gain.astype(w), bias.astype(w)
    d = x - x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + w(eps))
    return d * rstd * gain + bias, d * rstd, rstd


def norm_gradients(x, gain, gy, eps):
    w = WIDE[x.dtype.str[1:]]
    _y, xh, rstd = norm(x, gain, gain, eps)
    g = gy.astype(w)
    d = g * gain.astype(w)
    dx = rstd * (d - d.mean(1, keepdims=True) - xh * (d * xh).mean(1, keepdims=True))
    return dx, (g * xh).sum(0), g.sum(0)


def norm_bounds(x, gain, bias, gy, eps):
    """Bounds on the errors of y, dx, dgain, dbias. Any order of n additions is off by at most n * u * sum |terms|, so the mean
    by C u mean|x|; what follows is first-order propagation through the formulas, doubled for the terms of second order."""
    u = U[x.dtype.str[1:]]
    (R, C) = x.shape
    X = np.abs(x.astype("f8"))
    d = (x - x.astype(WIDE[x.dtype.str[1:]]).mean(1, keepdims=True)).astype("f8")
    v = (d * d).mean(1, keepdims=True) + eps
    rstd = 1 / np.sqrt(v)
    e_mean = (C + 1) * u * X.mean(1, keepdims=True)
    e_d = e_mean + u * np.abs(d)
    # the sum of squares around a mean that is off by e grows by e^2 only: sum d is 0
    e_v = (C + 3) * u * v + e_mean ** 2 + 2 * u * v
    rel = 0.5 * e_v / v + 3 * u            # of rstd; the root, the division and the sum with epsilon round once each
    xh = np.abs(d) * rstd
    e_xh = rstd * e_d + xh * (rel + u)
    g = np.abs(gain.astype("f8"))
    e_y = g * (e_xh + u * xh) + u * (xh * g + np.abs(bias.astype("f8"))) + u * g * xh
    if gy is None:
        return 2 * e_y
    G = np.abs(gy.astype("f8"))
    D = G * g
    s1, s2 = D.mean(1, keepdims=True), (D * xh).mean(1, keepdims=True)
    e_s1 = (C + 2) * u * s1
    e_s2 = (C + 3) * u * s2 + (D * e_xh).mean(1, keepdims=True)
    e_dx = rstd * (3 * u * D + e_s1 + xh * e_s2 + e_xh * s2 + 3 * u * (s1 + xh * s2)) + rstd * (D + s1 + xh * s2) * (rel + 2 * u)
    return 2 * e_y, 2 * e_dx, 2 * ((G * e_xh).sum(0) + (R + 2) * u * (G * xh).sum(0)), 2 * (R + 1) * u * G.sum(0)


def philox(blocks, step, site, seed):
    """[len(blocks), 4] words of the Philox4x32-10 blocks with counter (block, block >> 32, step, site)."""
    m, low, half = (np.uint64(0xD2511F53), np.uint64(0xCD9E8D57)), np.uint64(0xFFFFFFFF), np.uint64(32)
    b = np.asarray(blocks).astype(np.uint64)
    c = [b & low, b >> half, np.full_like(b, step & 0xFFFFFFFF), np.full_like(b, site)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p, q = c[0] * m[0], c[2] * m[1]
        c = [(q >> half) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> half) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1)


def kept(n, p, seed, step, site):
    words = philox(np.arange(-(-n // 4)), step, site, seed).reshape(-1)[:n]
    return words >= np.uint64(min(int(round(p * 2.0 ** 32)), 2 ** 32 - 1))


def dropout(x, p, seed, step, site):
    keep = kept(x.size, p, seed, step, site).reshape(x.shape)
    return np.where(keep, x * x.dtype.type(1 / (1 - p)), x.dtype.type(0))


def quantize(x):
    """Row by row, with whole numbers: the code k is the one for which |127 x - k a| is least, even where two are."""
    codes = np.zeros((x.shape[0], -(-x.shape[1] // 16) * 16), "i1")
    scales = np.zeros(x.shape[0], "f4")
    for r in range(x.shape[0]):
        a = np.abs(x[r]).max() if x.shape[1] else np.float32(0)
        scales[r] = a / np.float32(127) if np.isfinite(a) else np.nan
        if np.isfinite(a) and a > 0:
            q = 127 * x[r].astype(np.longdouble) / np.longdouble(a)   # 64 bits of mantissa: no tie is made or lost
            codes[r, :x.shape[1]] = np.rint(q)
    return codes, scales


def product(a, sa, b, sb, bias):
    """(result in 64 bits, bound): the sum is exact, then it, the two products and the sum with the bias round once each."""
    s = a.astype("i8") @ b.astype("i8").T
    p = s * sa.astype("f8")[:, None] * sb.astype("f8")
    y = p if bias is None else p + bias.astype("f8")
    u = U["f4"]
    # products of scales that leave the normal numbers lose up to a step of 2^-149
    return y, 3.1 * u * np.abs(p) + (0 if bias is None else u * np.abs(y)) + 2.0 ** -148
