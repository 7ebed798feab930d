"""Plain float64 forms of the training-block operators (LayerNorm, dropout, the
residual boundary) and the error bounds their fp32 kernels are held to."""
import numpy as np

U = 2.0 ** -24  # half a step of fp32, relative
# Half a step of each type relative to a value, and its smallest subnormal's half.
HALF = {"fp32": (2.0 ** -24, 2.0 ** -150), "bf16": (2.0 ** -8, 2.0 ** -134), "fp16": (2.0 ** -11, 2.0 ** -25)}
# Longest chain of fp32 additions in a row's sum: 128 are allowed for a thread's
# elements (kernels hold 16 to 24), a tree over 64 lanes (6) and up to 16 waves.
K = 160
# And in a column's sum over the rows: 128 for the rows of one thread and the
# waves of a workgroup in these tests' sizes, 512 for the partial sums (a
# thread adds at most 12 of the 768, and 16 more join the threads).
KR = 640


def philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 on uint64 arrays holding 32-bit words."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, np.uint64) for v in (c0, c1, c2, c3)]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def keep_scale(rows, cols, p, seed, offset):
    """([rows, cols] booleans, scale) of a mask. rows, cols: counts, or arrays of row and column numbers."""
    r = np.arange(rows) if np.isscalar(rows) else np.asarray(rows)
    c = np.arange(cols) if np.isscalar(cols) else np.asarray(cols)
    blocks, inverse = np.unique(c // 8, return_inverse=True)
    words = philox(blocks[None, :], r[:, None].astype(np.uint64), offset & 0xFFFFFFFF, offset >> 32,
                   seed & 0xFFFFFFFF, seed >> 32)
    words = np.stack(np.broadcast_arrays(*words), -1)  # [rows, blocks, 4]
    word = words[:, inverse, c % 8 // 2] if len(c) else np.zeros((len(r), 0), np.uint64)
    u16 = (word >> ((c % 2) * 16).astype(np.uint64)) & np.uint64(0xFFFF)
    t = int(np.rint(np.float64(np.float32(p)) * 65536))
    return u16 >= t, (65536 / (65536 - t) if t < 65536 else 0.0)


def drop(x, mask):
    keep, scale = mask
    return np.where(keep, np.where(keep, x, 0.0) * scale, 0.0)


def norm(x, w, b, eps):
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / np.sqrt((d * d).mean(1) + eps)
    y = d * rstd[:, None]
    y = y * w if w is not None else y
    return (y + b if b is not None else y), mean, rstd


def norm_grad(dy, x, w, mean, rstd):
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * w if w is not None else dy
    dx = rstd[:, None] * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def rounding(y, dtype):
    """Half a step of dtype at y: what one rounding may move it."""
    rel, least = HALF[dtype]
    return np.abs(y) * rel + least


def norm_bounds(x, w, b, eps, y, mean, rstd, dtype):
    """How far y, mean and rstd may be off: the row's mean carries K roundings
    of its terms, each difference one more, rstd half of the variance's K and
    its own few; y the products' and sum's and its own rounding."""
    size = np.abs(x).mean(1, keepdims=True)
    aw = 1.0 if w is None else np.abs(w)
    ab = 0.0 if b is None else np.abs(b)
    xh = (x - mean[:, None]) * rstd[:, None]
    e_mean = K * U * size
    e_rstd = (K + 8) * U + (e_mean[:, 0] * rstd) ** 2
    e_y = aw * (rstd[:, None] * (e_mean + 2 * U * np.abs(x)) + np.abs(xh) * e_rstd[:, None])
    e_y = e_y + 4 * U * (np.abs(y) + ab)
    return e_y + rounding(np.abs(y) + e_y, dtype), e_mean[:, 0] + U * np.abs(mean), rstd * e_rstd


def norm_grad_bounds(dy, x, w, mean, rstd, dx, dtype, extra=0.0):
    """extra: what else is added to dx before it is rounded (|dh|)."""
    xh = np.abs((x - mean[:, None]) * rstd[:, None])
    g = np.abs(dy * w if w is not None else dy)
    m1, m2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    e = rstd[:, None] * (6 * U * (g + m1 + xh * m2) + K * U * m1 + xh * (K + 8) * U * m2) + 2 * U * extra
    ady = np.abs(dy)
    return e + rounding(np.abs(dx) + e, dtype), (KR + 8) * U * (ady * xh).sum(0), KR * U * ady.sum(0)
