"""Plain float64 forms of the 8-bit operators and the error bounds their
kernels are held to."""
import numpy as np

import block_reference as block

U = block.U
BLOCK = 128
MOST = {"e4m3": 448.0, "e5m2": 57344.0}
LEAST = 2.0 ** -100
# Half a step of each type relative to a value, and half of its smallest subnormal.
HALF8 = {"e4m3": (2.0 ** -4, 2.0 ** -10), "e5m2": (2.0 ** -3, 2.0 ** -17)}


def blocks(n):
    return -(-n // BLOCK)


def scales(v, dtype, block_rows=1):
    """Scales of |v|'s blocks in float64, [column blocks, rows or row blocks]. NaNs are passed over."""
    rows, cols = v.shape
    tall = rows if block_rows == 1 else blocks(rows) * BLOCK
    a = np.zeros((tall, blocks(cols) * BLOCK))
    a[:rows, :cols] = np.where(np.isnan(v), 0.0, np.abs(v))
    a = a.reshape(tall // block_rows, block_rows, -1, BLOCK).max((1, 3))
    return np.maximum(a, LEAST).T / MOST[dtype]


def spread(scale, rows, cols, block_rows=1):
    """The scale of every element, [rows, cols]."""
    s = np.repeat(scale.T, BLOCK, 1)[:, :cols]
    return s if block_rows == 1 else np.repeat(s, BLOCK, 0)[:rows]


def rounding8(v, dtype):
    """Half a step of an 8-bit type at v."""
    rel, least = HALF8[dtype]
    return np.maximum(np.abs(v) * rel, least)


def quantised_bound(v, off, dtype):
    """How far a block's values may be from v (in units of the scale) that is known to `off`: the scale's inverse and
    the product are rounded once each, then the one rounding to 8 bits."""
    e = off + 2 * U * (np.abs(v) + off)
    return e + rounding8(np.abs(v) + e, dtype)


def rms(h, w, eps):
    rstd = 1 / np.sqrt((h * h).mean(1) + eps)
    y = h * rstd[:, None]
    return (y * w if w is not None else y), rstd


# The sum of squares carries block.K roundings of positive terms, the mean, eps
# and the root and its inverse a few more; y two products.
RMS_REL = (block.K + 8) * U


def rms_grad(dy, h, w, rstd):
    xh = h * rstd[:, None]
    g = dy * w if w is not None else dy
    return rstd[:, None] * (g - xh * (g * xh).mean(1, keepdims=True)), (dy * xh).sum(0)


def rms_grad_bounds(dy, h, w, rstd, dres, dtype, extra=0.0):
    """As block.norm_grad_bounds without the terms of the mean."""
    xh = np.abs(h * rstd[:, None])
    g = np.abs(dy * w if w is not None else dy)
    m2 = (g * xh).mean(1, keepdims=True)
    e = rstd[:, None] * (6 * U * (g + xh * m2) + xh * (block.K + 8) * U * m2) + 2 * U * extra
    return e + block.rounding(np.abs(dres) + e, dtype), (block.KR + 8) * U * (np.abs(dy) * xh).sum(0)


def gemm(a, sa, b, sb, b_rows):
    """(product, sum of the terms' magnitudes) of 8-bit values and scales."""
    a = a * spread(sa, *a.shape)
    b = b * spread(sb, *b.shape, b_rows)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def gemm_bound(size, blocks_k, want, dtype):
    """fp32 C: a block's 128 products are exact in fp32 (two significands of 4 bits); their sum takes at most 128
    roundings or truncations of a step of 2^-23, the two scales two roundings, the sum over the blocks one each, up to
    32 more where it is split, and the sum with C one. 16-bit C: the 8-bit matrix instruction adds eight products at a
    time in units of 2^-13 of the largest one, so seven of them may lose up to that each."""
    e = (128 * 2 + 2 + blocks_k + 32 + 1) * U * size
    if dtype != "fp32":
        e = e + 7 * 2.0 ** -13 * size
    return e + block.rounding(np.abs(want) + e, dtype)
