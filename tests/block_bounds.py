"""How far LayerNorm's kernels may be off for rows far from zero: what two
passes give, a mean and then the differences' own sum, which takes the mean's
rounding out of y, the stored mean and the variance."""
import numpy as np

from block_reference import U, rounding

# Longest chain of additions in a row's sum: 24 columns of a thread (16 in most
# shapes), six steps over the lanes, four over the waves.
K = 34


def two_pass_bounds(x, w, b, eps, y, mean, rstd, dtype):
    """Errors of (y, mean, rstd) of float64 rows x whose float64 results those are. m1, the first pass's mean, is
    off by e1; the differences d = x - m1 are rounded once each (exact where x is within a factor of two of m1), and
    their mean, which corrects m1, carries K + 4 roundings of |d|, not of |x|."""
    aw = 1.0 if w is None else np.abs(w)
    ab = 0.0 if b is None else np.abs(b)
    centred = x - mean[:, None]
    e1 = (K + 2) * U * np.abs(x).mean(1)
    d = np.abs(centred) + e1[:, None]
    e_m = (K + 4) * U * d.mean(1)
    var, square = (centred * centred).mean(1), (d * d).mean(1)
    e_var = (K + 6) * U * square + 2 * e1 * e_m
    e_rstd = e_var / (var + eps) / 2 + 4 * U
    xh = np.abs(centred) * rstd[:, None]
    e_y = aw * (rstd[:, None] * (e_m[:, None] + U * d + U * e1[:, None]) + xh * (e_rstd[:, None] + 2 * U))
    e_y = e_y + 2 * U * (np.abs(y) + ab)
    return e_y + rounding(np.abs(y) + e_y, dtype), e_m + U * np.abs(mean), rstd * e_rstd


def far_rows(rng, cols):
    """Rows of a spread of 1 or less around values up to 100,000 times it, and constant ones."""
    rows = [m + s * rng.standard_normal(cols) for m, s in ((1e3, 1.0), (1e4, 1.0), (1e5, 1.0), (-3e4, 0.5))]
    return np.float64(np.float32(rows + [np.full(cols, v) for v in (3.3, -7.1, 1e5 + 0.1)]))
