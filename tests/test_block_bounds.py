"""CPU checks of the bounds that LayerNorm's kernels are held to for rows far
from zero: fp32 arithmetic in the kernels' order stays within them, and the
same arithmetic with the correction of the mean left out does not."""
import numpy as np
import pytest

import block_reference as ref
from block_bounds import far_rows, two_pass_bounds

EPS = 1e-5
F = np.float32


def row_sum(v, lanes, vec):
    """fp32 sum of [rows, cols]: a lane's columns one after another, then the lanes' sums in a butterfly."""
    rows, cols = v.shape
    per = -(-cols // (lanes * vec))
    p = np.zeros((rows, per * lanes * vec), F)
    p[:, :cols] = v
    p = p.reshape(rows, per, lanes, vec).transpose(0, 2, 1, 3).reshape(rows, lanes, per * vec)
    s = np.zeros((rows, lanes), F)
    for i in range(p.shape[2]):
        s = s + p[:, :, i]
    while s.shape[1] > 1:
        s = s[:, 0::2] + s[:, 1::2]
    return s[:, 0]


def two_passes(x, lanes, vec, corrected=True, shift=0.0):
    """(y, mean, rstd) in fp32 as norm_kernel computes them; corrected: with the differences' own sum. shift: added
    to the first pass's mean."""
    x = F(x)
    inv = F(1) / F(x.shape[1])
    m1 = row_sum(x, lanes, vec) * inv + F(shift)
    d = x - m1[:, None]
    rest = row_sum(d, lanes, vec) * inv if corrected else np.zeros_like(m1)
    var = np.maximum(row_sum(d * d, lanes, vec) * inv - rest * rest, F(0))
    rstd = F(1) / np.sqrt(var + F(EPS))
    return d * rstd[:, None] - (rest * rstd)[:, None], m1 + rest, rstd


@pytest.mark.parametrize("cols,lanes,vec", [(100, 32, 4), (768, 64, 4), (1000, 64, 4), (4099, 512, 4), (8190, 512, 8)])
def test_the_correction_is_needed_and_enough(cols, lanes, vec):
    x = far_rows(np.random.default_rng(cols), cols)
    want = ref.norm(x, None, None, EPS)
    bounds = two_pass_bounds(x, None, None, EPS, *want, "fp32")

    def over(got):
        return [np.abs(np.float64(g) - w) > b for g, w, b in zip(got, want, bounds)]

    assert not any(o.any() for o in over(two_passes(x, lanes, vec)))
    # Without the correction y leaves its bound in several rows; with a mean that is off as well, in all of them.
    off = over(two_passes(x, lanes, vec, corrected=False))
    assert off[0].any(1).sum() >= 3, off[0].any(1)
    shifted = over(two_passes(x, lanes, vec, corrected=False, shift=8e-3))
    assert shifted[0].any(1).all() and shifted[1].sum() >= 3
