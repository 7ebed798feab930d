"""The training-block operators at the edges of their ranges."""
import numpy as np
import pytest
import torch

import block_reference as ref
from test_gpu_block_ops import BOUNDARY_TYPES, NORM_TYPES, Matrix, eng, f64, ptr, vec, within  # noqa: F401


pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [6, 520])
@pytest.mark.parametrize("cols", [1, 3, 5, 8, 100, 768, 1000, 3001, 5001, 9001])
def test_gradient_of_large_constant_rows(eng, cols, rows):
    """Rows of one value near 1e33 with the rstd of eps 1e-12: mean * rstd passes fp32's range, x - mean is 0 in
    every column. The gradient is rstd (g - mean(g)) and nothing reaches it, or the sums, from past the row."""
    rng = np.random.default_rng(cols)
    n = eng.norm_backward_workspace(rows, cols)
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    w = vec(1 + 0.2 * rng.standard_normal(cols))
    p, seed, offset = 0.2, 8, 9
    cases = [(d, s, s, False) for s, d in NORM_TYPES if s != "fp16"]
    cases += [(d, s, x, True) for d, s, x in BOUNDARY_TYPES if s != "fp16"]
    for dt, st, dxt, boundary in cases:
        v = torch.full((rows, cols), 1e33)
        v[1::2] *= -0.7
        h, dy = Matrix(rows, cols, st, v), Matrix(rows, cols, dt, torch.from_numpy(rng.standard_normal((rows, cols))))
        # dres of about 1e6 * 1e-3: within fp16, which dx may be of.
        dy.view.mul_(2.0 ** -10)
        dres, dx = Matrix(rows, cols, st), Matrix(rows, cols, dxt)
        mean, rstd = h.view[:, 0].float().contiguous(), torch.full((rows,), 1e6, device="cuda")
        dw, db = torch.full((cols,), 0.5, device="cuda"), torch.full((cols,), 0.5, device="cuda")
        sums = (ptr(dw), ptr(db), False, ptr(work), n)
        if boundary:
            eng.dropout_add_norm_backward_device(dt, st, dxt, rows, cols, dy.at, cols, None, 0, h.at, cols, p, seed,
                                                 offset, ptr(w), ptr(mean), ptr(rstd), dres.at, cols, dx.at, cols, *sums)
        else:
            eng.layer_norm_backward_device(dt, st, rows, cols, dy.at, cols, h.at, cols, ptr(w), ptr(mean), ptr(rstd),
                                           dres.at, cols, *sums)
        args = dy.f64(), h.f64(), f64(w), f64(mean), f64(rstd)
        want, gw, gb = ref.norm_grad(*args)
        bound, ew, eb = ref.norm_grad_bounds(*args, want, st)
        what = (rows, cols, dt, st, dxt, boundary)
        within(dres.f64(), want, bound, what)
        if boundary:
            keep, scale = ref.keep_scale(rows, cols, p, seed, offset)
            e = ref.norm_grad_bounds(*args, want, "fp32")[0] * scale
            wanted = ref.drop(want, (keep, scale))
            e = e + 2 * ref.U * np.abs(wanted)
            within(dx.f64(), wanted, np.where(keep, e + ref.rounding(np.abs(wanted) + e, dxt), 0.0), ("dx", *what))
        assert not gw.any() and torch.equal(dw, torch.zeros_like(dw)), what
        within(db, gb, eb + ref.U * np.abs(gb), ("db", *what))
