"""The training-block operators at the edges of their ranges: rows far from
zero against bounds that only a corrected mean keeps, rows whose padded columns
would leave fp32's range, the largest values the norms take, and dropout of
more elements than one launch takes."""
import numpy as np
import pytest
import torch

import block_reference as ref
from block_bounds import far_rows, two_pass_bounds
from test_gpu_block_ops import (BOUNDARY_TYPES, EPS, GUARD, NORM_TYPES, TYPES, Matrix, eng, f64, ptr,  # noqa: F401
                                vec, within)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [3, 7, 64, 100, 768, 1000, 1021, 2900, 4099, 8190, 16384])
def test_norm_of_rows_far_from_zero(eng, cols):
    """y, mean and rstd of rows up to 100,000 times their spread from zero, and of constant rows, as two passes
    give them (test_block_bounds.py: without the correction of the mean they are off by more)."""
    rng = np.random.default_rng(cols)
    rows = far_rows(rng, cols)
    w, b = vec(1 + 0.2 * rng.standard_normal(cols)), vec(0.3 * rng.standard_normal(cols))
    n = len(rows)
    for xt, yt in NORM_TYPES:
        for weights in ((None, None), (w, b)):
            x, y = Matrix(n, cols, xt, torch.from_numpy(rows).clamp(-6e4, 6e4)), Matrix(n, cols, yt)
            mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
            eng.layer_norm_device(xt, yt, n, cols, x.at, cols, ptr(weights[0]), ptr(weights[1]), EPS, y.at, cols,
                                  ptr(mean), ptr(rstd))
            args = x.f64(), f64(weights[0]), f64(weights[1]), EPS
            want = ref.norm(*args)
            for got, wanted, bound, what in zip((y.f64(), f64(mean), f64(rstd)), want,
                                                two_pass_bounds(*args, *want, yt), ("y", "mean", "rstd")):
                within(got, wanted, bound, (what, cols, xt, yt))
    # The boundary, h being those rows: res + 0.
    x, res = Matrix(n, cols, "fp32", torch.zeros(n, cols)), Matrix(n, cols, "fp32", torch.from_numpy(rows))
    h, y = Matrix(n, cols, "fp32"), Matrix(n, cols, "fp32")
    mean, rstd = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    eng.dropout_add_norm_device("fp32", "fp32", "fp32", n, cols, x.at, cols, res.at, cols, 0.1, 1, 2, ptr(w), ptr(b), EPS,
                                h.at, cols, y.at, cols, ptr(mean), ptr(rstd))
    assert torch.equal(h.view, res.view)
    args = h.f64(), f64(w), f64(b), EPS
    want = ref.norm(*args)
    for got, wanted, bound, what in zip((y.f64(), f64(mean), f64(rstd)), want, two_pass_bounds(*args, *want, "fp32"),
                                        ("y", "mean", "rstd")):
        within(got, wanted, bound, ("boundary", what, cols))


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


@pytest.mark.parametrize("cols", [5, 768, 4099, 16384])
def test_largest_values(eng, cols):
    """Elements of up to 1e17 in magnitude stay in fp32's range at every width."""
    rng = np.random.default_rng(cols)
    rows = 1e17 * rng.uniform(-1, 1, (6, cols))
    rows[1] = np.where(rng.random(cols) < 0.5, 1e17, -1e17)
    rows[2] = 1e17 - 1e10 * rng.random(cols)
    for xt, yt in (("fp32", "fp32"), ("fp32", "bf16"), ("bf16", "bf16")):
        x, y = Matrix(6, cols, xt, torch.from_numpy(rows)), Matrix(6, cols, yt)
        mean, rstd = torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
        eng.layer_norm_device(xt, yt, 6, cols, x.at, cols, None, None, EPS, y.at, cols, ptr(mean), ptr(rstd))
        want = ref.norm(x.f64(), None, None, EPS)
        bounds = two_pass_bounds(x.f64(), None, None, EPS, *want, yt)
        for got, wanted, bound, what in zip((y.f64(), f64(mean), f64(rstd)), want, bounds, ("y", "mean", "rstd")):
            within(got, wanted, bound, (what, cols, xt, yt))


def test_dropout_writes_nothing_past_a_long_row(eng):
    """A row of more than 2^31 columns, two launches, the last vector a part of one: its last columns are right and
    what stands behind them stays."""
    long = 2 ** 31 + 21
    buf = torch.full((long + 32,), GUARD, dtype=torch.bfloat16, device="cuda")
    buf[:long] = 1.0
    eng.dropout_device("bf16", "bf16", 1, long, ptr(buf), long, None, 0, 0.5, 3, 4, ptr(buf), long)
    for c0 in (0, 2 ** 31 - 64, long - 64):
        c = np.arange(c0, c0 + 64)
        keep, scale = ref.keep_scale(np.zeros(1, np.int64), c, 0.5, 3, 4)
        assert np.array_equal(buf[c0: c0 + 64].float().cpu().numpy(), (keep[0] * scale).astype(np.float32)), c0
    assert bool((buf[long:] == GUARD).all())


@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("bf16", "fp32")])
def test_dropout_of_more_elements_than_a_launch_takes(eng, xt, yt):
    """2^28 blocks of eight columns a launch: the second one starts inside a row."""
    cols, per = 8197, 1025
    split = 2 ** 28 // per
    rows = split + 5
    x = torch.zeros(rows, cols, dtype=TYPES[xt], device="cuda")
    y = torch.full((rows * cols + 32,), GUARD, dtype=TYPES[yt], device="cuda")
    at = [0, 1, split - 1, split, split + 1, rows - 1]
    x[at] = torch.from_numpy(np.random.default_rng(5).standard_normal((6, cols))).to(TYPES[xt]).cuda()
    eng.dropout_device(xt, yt, rows, cols, ptr(x), cols, None, 0, 0.25, 6, 7, ptr(y), cols)
    want = ref.drop(f64(x[at]), ref.keep_scale(np.array(at), cols, 0.25, 6, 7))
    got = y[:rows * cols].view(rows, cols)
    within(got[at], want, 2 * ref.U * np.abs(want) + ref.rounding(np.abs(want) * (1 + 2 * ref.U), yt), (xt, yt))
    assert bool((y[rows * cols:] == GUARD).all()) and not bool(got[2:split - 1].any())
