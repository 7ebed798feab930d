"""The training-block operators on the GPU (LayerNorm, dropout, the residual
boundary and their gradients) against plain float64 forms, at the sizes, types,
strides and values where they can go wrong. Bounds: block_reference.py."""
import numpy as np
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu

EPS = 1e-5
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NORM_TYPES = [("fp32", "fp32"), ("fp32", "bf16"), ("fp32", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")]
BOUNDARY_TYPES = [("fp32", "fp32", "fp32"), ("bf16", "fp32", "bf16"), ("fp16", "fp32", "fp16"),
                  ("fp32", "fp32", "bf16"), ("fp32", "fp32", "fp16"), ("bf16", "bf16", "bf16"),
                  ("fp16", "fp16", "fp16")]
# Around every size where a kernel changes: blocks of 8 columns, a wave's and a
# workgroup's rows, the widest row.
COLS = [1, 2, 3, 4, 5, 7, 8, 9, 31, 33, 100, 64, 127, 255, 256, 257, 384, 511, 512, 513, 768, 1000, 1023, 1024, 1025, 1152, 1536, 2047,
        2048, 2049, 4096, 4099, 6000, 8192, 8193, 6145, 9999, 12000, 16383, 16384]
ROWS = [1, 2, 3, 5, 7, 8, 9, 16, 17, 31, 33, 64, 65, 203, 530]
GUARD = 7.25  # what stands around an array's columns; exact in every type


@pytest.fixture(scope="module")
def eng():
    from decide_amd import Engine, NoGPUError
    from decide_amd.nn import Config

    cfg = Config(hidden=256, intermediate=384, heads=4, layers=1, vocab=8, layer_types=["full_attention"])
    try:
        e = Engine(cfg, None, precision="fp32")
    except NoGPUError:
        pytest.skip("no GPU")
    e.set_stream(torch.cuda.current_stream().cuda_stream)
    yield e
    e.close()


class Matrix:
    """rows x cols of a type inside a larger buffer: `lead` elements before, row stride cols + pad."""

    def __init__(self, rows, cols, dtype, values=None, lead=0, pad=0):
        self.rows, self.cols, self.ld, self.dtype, self.lead = rows, cols, cols + pad, dtype, lead
        self.buf = torch.full((lead + rows * self.ld + 16,), GUARD, dtype=TYPES[dtype], device="cuda")
        self.view = self.buf[lead: lead + rows * self.ld].view(rows, self.ld)[:, :cols]
        if values is not None:
            self.view.copy_(values)
        self.at = self.buf.data_ptr() + lead * self.buf.element_size()

    def f64(self):
        return self.view.double().cpu().numpy()

    def untouched_outside(self):
        b = self.buf.clone()
        b[self.lead: self.lead + self.rows * self.ld].view(self.rows, self.ld)[:, :self.cols] = GUARD
        return bool((b == GUARD).all())


def vec(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream_values(rng, rows, cols):
    """A residual stream: rows of different scale and offset, a few large columns."""
    v = rng.standard_normal((rows, cols)) * (0.3 + rng.random((rows, 1)) * 3) + rng.standard_normal((rows, 1))
    v[:, ::13] *= 10
    return torch.from_numpy(v).cuda()


def within(got, want, bound, what):
    got = f64(got) if torch.is_tensor(got) else got
    assert got.shape == want.shape
    assert np.array_equal(np.isfinite(got), np.isfinite(want)), what
    off = np.abs(got - want) - bound
    assert not (off > 0).any(), (what, float((np.abs(got - want) / np.maximum(bound, 1e-300)).max()))


def check_norm(eng, rng, rows, cols, xt, yt, lead=0, pad=0, weight=True, bias=True, values=None):
    x = Matrix(rows, cols, xt, stream_values(rng, rows, cols) if values is None else values, lead, pad)
    y = Matrix(rows, cols, yt, None, lead, pad)
    w = vec(1 + 0.2 * rng.standard_normal(cols)) if weight else None
    b = vec(0.3 * rng.standard_normal(cols)) if bias else None
    mean, rstd = torch.full((rows + 1,), GUARD, device="cuda"), torch.full((rows + 1,), GUARD, device="cuda")
    eng.layer_norm_device(xt, yt, rows, cols, x.at, x.ld, ptr(w), ptr(b), EPS, y.at, y.ld, ptr(mean), ptr(rstd))
    xv = x.f64()
    want = ref.norm(xv, f64(w), f64(b), EPS)
    bounds = ref.norm_bounds(xv, f64(w), f64(b), EPS, *want, yt)
    for got, wanted, bound, what in zip((y.f64(), f64(mean)[:rows], f64(rstd)[:rows]), want, bounds,
                                        ("y", "mean", "rstd")):
        within(got, wanted, bound, (what, rows, cols, xt, yt, pad))
    assert y.untouched_outside() and float(mean[rows]) == GUARD and float(rstd[rows]) == GUARD
    return y


@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_sizes(eng, cols):
    rng = np.random.default_rng(cols)
    for k, (xt, yt) in enumerate(NORM_TYPES):
        rows = ROWS[(cols + 3 * k) % len(ROWS)]
        check_norm(eng, rng, rows, cols, xt, yt, weight=k != 1, bias=k % 2 == 0)
        check_norm(eng, rng, rows, cols, xt, yt, lead=1 + k, pad=(1, 3, 8, 5, 2)[k])


def test_layer_norm_rows_far_from_zero(eng):
    """Rows whose spread is small against their mean (1,000 times): the squares of the differences, not
    the difference of the squares."""
    rng = np.random.default_rng(2)
    for cols in (64, 768, 4099):
        v = torch.from_numpy(1000 + rng.standard_normal((9, cols))).cuda()
        check_norm(eng, rng, 9, cols, "fp32", "fp32", values=v)


def test_layer_norm_values(eng):
    """Constant rows give the bias (rstd 1 / sqrt(eps)), zeros too; an infinity or a NaN makes its own
    row NaN and no other."""
    rng = np.random.default_rng(3)
    for cols in (1, 8, 100, 768, 2900, 9000):
        v = torch.from_numpy(rng.standard_normal((8, cols))).cuda()
        v[0], v[1] = 0.0, 3.5
        v[3, cols // 2], v[5, 0], v[6, cols - 1] = float("inf"), float("nan"), float("-inf")
        x = Matrix(8, cols, "fp32", v)
        y = Matrix(8, cols, "fp32")
        b = vec(0.3 * rng.standard_normal(cols))
        mean, rstd = torch.empty(8, device="cuda"), torch.empty(8, device="cuda")
        eng.layer_norm_device("fp32", "fp32", 8, cols, x.at, cols, None, ptr(b), EPS, y.at, cols, ptr(mean), ptr(rstd))
        got = y.view.cpu()
        assert torch.equal(got[0], b.cpu()) and torch.equal(got[1], b.cpu())
        assert float(mean[1]) == 3.5 and abs(float(rstd[1]) * EPS ** 0.5 - 1) < 1e-6
        for r in range(8):
            assert bool(got[r].isnan().all()) == (r in (3, 5, 6)), (cols, r)
            assert r in (3, 5, 6) or bool(got[r].isfinite().all())


def grad_case(rng, rows, cols, dt, st, dxt, lead=0, pad=0, weight=True):
    """Arrays of a gradient call, with the statistics as the forward gives them (rounded to fp32)."""
    h = Matrix(rows, cols, st, stream_values(rng, rows, cols), lead, pad)
    _, mean, rstd = ref.norm(h.f64(), None, None, EPS)
    c = {"rows": rows, "cols": cols, "h": h, "mean": vec(mean), "rstd": vec(rstd),
         "dy": Matrix(rows, cols, dt, torch.from_numpy(0.1 * rng.standard_normal((rows, cols))), lead, pad),
         "dh": Matrix(rows, cols, st, torch.from_numpy(0.1 * rng.standard_normal((rows, cols))), lead, pad),
         "dres": Matrix(rows, cols, st, None, lead, pad), "dx": Matrix(rows, cols, dxt, None, lead, pad),
         "w": vec(1 + 0.2 * rng.standard_normal(cols)) if weight else None}
    from decide_amd.nn import Engine

    c["work_bytes"] = Engine.norm_backward_workspace(rows, cols)
    c["work"] = torch.full((c["work_bytes"] // 4 + 8,), GUARD, device="cuda")
    c["dw"], c["db"] = torch.full((cols + 1,), 0.5, device="cuda"), torch.full((cols + 1,), -0.25, device="cuda")
    return c


def check_grad(eng, rng, rows, cols, dt, st, dxt, boundary, lead=0, pad=0, weight=True, dh=True, accumulate=False,
               sums=("dw", "db"), p=0.2):
    c = grad_case(rng, rows, cols, dt, st, dxt, lead, pad, weight)
    dw, db = (c[k] if k in sums else None for k in ("dw", "db"))
    seed, offset = int(rng.integers(0, 2 ** 63)) * 2 + 1, int(rng.integers(0, 2 ** 62)) * 4 + 3
    tail = (ptr(dw), ptr(db), accumulate, ptr(c["work"]), c["work_bytes"])
    if boundary:
        eng.dropout_add_norm_backward_device(
            dt, st, dxt, rows, cols, c["dy"].at, c["dy"].ld, c["dh"].at if dh else None, c["dh"].ld if dh else 0,
            c["h"].at, c["h"].ld, p, seed, offset, ptr(c["w"]), ptr(c["mean"]), ptr(c["rstd"]), c["dres"].at,
            c["dres"].ld, c["dx"].at, c["dx"].ld, *tail)
    else:
        eng.layer_norm_backward_device(dt, st, rows, cols, c["dy"].at, c["dy"].ld, c["h"].at, c["h"].ld, ptr(c["w"]),
                                       ptr(c["mean"]), ptr(c["rstd"]), c["dres"].at, c["dres"].ld, *tail)
    dy, h, w, mean, rstd = c["dy"].f64(), c["h"].f64(), f64(c["w"]), f64(c["mean"]), f64(c["rstd"])
    dx, gw, gb = ref.norm_grad(dy, h, w, mean, rstd)
    extra = c["dh"].f64() if boundary and dh else np.zeros_like(dx)
    dres = dx + extra
    e, ew, eb = ref.norm_grad_bounds(dy, h, w, mean, rstd, dres, st, np.abs(extra))
    what = (rows, cols, dt, st, dxt, pad)
    within(c["dres"].f64(), dres, e, ("dres", *what))
    if boundary:
        mask = ref.keep_scale(rows, cols, p, seed, offset)
        e32 = ref.norm_grad_bounds(dy, h, w, mean, rstd, dres, "fp32", np.abs(extra))[0] * mask[1]
        want = ref.drop(dres, mask)
        # The unrounded sum scaled (two roundings in fp32), then rounded to dx's type; dropped ones are 0.
        bound = np.where(mask[0], e32 + 2 * ref.U * np.abs(want) + ref.rounding(np.abs(want) + e32, dxt), 0.0)
        within(c["dx"].f64(), want, bound, ("dx", *what))
    else:
        assert bool((c["dx"].buf == GUARD).all())
    for name, got, want, bound, start in (("dw", c["dw"], gw, ew, 0.5), ("db", c["db"], gb, eb, -0.25)):
        assert float(got[cols]) == start
        if name not in sums:
            assert bool((got == start).all())
            continue
        base = start if accumulate else 0.0
        within(got[:cols], want + base, bound + ref.U * (np.abs(want) + 1), (name, *what))
    for m in ("dy", "dh", "h", "dres", "dx"):
        assert c[m].untouched_outside()
    assert bool((c["work"][c["work_bytes"] // 4:] == GUARD).all())


@pytest.mark.parametrize("cols", COLS)
def test_norm_gradient_sizes(eng, cols):
    rng = np.random.default_rng(cols + 1)
    for k, (st, dt) in enumerate(NORM_TYPES):
        rows = ROWS[(cols + 5 * k) % len(ROWS)]
        check_grad(eng, rng, rows, cols, dt, st, st, False, weight=k != 1, accumulate=k % 2 == 0)
        check_grad(eng, rng, rows, cols, dt, st, st, False, lead=1 + k, pad=(1, 3, 8, 5, 2)[k], accumulate=k % 2 == 1)


@pytest.mark.parametrize("cols", COLS)
def test_boundary_gradient_sizes(eng, cols):
    rng = np.random.default_rng(cols + 2)
    for k, (dt, st, dxt) in enumerate(BOUNDARY_TYPES):
        rows = ROWS[(cols + 5 * k) % len(ROWS)]
        check_grad(eng, rng, rows, cols, dt, st, dxt, True, weight=k != 1, dh=k != 2, accumulate=k % 2 == 0)
        check_grad(eng, rng, rows, cols, dt, st, dxt, True, lead=1 + k, pad=(1, 3, 8, 5, 2, 4, 16)[k],
                   accumulate=k % 2 == 1)


@pytest.mark.parametrize("cols", [4100, 8196, 8197, 12288, 12289, 16380])
@pytest.mark.parametrize("boundary", [False, True])
def test_gradient_of_wide_rows(eng, cols, boundary):
    """Rows of every shape past 4,096 columns, of every type, in more rows than one launch takes."""
    rng = np.random.default_rng(cols + boundary)
    for k, (dt, st, dxt) in enumerate(BOUNDARY_TYPES if boundary else [(d, s, s) for s, d in NORM_TYPES]):
        check_grad(eng, rng, 517 + k, cols, dt, st, dxt, boundary, accumulate=k % 2 == 0, pad=k % 3)


@pytest.mark.parametrize("rows", [64, 257, 512, 513, 1000, 4097, 12288])
def test_gradient_many_rows(eng, rows):
    """Rows past every workgroup's first ones; the sums over them, and each alone."""
    rng = np.random.default_rng(rows)
    check_grad(eng, rng, rows, 96, "bf16", "fp32", "bf16", True)
    check_grad(eng, rng, rows, 96, "bf16", "bf16", "bf16", False, sums=("dw",))
    check_grad(eng, rng, rows, 100, "fp32", "fp32", "fp32", False, sums=("db",), accumulate=True)
    check_grad(eng, rng, rows, 100, "fp32", "fp32", "bf16", True, sums=())
    if rows <= 4097:
        check_grad(eng, rng, rows, 768, "bf16", "fp32", "bf16", True)
        check_grad(eng, rng, rows, 2050, "fp16", "fp16", "fp16", False)


def check_dropout(eng, rng, rows, cols, xt, yt, p, residual=False, lead=0, pad=0, seed=None, offset=None):
    seed = int(rng.integers(0, 2 ** 63)) * 2 + 1 if seed is None else seed
    offset = int(rng.integers(0, 2 ** 63)) * 2 if offset is None else offset
    x = Matrix(rows, cols, xt, torch.from_numpy(rng.standard_normal((rows, cols))), lead, pad)
    res = Matrix(rows, cols, yt, torch.from_numpy(rng.standard_normal((rows, cols))), lead + 1, pad) if residual else None
    y = Matrix(rows, cols, yt, None, lead, pad)
    eng.dropout_device(xt, yt, rows, cols, x.at, x.ld, res.at if res else None, res.ld if res else 0, p, seed, offset,
                       y.at, y.ld)
    mask = ref.keep_scale(rows, cols, p, seed, offset)
    d = ref.drop(x.f64(), mask)
    want = d + (res.f64() if res else 0.0)
    # The scale's and the product's rounding, the sum's, and the output's; without a residual dropped ones are 0.
    e = 2 * ref.U * np.abs(d) + (ref.U * np.abs(want) if residual else 0.0)
    bound = e + ref.rounding(np.abs(want) + e, yt)
    if not residual:
        bound = np.where(mask[0], bound, 0.0)
    within(y.f64(), want, bound, (rows, cols, xt, yt, p, residual, pad))
    assert y.untouched_outside()


@pytest.mark.parametrize("cols", [1, 3, 8, 15, 16, 100, 768, 1152, 4099, 40001])
def test_dropout(eng, cols):
    rng = np.random.default_rng(cols + 5)
    pairs = [("fp32", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp32"), ("fp32", "bf16"),
             ("fp16", "fp32"), ("fp32", "fp16")]
    for k, (xt, yt) in enumerate(pairs):
        rows = ROWS[(cols + k) % len(ROWS)]
        p = (0.1, 0.5, 0.0, 0.25, 0.9, 1.0, 1e-4)[k]
        check_dropout(eng, rng, rows, cols, xt, yt, p)
        check_dropout(eng, rng, rows, cols, xt, yt, p, residual=True, lead=k, pad=(0, 1, 8, 3, 2, 5, 16)[k])


def test_dropout_seed_and_offset_words(eng):
    """Every bit of the 64-bit seed and offset counts."""
    rng = np.random.default_rng(6)
    for bit in (0, 1, 31, 32, 47, 63):
        check_dropout(eng, rng, 5, 100, "fp32", "fp32", 0.3, seed=1 << bit, offset=0)
        check_dropout(eng, rng, 5, 100, "fp32", "fp32", 0.3, seed=0, offset=1 << bit)


def test_dropped_values_are_zero(eng):
    """An infinity or a NaN that is dropped leaves no trace, in the output or in its row's norm."""
    rows, cols, p, seed, offset = 6, 768, 0.5, 11, 12
    keep, scale = ref.keep_scale(rows, cols, p, seed, offset)
    dropped = torch.from_numpy(~keep).cuda()
    x = Matrix(rows, cols, "bf16", torch.ones(rows, cols))
    x.view[dropped] = float("nan")
    x.view[0][dropped[0]] = float("inf")
    y = Matrix(rows, cols, "bf16")
    eng.dropout_device("bf16", "bf16", rows, cols, x.at, cols, None, 0, p, seed, offset, y.at, cols)
    assert torch.equal(y.view, torch.from_numpy(keep * scale).to(torch.bfloat16).cuda())
    res, h, n = Matrix(rows, cols, "fp32", torch.zeros(rows, cols)), Matrix(rows, cols, "fp32"), Matrix(rows, cols, "bf16")
    eng.dropout_add_norm_device("bf16", "fp32", "bf16", rows, cols, x.at, cols, res.at, cols, p, seed, offset, None, None,
                                EPS, h.at, cols, n.at, cols)
    assert torch.equal(h.view, torch.from_numpy(keep * scale).float().cuda()) and bool(n.view.isfinite().all())


def check_boundary(eng, rng, rows, cols, xt, st, yt, lead=0, pad=0, p=0.15, weight=True, bias=True):
    x = Matrix(rows, cols, xt, torch.from_numpy(rng.standard_normal((rows, cols))), lead, pad)
    res = Matrix(rows, cols, st, stream_values(rng, rows, cols), lead, pad)
    h, y = Matrix(rows, cols, st, None, lead, pad), Matrix(rows, cols, yt, None, lead, pad)
    w = vec(1 + 0.2 * rng.standard_normal(cols)) if weight else None
    b = vec(0.3 * rng.standard_normal(cols)) if bias else None
    mean, rstd = torch.full((rows + 1,), GUARD, device="cuda"), torch.full((rows + 1,), GUARD, device="cuda")
    seed, offset = int(rng.integers(0, 2 ** 63)), int(rng.integers(0, 2 ** 63))
    eng.dropout_add_norm_device(xt, st, yt, rows, cols, x.at, x.ld, res.at, res.ld, p, seed, offset, ptr(w), ptr(b),
                                EPS, h.at, h.ld, y.at, y.ld, ptr(mean), ptr(rstd))
    d = ref.drop(x.f64(), ref.keep_scale(rows, cols, p, seed, offset))
    want = res.f64() + d
    e = 2 * ref.U * np.abs(d) + ref.U * np.abs(want)
    within(h.f64(), want, e + ref.rounding(np.abs(want) + e, st), ("h", rows, cols, xt, st, yt, pad))
    hv = h.f64()  # the norm is of h as it is stored
    n = ref.norm(hv, f64(w), f64(b), EPS)
    for got, wanted, bound, what in zip((y.f64(), f64(mean)[:rows], f64(rstd)[:rows]), n,
                                        ref.norm_bounds(hv, f64(w), f64(b), EPS, *n, yt), ("y", "mean", "rstd")):
        within(got, wanted, bound, (what, rows, cols, xt, st, yt, pad))
    for m in (x, res, h, y):
        assert m.untouched_outside()
    assert float(mean[rows]) == GUARD and float(rstd[rows]) == GUARD


@pytest.mark.parametrize("cols", COLS)
def test_boundary_sizes(eng, cols):
    rng = np.random.default_rng(cols + 9)
    for k, (xt, st, yt) in enumerate(BOUNDARY_TYPES):
        rows = ROWS[(cols + 3 * k) % len(ROWS)]
        check_boundary(eng, rng, rows, cols, xt, st, yt, p=(0.15, 0.0, 1.0, 0.5)[k % 4], weight=k != 1, bias=k % 2 == 0)
        check_boundary(eng, rng, rows, cols, xt, st, yt, lead=1 + k, pad=(1, 3, 8, 5, 2, 4, 16)[k])


def test_boundary_many_rows(eng):
    rng = np.random.default_rng(31)
    for rows, cols in ((20011, 40), (4099, 768), (3001, 1300)):
        check_boundary(eng, rng, rows, cols, "bf16", "fp32", "bf16")
        check_norm(eng, rng, rows, cols, "fp32", "bf16")


def test_more_rows_than_a_launch_takes(eng):
    """A row per workgroup and 2^20 workgroups a launch: rows on both sides of the second launch's first."""
    rows, cols = 2 ** 20 + 5, 1040
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    res, h, y = (torch.zeros_like(x) for _ in range(3))
    at = [0, 1, 2 ** 20 - 1, 2 ** 20, rows - 1]
    rng = np.random.default_rng(77)
    x[at] = torch.from_numpy(rng.standard_normal((5, cols))).to(torch.bfloat16).cuda()
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    eng.dropout_add_norm_device("bf16", "bf16", "bf16", rows, cols, ptr(x), cols, ptr(res), cols, 0.25, 9, 8, None, None,
                                EPS, ptr(h), cols, ptr(y), cols, ptr(mean), ptr(rstd))
    keep = ref.keep_scale(np.array(at), cols, 0.25, 9, 8)
    want = ref.drop(f64(x[at]), keep)
    within(h[at], want, 2 * ref.U * np.abs(want) + ref.rounding(np.abs(want) * (1 + 2 * ref.U), "bf16"), "h")
    n = ref.norm(f64(h[at]), None, None, EPS)
    bounds = ref.norm_bounds(f64(h[at]), None, None, EPS, *n, "bf16")
    for got, wanted, bound in zip((y[at], mean[at], rstd[at]), n, bounds):
        within(got, wanted, bound, "rows")


def test_no_rows(eng):
    """No rows: nothing is touched, and the sums are the empty sum (stored, or added to what is there)."""
    g = torch.full((16,), GUARD, device="cuda")
    for acc in (False, True):
        dw, db = torch.full((8,), 3.0, device="cuda"), torch.full((8,), 4.0, device="cuda")
        eng.layer_norm_backward_device("fp32", "fp32", 0, 8, None, 8, None, 8, None, None, None, None, 8, ptr(dw),
                                       ptr(db), acc, ptr(g), 64)
        assert dw.tolist() == [3.0 if acc else 0.0] * 8 and db.tolist() == [4.0 if acc else 0.0] * 8
    eng.layer_norm_device("fp32", "bf16", 0, 8, None, 8, None, None, EPS, None, 8)
    eng.dropout_device("fp32", "bf16", 0, 8, None, 8, None, 0, 0.1, 1, 2, None, 8)
    eng.dropout_device("fp32", "bf16", 8, 0, None, 8, None, 0, 0.1, 1, 2, None, 8)
    assert bool((g == GUARD).all())


@pytest.mark.parametrize("rows", [37, 530])
@pytest.mark.parametrize("cols", [5, 100, 768, 2049, 12001])
def test_in_place(eng, cols, rows):
    """An output in an input's array gives the bits of the call with arrays of its own."""
    rng = np.random.default_rng(cols)
    p, seed, offset = 0.2, 5, 6
    v, r = stream_values(rng, rows, cols), stream_values(rng, rows, cols)
    w = vec(1 + 0.2 * rng.standard_normal(cols))
    x, res = Matrix(rows, cols, "bf16", v), Matrix(rows, cols, "bf16", r)
    h, y = Matrix(rows, cols, "bf16"), Matrix(rows, cols, "bf16")

    def boundary(h, y, x=x, res=res):
        eng.dropout_add_norm_device("bf16", "bf16", "bf16", rows, cols, x.at, cols, res.at, cols, p, seed, offset,
                                    ptr(w), None, EPS, h.at, cols, y.at, cols, ptr(mean), ptr(rstd))

    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    boundary(h, y)
    x2, r2 = Matrix(rows, cols, "bf16", v), Matrix(rows, cols, "bf16", r)
    boundary(r2, x2, x2, r2)
    assert torch.equal(r2.view, h.view) and torch.equal(x2.view, y.view)
    x2, r2 = Matrix(rows, cols, "bf16", v), Matrix(rows, cols, "bf16", r)
    boundary(x2, r2, x2, r2)
    assert torch.equal(x2.view, h.view) and torch.equal(r2.view, y.view)
    n = Matrix(rows, cols, "bf16")
    eng.layer_norm_device("bf16", "bf16", rows, cols, h.at, cols, ptr(w), None, EPS, n.at, cols)
    h2 = Matrix(rows, cols, "bf16", h.view)
    eng.layer_norm_device("bf16", "bf16", rows, cols, h2.at, cols, ptr(w), None, EPS, h2.at, cols)
    assert torch.equal(h2.view, n.view) and torch.equal(n.view, y.view)
    c = grad_case(rng, rows, cols, "bf16", "bf16", "bf16")

    def grad(dres, dx, dy, dh, dw):
        eng.dropout_add_norm_backward_device("bf16", "bf16", "bf16", rows, cols, dy.at, cols, dh.at, cols, c["h"].at,
                                             cols, p, seed, offset, ptr(w), ptr(c["mean"]), ptr(c["rstd"]), dres.at,
                                             cols, dx.at, cols, ptr(dw), None, False, ptr(c["work"]), c["work_bytes"])

    dw1, dw2, dw3 = (torch.empty(cols, device="cuda") for _ in range(3))
    grad(c["dres"], c["dx"], c["dy"], c["dh"], dw1)
    dy3 = Matrix(rows, cols, "bf16", c["dy"].view)
    dx3 = Matrix(rows, cols, "bf16")
    grad(dy3, dx3, dy3, c["dh"], dw3)
    assert torch.equal(dy3.view, c["dres"].view) and torch.equal(dx3.view, c["dx"].view) and torch.equal(dw1, dw3)
    dy2, dh2 = Matrix(rows, cols, "bf16", c["dy"].view), Matrix(rows, cols, "bf16", c["dh"].view)
    grad(dh2, dy2, dy2, dh2, dw2)
    assert torch.equal(dh2.view, c["dres"].view) and torch.equal(dy2.view, c["dx"].view) and torch.equal(dw1, dw2)


def test_columns_of_one_buffer(eng):
    """Inputs and outputs as columns of one [rows x 3n] buffer."""
    rng = np.random.default_rng(8)
    rows, n = 19, 100
    buf = torch.from_numpy(rng.standard_normal((rows, 3 * n))).float().cuda()
    before = buf.clone()
    at = [buf.data_ptr() + 4 * n * k for k in range(3)]
    eng.dropout_add_norm_device("fp32", "fp32", "fp32", rows, n, at[0], 3 * n, at[1], 3 * n, 0.1, 1, 2, None, None, EPS,
                                at[1], 3 * n, at[2], 3 * n)
    keep = ref.keep_scale(rows, n, 0.1, 1, 2)
    want = f64(before[:, n:2 * n]) + ref.drop(f64(before[:, :n]), keep)
    assert torch.equal(buf[:, :n], before[:, :n])
    within(buf[:, n:2 * n], want, 4 * ref.U * (np.abs(want) + 3), "h")
    y = ref.norm(f64(buf[:, n:2 * n]), None, None, EPS)
    within(buf[:, 2 * n:], y[0], ref.norm_bounds(f64(buf[:, n:2 * n]), None, None, EPS, *y, "fp32")[0], "y")


def test_offsets_past_32_bits(eng):
    """Rows whose byte and element offsets pass 2^32 (a row stride of 2^31 + 9 elements), and columns past 2^31."""
    ld, cols = 2 ** 31 + 9, 40
    buf = torch.zeros(2 * ld + 64, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(9)
    v = torch.from_numpy(rng.standard_normal((3, cols))).to(torch.bfloat16).cuda()
    for r in range(3):
        buf[r * ld: r * ld + cols] = v[r]
    y, y2 = Matrix(3, cols, "bf16"), Matrix(3, cols, "bf16")
    eng.layer_norm_device("bf16", "bf16", 3, cols, ptr(buf), ld, None, None, EPS, y.at, cols)
    eng.layer_norm_device("bf16", "bf16", 3, cols, ptr(v), cols, None, None, EPS, y2.at, cols)
    assert torch.equal(y.view, y2.view)
    eng.dropout_device("bf16", "bf16", 3, cols, ptr(v), cols, None, 0, 0.3, 1, 2, ptr(buf), ld)
    eng.dropout_device("bf16", "bf16", 3, cols, ptr(v), cols, None, 0, 0.3, 1, 2, y.at, cols)
    for r in range(3):
        assert torch.equal(buf[r * ld: r * ld + cols], y.view[r])
    long = 2 ** 31 + 21
    buf[:long] = 1.0
    eng.dropout_device("bf16", "bf16", 1, long, ptr(buf), long, None, 0, 0.5, 3, 4, ptr(buf), long)
    for c0 in (0, 2 ** 30 - 8, 2 ** 31 - 24, 2 ** 31):
        c = np.arange(c0, min(c0 + 64, long))
        keep, scale = ref.keep_scale(np.zeros(1, np.int64), c, 0.5, 3, 4)
        assert np.array_equal(buf[c0: c0 + len(c)].float().cpu().numpy(), (keep[0] * scale).astype(np.float32)), c0
    assert float(buf[long]) == 0.0 or ld < long + 1


def test_gradient_of_rows_that_are_not_finite(eng):
    """A NaN or an infinity in dy, dh or h makes its own row's gradient NaN (or infinite) and the sums of its
    column, and nothing else; dropped elements of dx are 0 all the same."""
    for rows, cols in ((40, 96), (700, 96), (40, 3001), (40, 5001)):
        rng = np.random.default_rng(rows + cols)
        c = grad_case(rng, rows, cols, "fp32", "fp32", "fp32")
        c["dy"].view[3, 5], c["dh"].view[7, 6], c["dy"].view[9, cols - 1] = float("nan"), float("inf"), float("-inf")
        eng.dropout_add_norm_backward_device(
            "fp32", "fp32", "fp32", rows, cols, c["dy"].at, cols, c["dh"].at, cols, c["h"].at, cols, 0.5, 1, 2, None,
            ptr(c["mean"]), ptr(c["rstd"]), c["dres"].at, cols, c["dx"].at, cols, ptr(c["dw"]), ptr(c["db"]), False,
            ptr(c["work"]), c["work_bytes"])
        keep, _ = ref.keep_scale(rows, cols, 0.5, 1, 2)
        dres, dx = c["dres"].f64(), c["dx"].f64()
        bad = ~np.isfinite(dres)
        assert bad[3].all() and bad[9].all() and bad[7].sum() == 1 and bad[7, 6] and dres[7, 6] == np.inf
        bad[[3, 7, 9]] = False
        assert not bad.any()
        assert (dx[~keep] == 0).all() and np.array_equal(~np.isfinite(dx), keep & ~np.isfinite(dres))
        for t in (c["dw"], c["db"]):
            assert np.flatnonzero(~np.isfinite(f64(t)[:cols])).tolist() == [5, cols - 1]


def test_equal_calls_give_equal_bits(eng):
    rng = np.random.default_rng(10)
    c = grad_case(rng, 3001, 768, "bf16", "fp32", "bf16")
    got = []
    for k in range(3):
        eng.dropout_add_norm_backward_device(
            "bf16", "fp32", "bf16", 3001, 768, c["dy"].at, 768, c["dh"].at, 768, c["h"].at, 768, 0.1, 1, 2, ptr(c["w"]),
            ptr(c["mean"]), ptr(c["rstd"]), c["dres"].at, 768, c["dx"].at, 768, ptr(c["dw"]), ptr(c["db"]), False,
            ptr(c["work"]), c["work_bytes"])
        got.append([t.clone() for t in (c["dres"].view, c["dx"].view, c["dw"], c["db"])])
        c["work"].normal_()
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_gradients_against_differences(eng):
    """Directional derivatives of sum(y * dy) + sum(h * dh) by central differences of the float64 forward.
    Second differences of a LayerNorm are O(step^2): with a step of 1e-4 they are far under the 1e-4 held here."""
    rng = np.random.default_rng(11)
    rows, cols, p, seed, offset = 13, 96, 0.3, 21, 22
    x, res = rng.standard_normal((rows, cols)), rng.standard_normal((rows, cols))
    w, b = 1 + 0.2 * rng.standard_normal(cols), 0.1 * rng.standard_normal(cols)
    x, res, w, b = (np.float64(np.float32(v)) for v in (x, res, w, b))
    dy, dh = (np.float64(np.float32(rng.standard_normal((rows, cols)))) for _ in range(2))
    mask = ref.keep_scale(rows, cols, p, seed, offset)

    def loss(x, res, w, b):
        h = res + ref.drop(x, mask)
        return (ref.norm(h, w, b, EPS)[0] * dy).sum() + (h * dh).sum()

    X, R = Matrix(rows, cols, "fp32", torch.from_numpy(x)), Matrix(rows, cols, "fp32", torch.from_numpy(res))
    H, Y, DR, DX = (Matrix(rows, cols, "fp32") for _ in range(4))
    DY, DH = Matrix(rows, cols, "fp32", torch.from_numpy(dy)), Matrix(rows, cols, "fp32", torch.from_numpy(dh))
    W, B, dw, db = vec(w), vec(b), torch.zeros(cols, device="cuda"), torch.zeros(cols, device="cuda")
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    n = eng.norm_backward_workspace(rows, cols)
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    eng.dropout_add_norm_device("fp32", "fp32", "fp32", rows, cols, X.at, cols, R.at, cols, p, seed, offset, ptr(W),
                                ptr(B), EPS, H.at, cols, Y.at, cols, ptr(mean), ptr(rstd))
    eng.dropout_add_norm_backward_device("fp32", "fp32", "fp32", rows, cols, DY.at, cols, DH.at, cols, H.at, cols, p,
                                         seed, offset, ptr(W), ptr(mean), ptr(rstd), DR.at, cols, DX.at, cols, ptr(dw),
                                         ptr(db), False, ptr(work), n)
    for k, grad in enumerate((DX.f64(), DR.f64(), f64(dw), f64(db))):
        for _ in range(4):
            v = rng.standard_normal(grad.shape)
            args = [x, res, w, b]
            up, down = list(args), list(args)
            up[k], down[k] = args[k] + 1e-4 * v, args[k] - 1e-4 * v
            want = (loss(*up) - loss(*down)) / 2e-4
            assert abs((grad * v).sum() - want) <= 1e-4 * np.sqrt((grad ** 2).sum() * (v ** 2).sum()), k


def test_block_of_sublayers(eng):
    """Two sub-layers as a program chains them: norm, product, boundary, product, boundary, forward and
    backward with the masks regenerated, against float64 autograd of the same network and masks."""
    rng = np.random.default_rng(12)
    rows, n, p, seed = 48, 768, 0.1, 99
    x0 = torch.from_numpy(np.float32(rng.standard_normal((rows, n)))).cuda()
    W = [torch.from_numpy(np.float32(rng.standard_normal((n, n)) / n ** 0.5)).cuda() for _ in range(2)]
    g = [vec(1 + 0.1 * rng.standard_normal(n)) for _ in range(3)]
    b = [vec(0.1 * rng.standard_normal(n)) for _ in range(3)]
    top = torch.from_numpy(np.float32(rng.standard_normal((rows, n)))).cuda()
    new = lambda: torch.empty(rows, n, device="cuda")  # noqa: E731
    mean, rstd = [torch.empty(3, rows, device="cuda").unbind(0) for _ in range(2)]
    y, h = [new() for _ in range(3)], [x0, new(), new()]
    eng.layer_norm_device("fp32", "fp32", rows, n, ptr(x0), n, ptr(g[0]), ptr(b[0]), EPS, ptr(y[0]), n, ptr(mean[0]),
                          ptr(rstd[0]))
    for k in (0, 1):
        u = y[k] @ W[k]
        eng.dropout_add_norm_device("fp32", "fp32", "fp32", rows, n, ptr(u), n, ptr(h[k]), n, p, seed, k, ptr(g[k + 1]),
                                    ptr(b[k + 1]), EPS, ptr(h[k + 1]), n, ptr(y[k + 1]), n, ptr(mean[k + 1]),
                                    ptr(rstd[k + 1]))
    bytes_ = eng.norm_backward_workspace(rows, n)
    work = torch.empty(bytes_, dtype=torch.uint8, device="cuda")
    dg, db = [torch.zeros(n, device="cuda") for _ in range(3)], [torch.zeros(n, device="cuda") for _ in range(3)]
    dW, dy, dh = [None, None], top, None
    for k in (1, 0):
        du, dr = new(), new()
        eng.dropout_add_norm_backward_device("fp32", "fp32", "fp32", rows, n, ptr(dy), n, ptr(dh), n, ptr(h[k + 1]), n,
                                             p, seed, k, ptr(g[k + 1]), ptr(mean[k + 1]), ptr(rstd[k + 1]), ptr(dr), n,
                                             ptr(du), n, ptr(dg[k + 1]), ptr(db[k + 1]), True, ptr(work), bytes_)
        dW[k], dy, dh = y[k].T @ du, du @ W[k].T, dr
    dx = new()
    eng.layer_norm_backward_device("fp32", "fp32", rows, n, ptr(dy), n, ptr(x0), n, ptr(g[0]), ptr(mean[0]),
                                   ptr(rstd[0]), ptr(dx), n, ptr(dg[0]), ptr(db[0]), True, ptr(work), bytes_)
    dx = dx + dh
    X, WW, G, B = (t if isinstance(t, torch.Tensor) else t for t in (
        x0.double().cpu().requires_grad_(), [w.double().cpu().requires_grad_() for w in W],
        [v.double().cpu().requires_grad_() for v in g], [v.double().cpu().requires_grad_() for v in b]))

    def norm(v, k):
        d = v - v.mean(1, keepdim=True)
        return d / (d.square().mean(1, keepdim=True) + EPS).sqrt() * G[k] + B[k]

    s, yy = X, norm(X, 0)
    for k in (0, 1):
        keep, scale = ref.keep_scale(rows, n, p, seed, k)
        s = s + torch.from_numpy(keep * scale) * (yy @ WW[k])
        yy = norm(s, k + 1)
    (yy * top.double().cpu()).sum().backward()
    # Each product and norm adds a few hundred roundings of 2^-24 at most: 1e-5 of the norm is far over them.
    for got, want in [(y[2], yy.detach()), (dx, X.grad)] + list(zip(dW, [w.grad for w in WW])) + \
            list(zip(dg, [v.grad for v in G])) + list(zip(db, [v.grad for v in B])):
        assert float((got.double().cpu() - want).norm() / want.norm()) < 1e-5


@pytest.mark.parametrize("rows", [60, 515])
def test_other_stream_and_graph(eng, rows):
    """The calls on another stream, captured into a graph and replayed on new inputs, with eager calls and
    synchronizations between the replays; two graphs with workspaces of their own replay side by side."""
    rng = np.random.default_rng(13)
    cols, p, seed, offset = 768, 0.1, 31, 32
    w = vec(1 + 0.2 * rng.standard_normal(cols))
    n = eng.norm_backward_workspace(rows, cols)

    def arrays():
        f, half = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.bfloat16, device="cuda")
        return {"x": torch.zeros(rows, cols, **half), "res": torch.zeros(rows, cols, **f), "h": torch.zeros(rows, cols, **f),
                "y": torch.zeros(rows, cols, **half), "mean": torch.zeros(rows, **f), "rstd": torch.zeros(rows, **f),
                "dres": torch.zeros(rows, cols, **f), "dx": torch.zeros(rows, cols, **half),
                "dw": torch.zeros(cols, **f), "db": torch.zeros(cols, **f),
                "work": torch.zeros(n + 16, dtype=torch.uint8, device="cuda")}

    def calls(a):
        q = {k: ptr(v) for k, v in a.items()}
        eng.dropout_add_norm_device("bf16", "fp32", "bf16", rows, cols, q["x"], cols, q["res"], cols, p, seed, offset,
                                    ptr(w), None, EPS, q["h"], cols, q["y"], cols, q["mean"], q["rstd"])
        eng.dropout_add_norm_backward_device("bf16", "fp32", "bf16", rows, cols, q["y"], cols, q["res"], cols, q["h"],
                                             cols, p, seed, offset, ptr(w), q["mean"], q["rstd"], q["dres"], cols,
                                             q["dx"], cols, q["dw"], q["db"], False, q["work"], n)
        eng.dropout_device("fp32", "fp32", rows, cols, q["dres"], cols, None, 0, 0.5, seed, 1, q["dres"], cols)

    outs = ("h", "y", "mean", "rstd", "dres", "dx", "dw", "db")
    sets, graphs = [arrays(), arrays()], []
    side = torch.cuda.Stream()
    before = torch.cuda.current_stream().cuda_stream
    try:
        for a in sets:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side):
                eng.set_stream(torch.cuda.current_stream().cuda_stream)
                calls(a)
            graphs.append(graph)
        eng.set_stream(before)
        for trial in range(4):
            fresh = arrays()
            fresh["x"].normal_()
            fresh["res"].normal_()
            for k, a in enumerate(sets):
                a["x"].copy_(fresh["x"])
                a["res"].copy_(fresh["res"])
                for o in outs:
                    a[o].zero_()
            torch.cuda.synchronize()
            other = torch.cuda.Stream()
            with torch.cuda.stream(other):
                graphs[1].replay()
            graphs[0].replay()
            eng.set_stream(side.cuda_stream)  # eager, on a stream that is not the current one
            calls(fresh)
            eng.synchronize()
            eng.set_stream(before)
            torch.cuda.synchronize()
            for a in sets:
                for o in outs:
                    assert torch.equal(a[o], fresh[o]), (trial, o)
    finally:
        eng.set_stream(before)


def test_two_contexts_at_once():
    """Two contexts without a model, each on a stream of its own, give what each gives alone."""
    import ctypes

    from decide_amd import native

    lib, rows, cols = native.lib, 4097, 768
    handles, streams = [], [torch.cuda.Stream() for _ in range(2)]
    try:
        for s in streams:
            h = ctypes.c_void_p()
            if lib.dn_open(0, ctypes.byref(h)) == native.DN_NO_GPU:
                pytest.skip("no GPU")
            handles.append(h)
            assert lib.dn_set_stream(h, s.cuda_stream) == 0
        n = lib.dn_norm_backward_workspace(rows, cols)
        data = []
        for k in range(2):
            g = torch.Generator(device="cuda").manual_seed(k)
            d = {name: torch.randn(rows, cols, generator=g, device="cuda") for name in ("dy", "dh", "h", "dres", "dx")}
            d["mean"], d["rstd"] = d["h"].mean(1), 1 / d["h"].std(1)
            d["dw"], d["work"] = torch.zeros(cols, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
            data.append(d)

        def call(h, d, k):
            q = {name: t.data_ptr() for name, t in d.items()}
            assert lib.dn_dropout_add_norm_backward_device(
                h, 0, 0, 0, rows, cols, q["dy"], cols, q["dh"], cols, q["h"], cols, 0.1, 5 + k, 6, None, q["mean"],
                q["rstd"], q["dres"], cols, q["dx"], cols, q["dw"], None, 0, q["work"], n) == 0

        alone = []
        for k in range(2):
            torch.cuda.synchronize()
            call(handles[k], data[k], k)
            torch.cuda.synchronize()
            alone.append([data[k][o].clone() for o in ("dres", "dx", "dw")])
            for o in ("dres", "dx", "dw"):
                data[k][o].zero_()
        torch.cuda.synchronize()
        for _ in range(10):
            for k in range(2):
                call(handles[k], data[k], k)
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(data[k][o], a) for o, a in zip(("dres", "dx", "dw"), alone[k]))
    finally:
        for h in handles:
            lib.dn_close(h)


def test_refusals_reach_the_caller(eng):
    """A refused call names its reason and writes nothing."""
    from decide_amd import InvalidArgument, Unsupported

    x, y = Matrix(4, 64, "fp32", torch.zeros(4, 64)), Matrix(4, 64, "fp32")
    with pytest.raises(InvalidArgument, match="y overlaps|x overlaps"):
        eng.layer_norm_device("fp32", "fp32", 4, 64, x.at, 64, None, None, EPS, x.at + 64, 64)
    with pytest.raises(InvalidArgument, match="eps"):
        eng.layer_norm_device("fp32", "fp32", 4, 64, x.at, 64, None, None, 0.0, y.at, 64)
    with pytest.raises(Unsupported, match="not built"):
        eng.layer_norm_device("bf16", "fp32", 4, 64, x.at, 64, None, None, EPS, y.at, 64)
    with pytest.raises(InvalidArgument, match="probability"):
        eng.dropout_device("fp32", "fp32", 4, 64, x.at, 64, None, 0, 1.5, 1, 2, y.at, 64)
    with pytest.raises(InvalidArgument, match="x is NULL"):
        eng.dropout_device("fp32", "fp32", 4, 64, None, 64, None, 0, 0.5, 1, 2, y.at, 64)
    for rows, cols in ((2 ** 63 - 1, 64), (2 ** 31, 64), (600, 2 ** 31 - 1), (2 ** 63 - 1, 2 ** 31 - 1)):
        for dw in (None, y.at):
            with pytest.raises(Unsupported, match="at most"):
                eng.layer_norm_backward_device("fp32", "fp32", rows, cols, x.at, 64, x.at, 64, None, x.at, x.at, y.at,
                                               64, dw)
    for rows, cols in ((-1, 64), (600, -1), (-2 ** 63, -2 ** 31)):
        with pytest.raises(InvalidArgument, match="rows or columns"):
            eng.layer_norm_backward_device("fp32", "fp32", rows, cols, x.at, 64, x.at, 64, None, x.at, x.at, y.at, 64)
    torch.cuda.synchronize()
    assert bool((y.buf == GUARD).all())
