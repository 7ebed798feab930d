"""The 8-bit operators on the GPU (RMS norm with an 8-bit output and its
gradient, block quantiser, block-scaled product) against plain float64 forms,
at the sizes, types, strides and values where they can go wrong. Bounds:
fp8_reference.py."""
import numpy as np
import pytest
import torch

import block_reference as block
import fp8_reference as ref
from fp8_reference import U

pytestmark = pytest.mark.gpu

EPS = 1e-5
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn,
         "e5m2": torch.float8_e5m2}
BOUNDARY_TYPES = [("fp32", "fp32", "fp32"), ("bf16", "fp32", "bf16"), ("fp16", "fp32", "fp16"),
                  ("fp32", "fp32", "bf16"), ("fp32", "fp32", "fp16"), ("bf16", "bf16", "bf16"),
                  ("fp16", "fp16", "fp16")]
# Around every size where a kernel changes: vectors of 4 and 8 columns, blocks of 128, a wave's and a workgroup's rows.
COLS = [1, 2, 3, 4, 5, 7, 8, 9, 31, 33, 64, 100, 127, 128, 129, 255, 256, 257, 384, 513, 768, 1000, 1024, 1025, 1152,
        2047, 2048, 2304, 4099, 8192, 8193, 16383, 16384]
ROWS = [1, 2, 3, 5, 8, 9, 17, 33, 64, 65, 127, 129, 203]
GUARD = 0xA5


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
    """rows x cols of a type inside a larger buffer of guard bytes: `lead` elements before, row stride cols + pad."""

    def __init__(self, rows, cols, dtype, values=None, lead=0, pad=0):
        self.rows, self.cols, self.ld, self.dtype, self.lead = rows, cols, cols + pad, dtype, lead
        self.es = torch.empty((), dtype=TYPES[dtype]).element_size()
        # Nothing behind the last row's columns but 16 elements.
        self.n = lead + max(0, rows - 1) * self.ld + cols + 16
        self.bytes = torch.full((self.n * self.es,), GUARD, dtype=torch.uint8, device="cuda")
        self.view = self.bytes.view(TYPES[dtype]).as_strided((rows, cols), (self.ld, 1), lead)
        if values is not None:
            v = torch.as_tensor(values).cuda()
            if v.dtype != TYPES[dtype]:
                v = v.float().to(TYPES[dtype])
            self.raw().copy_(v.contiguous().view(self.bits))
        self.at = self.bytes.data_ptr() + lead * self.es

    @property
    def bits(self):
        return {1: torch.uint8, 2: torch.int16, 4: torch.int32}[self.es]

    def raw(self):
        return self.bytes.view(self.bits).as_strided((self.rows, self.cols), (self.ld, 1), self.lead)

    def f64(self):
        return self.raw().contiguous().view(TYPES[self.dtype]).float().double().cpu().numpy()

    def untouched_outside(self):
        b = self.bytes.clone()
        b.view(self.bits).as_strided((self.rows, self.cols), (self.ld, 1), self.lead).fill_(
            {1: 0xA5, 2: 0xA5A5 - 0x10000, 4: 0xA5A5A5A5 - 0x100000000}[self.es])
        return bool((b == GUARD).all())

    def untouched(self):
        return bool((self.bytes == GUARD).all())


def vec(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def f64(t):
    return None if t is None else t.double().cpu().numpy()


def at(m):
    return (None, 0) if m is None else (m.at, m.ld)


def ptr(t):
    return None if t is None else t.data_ptr()


def stream_values(rng, rows, cols):
    """A residual stream: rows of different scale and offset, a few large columns."""
    v = rng.standard_normal((rows, cols)) * (0.3 + rng.random((rows, 1)) * 3) + 0.3 * rng.standard_normal((rows, 1))
    v[:, ::13] *= 10
    return v


def within(got, want, bound, what):
    got = f64(got) if torch.is_tensor(got) else got
    assert got.shape == want.shape, what
    assert np.array_equal(np.isfinite(got), np.isfinite(want)), what
    fine = np.isfinite(want)
    off = np.abs(got - want)[fine] - np.broadcast_to(bound, want.shape)[fine]
    assert not (off > 0).any(), (what, float(off.max()))


def scale_matrix(rows, cols, block_rows=1, pad=0):
    return Matrix(ref.blocks(cols), rows if block_rows == 1 else ref.blocks(rows), "fp32", pad=pad)


def check_quantised(q, scale, want, off, dtype, what, block_rows=1):
    """Values and scales of an array that is known to `off` (0: exactly)."""
    rows, cols = want.shape
    s = ref.scales(want, dtype, block_rows)
    worst = ref.scales(np.broadcast_to(off, want.shape), dtype, block_rows) if np.any(off) else 0.0
    got = scale.f64()
    within(got, s, worst + U * s, ("scale", *what))
    each = ref.spread(got, rows, cols, block_rows)
    within(q.f64(), want / each, ref.quantised_bound(want / each, off / each, dtype), ("q", *what))
    assert q.untouched_outside() and scale.untouched_outside(), what


def check_rms(eng, rng, rows, cols, xt, st, yt, qt="e4m3", lead=0, pad=0, residual=True, weight=True, y=True, q=True):
    x = Matrix(rows, cols, xt, rng.standard_normal((rows, cols)) if residual else stream_values(rng, rows, cols), lead,
               pad)
    res = Matrix(rows, cols, st, stream_values(rng, rows, cols), lead, pad) if residual else None
    h = Matrix(rows, cols, st, None, lead, pad) if residual else None
    w = vec(1 + 0.2 * rng.standard_normal(cols)) if weight else None
    Y = Matrix(rows, cols, yt, None, lead, pad) if y else None
    Q = Matrix(rows, cols, qt, None, lead, pad) if q else None
    scale = scale_matrix(rows, cols, pad=pad) if q else None
    rstd = torch.full((rows + 1,), 7.25, device="cuda")
    eng.add_rms_norm_device(xt, st, yt, qt, rows, cols, *at(x), *at(res), ptr(w), EPS, *at(h), *at(Y), *at(Q),
                            *at(scale), ptr(rstd))
    what = (rows, cols, xt, st, yt, qt, pad, residual, weight)
    hv = x.f64()
    if residual:
        want = res.f64() + hv
        e = U * np.abs(want)
        within(h.f64(), want, e + block.rounding(np.abs(want) + e, st), ("h", *what))
        hv = h.f64()  # the norm is of h as it is stored
        assert h.untouched_outside()
    wanted, r = ref.rms(hv, f64(w), EPS)
    within(f64(rstd)[:rows], r, ref.RMS_REL * r, ("rstd", *what))
    assert float(rstd[rows]) == 7.25
    e = (ref.RMS_REL + 2 * U) * np.abs(wanted)
    if y:
        within(Y.f64(), wanted, e + block.rounding(np.abs(wanted) + e, yt), ("y", *what))
        assert Y.untouched_outside()
    if q:
        check_quantised(Q, scale, wanted, e, qt, what)


@pytest.mark.parametrize("cols", COLS)
def test_rms_sizes(eng, cols):
    rng = np.random.default_rng(cols)
    for k, (xt, st, yt) in enumerate(BOUNDARY_TYPES):
        rows = ROWS[(cols + 3 * k) % len(ROWS)]
        check_rms(eng, rng, rows, cols, xt, st, yt, weight=k != 1, y=k % 2 == 0, qt=("e4m3", "e5m2")[k % 3 == 2])
        check_rms(eng, rng, rows, cols, xt, st, yt, lead=1 + k, pad=(1, 3, 8, 5, 2, 16, 13)[k], q=k != 3,
                  y=k in (1, 3, 6), qt=("e4m3", "e5m2")[k % 2])
        if xt == st:
            check_rms(eng, rng, rows, cols, xt, st, yt, residual=False, lead=k, pad=k)


def test_rms_values(eng):
    """Rows of zeros give zeros with the least scale; a NaN makes its own row NaN and no other, an infinity rstd 0:
    zeros, and a NaN in its place; large and small rows keep their relative precision."""
    rng = np.random.default_rng(3)
    for cols in (1, 8, 100, 768, 2900, 9000):
        v = rng.standard_normal((9, cols))
        v[0], v[1], v[2] = 0.0, v[1] * 1e16, v[2] * 1e-20
        v[3, cols // 2], v[5, 0], v[6, cols - 1] = float("inf"), float("nan"), float("-inf")
        x, y, q = Matrix(9, cols, "fp32", v), Matrix(9, cols, "fp32"), Matrix(9, cols, "e4m3")
        scale, rstd = scale_matrix(9, cols), torch.empty(9, device="cuda")
        eng.add_rms_norm_device("fp32", "fp32", "fp32", "e4m3", 9, cols, *at(x), None, 0, None, EPS, None, 0, *at(y),
                                *at(q), *at(scale), ptr(rstd))
        got, q8, s = y.f64(), q.f64(), scale.f64()
        for r in range(9):
            bad = np.isnan(v[r]) | np.isinf(v[r]) | np.isnan(v[r]).any()
            assert np.array_equal(np.isnan(got[r]), bad) and np.array_equal(np.isnan(q8[r]), bad), (cols, r)
            assert r not in (3, 6) or float(rstd[r]) == 0 and not got[r][~bad].any() and not q8[r][~bad].any()
            assert np.isfinite(s[:, r]).all()
        assert (got[0] == 0).all() and (q8[0] == 0).all() and (s[:, 0] == np.float32(2.0 ** -100 / 448)).all()
        fine = [0, 1, 2, 4, 7, 8]
        want, r64 = ref.rms(x.f64()[fine], None, EPS)
        within(got[fine], want, (ref.RMS_REL + 3 * U) * np.abs(want) + 2.0 ** -149, cols)


def check_rms_grad(eng, rng, rows, cols, dt, st, xt, lead=0, pad=0, weight=True, dh=True, dx=True, dw=True,
                   accumulate=False, place=None):
    from decide_amd.nn import Engine

    h = Matrix(rows, cols, st, stream_values(rng, rows, cols), lead, pad)
    rstd = vec(ref.rms(h.f64(), None, EPS)[1])
    dy = Matrix(rows, cols, dt, 0.1 * rng.standard_normal((rows, cols)), lead, pad)
    DH = Matrix(rows, cols, st, 0.1 * rng.standard_normal((rows, cols)), lead, pad) if dh else None
    inputs = {"dy": dy, "h": h, "dh": DH}
    values = {k: m.f64() for k, m in inputs.items() if m}
    dres = inputs[place[0]] if place else Matrix(rows, cols, st, None, lead, pad)
    DX = (inputs[place[1]] if place and place[1] else Matrix(rows, cols, xt, None, lead, pad)) if dx else None
    w = vec(1 + 0.2 * rng.standard_normal(cols)) if weight else None
    size = Engine.norm_backward_workspace(rows, cols)
    work = torch.full((size // 4 + 8,), 7.25, device="cuda")
    gw = torch.full((cols + 1,), 0.5, device="cuda")
    eng.add_rms_norm_backward_device(dt, st, xt, rows, cols, *at(dy), *at(DH), *at(h), ptr(w), ptr(rstd), *at(dres),
                                     *at(DX), ptr(gw) if dw else None, accumulate, ptr(work), size)
    what = (rows, cols, dt, st, xt, pad, place)
    extra = values["dh"] if dh else 0.0
    dx64, dw64 = ref.rms_grad(values["dy"], values["h"], f64(w), f64(rstd))
    want = dx64 + extra
    bounds = [ref.rms_grad_bounds(values["dy"], values["h"], f64(w), f64(rstd), want, t, np.abs(extra))
              for t in (st, xt)]
    within(dres.f64(), want, bounds[0][0], ("dres", *what))
    if dx:
        within(DX.f64(), want, bounds[1][0], ("dx", *what))
    got, start = f64(gw), 0.5 if accumulate else 0.0
    assert got[cols] == 0.5
    if dw:
        within(got[:cols], dw64 + start, bounds[0][1] + U * (np.abs(dw64) + 1), ("dw", *what))
    else:
        assert (got == 0.5).all()
    for m in (*inputs.values(), dres, DX):
        assert m is None or m.untouched_outside()
    assert bool((work[size // 4:] == 7.25).all())


@pytest.mark.parametrize("cols", COLS)
def test_rms_gradient_sizes(eng, cols):
    rng = np.random.default_rng(cols + 1)
    for k, (dt, st, xt) in enumerate(BOUNDARY_TYPES):
        rows = ROWS[(cols + 5 * k) % len(ROWS)]
        check_rms_grad(eng, rng, rows, cols, dt, st, xt, weight=k != 1, dh=k != 2, dx=k != 5, accumulate=k % 2 == 0)
        check_rms_grad(eng, rng, rows, cols, dt, st, xt, lead=1 + k, pad=(1, 3, 8, 5, 2, 4, 16)[k], dx=k % 2 == 0,
                       dw=k != 4, accumulate=k % 2 == 1)


@pytest.mark.parametrize("rows", [257, 512, 513, 1000, 4097])
def test_rms_gradient_many_rows(eng, rows):
    rng = np.random.default_rng(rows)
    check_rms_grad(eng, rng, rows, 96, "bf16", "fp32", "bf16")
    check_rms_grad(eng, rng, rows, 768, "bf16", "fp32", "bf16", accumulate=True)
    check_rms_grad(eng, rng, rows, 2050, "fp16", "fp16", "fp16", dx=False)
    check_rms_grad(eng, rng, rows, 100, "fp32", "fp32", "bf16", dw=False)


@pytest.mark.parametrize("rows,cols", [(40, 768), (600, 768), (300, 4100), (520, 9000)])
def test_rms_gradient_in_place(eng, rows, cols):
    rng = np.random.default_rng(rows)
    for place in (("dh", "dy"), ("dy", "h"), ("h", None), ("h", "dh")):
        check_rms_grad(eng, rng, rows, cols, "fp32", "fp32", "fp32", place=place, accumulate=True)
        check_rms_grad(eng, rng, rows, cols, "bf16", "bf16", "bf16", place=place)
    check_rms_grad(eng, rng, rows, cols, "bf16", "fp32", "bf16", place=("dh", "dy"))


def check_quantise(eng, rng, rows, cols, xt, qt, block_rows, plain=True, transposed=False, lead=0, pad=0, values=None):
    x = Matrix(rows, cols, xt, 0.05 * stream_values(rng, rows, cols) if values is None else values, lead, pad)
    q = Matrix(rows, cols, qt, None, lead, pad) if plain else None
    scale = scale_matrix(rows, cols, block_rows, pad) if plain else None
    t = Matrix(cols, rows, qt, None, lead + 1, pad) if transposed else None
    scalet = scale_matrix(cols, rows, block_rows, pad) if transposed else None
    eng.quantize_blocks_device(xt, qt, rows, cols, block_rows, *at(x), *at(q), *at(scale), *at(t), *at(scalet))
    what = (rows, cols, xt, qt, block_rows, plain, transposed, lead, pad)
    v = x.f64()
    if plain:
        check_quantised(q, scale, v, 0.0, qt, what, block_rows)
    if transposed:
        check_quantised(t, scalet, v.T.copy(), 0.0, qt, ("transposed", *what), block_rows)
    return x, q, scale, t, scalet


@pytest.mark.parametrize("cols", [1, 3, 4, 7, 8, 9, 15, 100, 127, 128, 129, 257, 384, 1152, 2305, 4099])
def test_quantise_sizes(eng, cols):
    rng = np.random.default_rng(cols + 5)
    for k, xt in enumerate(("fp32", "bf16", "fp16") * 2):
        rows = (1, 127, 7, 128, 300, 16)[(cols + k) % 6]
        qt, r = ("e4m3", "e5m2")[k % 2], (1, 128)[(cols + k) // 3 % 2]
        check_quantise(eng, rng, rows, cols, xt, qt, 1)
        check_quantise(eng, rng, rows, cols, xt, qt, 1, lead=1 + k, pad=(1, 3, 8, 5, 2, 16)[k])
        check_quantise(eng, rng, rows, cols, xt, qt, r, transposed=True, lead=k, pad=(0, 1, 8, 3, 2, 5)[k])
        check_quantise(eng, rng, rows, cols, xt, qt, r, plain=False, transposed=True)
        check_quantise(eng, rng, rows, cols, xt, qt, 128, pad=k)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 127, 129, 255, 1000])
def test_quantise_rows(eng, rows):
    rng = np.random.default_rng(rows + 6)
    for k, cols in enumerate((1, 5, 8, 130, 768)):
        check_quantise(eng, rng, rows, cols, ("bf16", "fp32")[k % 2], "e4m3", (1, 128)[k // 2 % 2], transposed=True,
                       pad=k)


def test_quantise_values(eng):
    """Zeros, tiny and huge blocks, blocks of one value, subnormal results; an infinity marks its own blocks, a NaN
    its own element."""
    rng = np.random.default_rng(9)
    v = rng.standard_normal((260, 400))
    v[0], v[1], v[2], v[3] = 0.0, v[1] * 1e-35, v[2] * 1e35, -3.5
    v[4, 1:] *= 1e-4  # far below the block's largest: subnormal values, and zeros
    v[4, 0] = 10.0
    for qt in ("e4m3", "e5m2"):
        for r in (1, 128):
            check_quantise(eng, rng, 260, 400, "fp32", qt, r, transposed=True, values=v)
            check_quantise(eng, rng, 260, 400, "fp32", qt, r, values=v)
    v[5, 130], v[6, 0], v[131, 399] = float("inf"), float("nan"), float("-inf")
    for r in (1, 128):
        for transposed in (False, True):
            x, q, s, t, s2 = (Matrix(260, 400, "fp32", v), Matrix(260, 400, "e4m3"), scale_matrix(260, 400, r),
                              Matrix(400, 260, "e4m3"), scale_matrix(400, 260, r))
            eng.quantize_blocks_device("fp32", "e4m3", 260, 400, r, *at(x), *at(q), *at(s),
                                       *((*at(t), *at(s2)) if transposed else ()))
            for got, scale, a in ((q, s, v),) + (((t, s2, v.T),) if transposed else ()):
                with np.errstate(invalid="ignore"):
                    stands = got.f64() * ref.spread(scale.f64(), *a.shape, r)
                    inf = np.isinf(ref.spread(ref.scales(a, "e4m3", r), *a.shape, r))
                assert np.array_equal(np.isnan(stands), inf | np.isnan(a))


def test_quantise_more_blocks_than_a_launch_takes(eng):
    """2^20 workgroups of 16 (fp32: 8) blocks, rows of one block each."""
    rows = (1 << 20) * 8 + 37
    x = torch.randn(rows, 4, device="cuda")
    q = torch.zeros(rows, 4, dtype=torch.uint8, device="cuda")
    s = torch.zeros(rows, device="cuda")
    eng.quantize_blocks_device("fp32", "e4m3", rows, 4, 1, ptr(x), 4, ptr(q), 4, ptr(s), rows)
    assert torch.equal(s, (x.abs().amax(1).double() / 448).float())  # rounded once
    off = (q.view(torch.float8_e4m3fn).float() * s[:, None] - x).abs()
    assert bool((off <= x.abs() * (2.0 ** -4 + 2.0 ** -20) + s[:, None] * 2.0 ** -10).all())


GEMM_TYPES = [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")]


def operand(rng, rows, K, dtype, block_rows, lead=0, pad=0, scale_pad=0):
    """Values over the type's whole range with a scale a block of their own."""
    v = rng.standard_normal((rows, K)) * np.exp2(rng.integers(-6, 5, (rows, K)))
    m = Matrix(rows, K, dtype, v, lead, pad)
    s = scale_matrix(rows, K, block_rows, scale_pad)
    s.view.copy_(torch.from_numpy(np.exp(rng.standard_normal(tuple(s.view.shape)))))
    return m, s


def check_gemm(eng, rng, M, N, K, types=("e4m3", "e4m3"), ct="fp32", b_rows=128, lead=0, pad=0, accumulate=False,
               c_pad=0):
    from decide_amd.nn import Engine

    a, sa = operand(rng, M, K, types[0], 1, lead, pad, pad)
    b, sb = operand(rng, N, K, types[1], b_rows, lead, pad, pad)
    c0 = rng.standard_normal((M, N)) * 3
    c = Matrix(M, N, ct, c0, lead, c_pad)
    before = c.f64()
    size = Engine.gemm_fp8_workspace(M, N, K)
    work = torch.full((size // 4 + 8,), 7.25, device="cuda")
    eng.gemm_fp8_device(*types, ct, M, N, K, *at(a), *at(sa), *at(b), b_rows, *at(sb), *at(c), accumulate, ptr(work),
                        size)
    want, terms = ref.gemm(a.f64(), sa.f64(), b.f64(), sb.f64(), b_rows)
    if accumulate:
        want, terms = want + before, terms + np.abs(before)
    what = (M, N, K, types, ct, b_rows, lead, pad, accumulate)
    bound, got = ref.gemm_bound(terms, ref.blocks(K), want, ct), c.f64()
    if ct == "fp16":  # past 65,520, half a step above the largest value, lies infinity
        assert (np.isinf(got) | (np.abs(want) - bound < 65520)).all(), what
        over = np.isinf(got) & (np.abs(want) + bound >= 65520)
        assert (np.sign(got[over]) == np.sign(want[over])).all(), what
        got, want = np.where(over, 0.0, got), np.where(over, 0.0, want)
    within(got, want, bound, what)
    for m in (a, sa, b, sb, c):
        assert m.untouched_outside(), what
    assert bool((work[size // 4:] == 7.25).all()), what


# (M, N, K): around tiles, vectors and blocks; single rows, columns and elements; K inside, at and past a block.
GEMM_SIZES = [(1, 1, 1), (1, 1, 128), (1, 7, 129), (2, 3, 15), (3, 2, 17), (5, 300, 64), (16, 16, 128), (17, 33, 127),
              (1, 2304, 768), (8, 384, 1000), (31, 100, 256), (64, 768, 1152), (65, 129, 257), (127, 128, 2048),
              (128, 127, 300), (129, 257, 640), (256, 256, 384), (300, 70, 4100), (257, 511, 16), (500, 768, 768),
              (70, 1000, 8200), (1, 50, 20000), (33, 16, 12345), (640, 640, 128)]


@pytest.mark.parametrize("M,N,K", GEMM_SIZES)
def test_gemm_sizes(eng, M, N, K):
    rng = np.random.default_rng(M * 31 + N * 7 + K)
    up = -K % 16
    for k, ct in enumerate(("fp32", "bf16", "fp16")):
        check_gemm(eng, rng, M, N, K, GEMM_TYPES[(M + k) % 4], ct, pad=up, c_pad=-N % 8)
        check_gemm(eng, rng, M, N, K, GEMM_TYPES[(K + k) % 4], ct, b_rows=1, pad=up + 16 * k)
        check_gemm(eng, rng, M, N, K, GEMM_TYPES[(N + k) % 4], ct, b_rows=(1, 128)[k % 2], lead=1 + k, pad=(0, 3, 8)[k],
                   c_pad=(1, 0, 5)[k])
    check_gemm(eng, rng, M, N, K, b_rows=1, pad=up, accumulate=True)
    check_gemm(eng, rng, M, N, K, pad=up, lead=16, accumulate=True, c_pad=3)


@pytest.mark.parametrize("M,N,K", [(4001, 1155, 776), (1155, 384, 9000), (384, 1152, 4097), (1030, 1030, 1030)])
def test_gemm_larger(eng, M, N, K):
    rng = np.random.default_rng(M)
    for k, types in enumerate(GEMM_TYPES):
        check_gemm(eng, rng, M, N, K, types, ("fp32", "bf16", "fp16", "fp32")[k], b_rows=(1, 128)[k // 2], pad=-K % 16,
                   accumulate=k == 3)
    check_gemm(eng, rng, M, N, K, pad=1, lead=1)


@pytest.mark.parametrize("M,N,K", [(32641, 385, 300), (16385, 1024, 256), (8065, 2051, 2060)])
def test_gemm_many_tiles(eng, M, N, K):
    """512 tiles of 128 x 256 and more: K ending inside a block, whole blocks, a last column of tiles of its own."""
    rng = np.random.default_rng(N)
    for k, types in enumerate(GEMM_TYPES if N < 1000 else GEMM_TYPES[:1]):
        check_gemm(eng, rng, M, N, K, types, ("bf16", "fp16")[k % 2], pad=-K % 16 + 16 * (k % 2), c_pad=(0, 3, 8, 1)[k])


def test_gemm_empty(eng):
    """No rows, no columns: nothing happens. No depth: zeros, or C as it was."""
    rng = np.random.default_rng(1)
    c = Matrix(5, 9, "bf16", np.ones((5, 9)))
    for m, n in ((0, 9), (5, 0), (0, 0)):
        eng.gemm_fp8_device("e4m3", "e4m3", "bf16", m, n, 300, None, 0, None, 0, None, 0, 1, None, 0, None, 0)
    for ct, acc in (("bf16", False), ("fp32", False), ("fp32", True)):
        c = Matrix(5, 9, ct, np.ones((5, 9)), pad=2)
        eng.gemm_fp8_device("e4m3", "e4m3", ct, 5, 9, 0, None, 0, None, 0, None, 0, 1, None, 0, *at(c), acc)
        assert (c.f64() == (1.0 if acc else 0.0)).all() and c.untouched_outside()
    check_gemm(eng, rng, 5, 9, 1)


def test_gemm_values(eng):
    """A NaN, or an infinite scale, reaches its own row or column and no other; e5m2 infinities too. Rows and columns
    past the ends and the bytes behind a row's K take no part, whatever they hold."""
    rng = np.random.default_rng(2)
    for M, N, K in ((40, 50, 200), (300, 260, 1000), (4, 300, 520)):
        for b_rows in (1, 128):
            a, sa = operand(rng, M, K, "e5m2", 1, pad=-K % 16)
            b, sb = operand(rng, N, K, "e4m3", b_rows, pad=-K % 16)
            a.raw()[1, K - 1] = 0x7C  # +inf
            a.raw()[3, 0] = 0x7E  # NaN
            b.raw()[7, K // 2] = 0x7F  # NaN
            b.raw()[8] = 0  # inf * 0 too
            sa.view[0, 2] = float("inf")
            c = Matrix(M, N, "fp32")
            from decide_amd.nn import Engine

            work = torch.empty(max(1, Engine.gemm_fp8_workspace(M, N, K)), dtype=torch.uint8, device="cuda")
            eng.gemm_fp8_device("e5m2", "e4m3", "fp32", M, N, K, *at(a), *at(sa), *at(b), b_rows, *at(sb), *at(c), False,
                                ptr(work), work.numel())
            got = c.f64()
            bad = np.zeros((M, N), bool)
            bad[[1, 2, 3]] = True
            bad[:, 7] = True
            assert np.array_equal(~np.isfinite(got), bad), (M, N, K, b_rows)
            assert np.isnan(got[3]).all() and np.isnan(got[:, 7]).all() and np.isnan(got[1, 8])


def test_offsets_past_32_bits(eng):
    """Rows that lie more than 2^32 elements apart, in every array."""
    rng = np.random.default_rng(4)
    far = (1 << 32) + 48

    def apart(rows, cols, dtype, values=None, ld=far):
        m = Matrix.__new__(Matrix)
        m.rows, m.cols, m.ld, m.dtype, m.lead, m.es = rows, cols, ld, dtype, 0, TYPES[dtype].itemsize
        m.bytes = torch.empty(((rows - 1) * ld + cols + 16) * m.es, dtype=torch.uint8, device="cuda")
        m.at = m.bytes.data_ptr()
        if values is not None:
            m.raw().copy_(torch.as_tensor(values).cuda().float().to(TYPES[dtype]).view(m.bits))
        return m

    M, N, K = 3, 5, 260
    va, vb = rng.standard_normal((M, K)), rng.standard_normal((N, K))
    a, b = apart(M, K, "e4m3", va), apart(2, K, "e4m3", vb[:2])
    sa, sb = Matrix(3, M, "fp32", 1 + rng.random((3, M))), apart(3, 2, "fp32", 1 + rng.random((3, 2)), (1 << 30) + 8)
    c = apart(M, 2, "fp32", None, (1 << 30) + 8)
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    eng.gemm_fp8_device("e4m3", "e4m3", "fp32", M, 2, K, *at(a), *at(sa), *at(b), 1, *at(sb), *at(c), False, ptr(work),
                        work.numel())
    want, terms = ref.gemm(a.f64(), sa.f64(), b.f64(), sb.f64(), 1)
    within(c.f64(), want, ref.gemm_bound(terms, 3, want, "fp32"), "gemm")
    del b, c
    q, s = apart(M, K, "e4m3"), apart(3, M, "fp32", None, (1 << 30) + 8)
    x = apart(M, K, "bf16", va, (1 << 31) + 24)
    eng.quantize_blocks_device("bf16", "e4m3", M, K, 1, *at(x), *at(q), *at(s))
    first = q.f64(), s.f64()
    eng.add_rms_norm_device("bf16", "bf16", "bf16", "e4m3", M, K, *at(x), None, 0, None, EPS, None, 0, None, 0, *at(q),
                            *at(s))
    xv = x.f64()
    for (got, scale), want in ((first, xv), ((q.f64(), s.f64()), ref.rms(xv, None, EPS)[0])):
        each = ref.spread(scale, M, K)
        within(got, want / each, ref.quantised_bound(want / each, (ref.RMS_REL + 2 * U) * np.abs(want / each), "e4m3"), "q")
    # One array of more than 2^32 elements: its last rows.
    rows = (1 << 32) // 2048 + 200
    x = torch.empty(rows, 2048, dtype=torch.bfloat16, device="cuda")
    x[-200:] = torch.randn(200, 2048, device="cuda")
    q, s = torch.empty(rows, 2048, dtype=torch.uint8, device="cuda"), torch.empty(16, rows, device="cuda")
    x[:-200] = 0
    eng.quantize_blocks_device("bf16", "e4m3", rows, 2048, 1, ptr(x), 2048, ptr(q), 2048, ptr(s), rows)
    last = x[-200:].double().cpu().numpy()
    scale = s[:, -200:].double().cpu().numpy()
    within(scale, ref.scales(last, "e4m3"), U * scale, "scale")
    each = ref.spread(scale, 200, 2048)
    within(f64(q[-200:].view(torch.float8_e4m3fn).float()), last / each,
           ref.quantised_bound(last / each, 0.0, "e4m3"), "q")
    assert not q[:-200].any()


class Block:
    """A block's buffers: h, q = RMSNorm(res + x); z = q . Wq^T; and the gradients of h's inputs, the norm's weight and
    W from dz: everything a training step of an 8-bit projection calls, in order."""

    def __init__(self, rng, T, D, N):
        from decide_amd.nn import Engine

        self.T, self.D, self.N = T, D, N
        self.x = Matrix(T, D, "bf16", rng.standard_normal((T, D)))
        self.res = Matrix(T, D, "fp32", stream_values(rng, T, D))
        self.w = vec(1 + 0.2 * rng.standard_normal(D))
        self.W = Matrix(N, D, "fp32", 0.05 * rng.standard_normal((N, D)))
        self.dz = Matrix(T, N, "bf16", 0.1 * rng.standard_normal((T, N)))
        self.dh = Matrix(T, D, "fp32", 0.1 * rng.standard_normal((T, D)))

        def pair(rows, cols, dtype, block_rows=1):
            return Matrix(rows, cols, dtype, pad=-cols % 16), scale_matrix(rows, cols, block_rows)

        self.Wq, self.WqT = pair(N, D, "e4m3", 128), pair(D, N, "e4m3", 128)
        self.q, self.yT = pair(T, D, "e4m3"), pair(D, T, "e4m3")
        self.dzq, self.dzT = pair(T, N, "e5m2"), pair(N, T, "e5m2")
        self.h, self.y, self.z = Matrix(T, D, "fp32"), Matrix(T, D, "bf16"), Matrix(T, N, "bf16")
        self.dy, self.dres, self.dx = Matrix(T, D, "bf16"), Matrix(T, D, "fp32"), Matrix(T, D, "bf16")
        self.rstd, self.dw = torch.empty(T, device="cuda"), torch.zeros(D, device="cuda")
        self.dW = Matrix(N, D, "fp32", np.zeros((N, D)))
        self.work = torch.empty(max(1, Engine.norm_backward_workspace(T, D),
                                    *(Engine.gemm_fp8_workspace(*s) for s in ((T, N, D), (T, D, N), (N, D, T)))),
                                dtype=torch.uint8, device="cuda")

    def step(self, eng):
        T, D, N, room = self.T, self.D, self.N, (ptr(self.work), self.work.numel())
        eng.quantize_blocks_device("fp32", "e4m3", N, D, 128, *at(self.W), *at(self.Wq[0]), *at(self.Wq[1]),
                                   *at(self.WqT[0]), *at(self.WqT[1]))
        eng.add_rms_norm_device("bf16", "fp32", "bf16", "e4m3", T, D, *at(self.x), *at(self.res), ptr(self.w), EPS,
                                *at(self.h), *at(self.y), *at(self.q[0]), *at(self.q[1]), ptr(self.rstd))
        eng.gemm_fp8_device("e4m3", "e4m3", "bf16", T, N, D, *at(self.q[0]), *at(self.q[1]), *at(self.Wq[0]), 128,
                            *at(self.Wq[1]), *at(self.z), False, *room)
        eng.quantize_blocks_device("bf16", "e4m3", T, D, 1, *at(self.y), None, 0, None, 0, *at(self.yT[0]),
                                   *at(self.yT[1]))
        eng.quantize_blocks_device("bf16", "e5m2", T, N, 1, *at(self.dz), *at(self.dzq[0]), *at(self.dzq[1]),
                                   *at(self.dzT[0]), *at(self.dzT[1]))
        eng.gemm_fp8_device("e5m2", "e4m3", "bf16", T, D, N, *at(self.dzq[0]), *at(self.dzq[1]), *at(self.WqT[0]), 128,
                            *at(self.WqT[1]), *at(self.dy), False, *room)
        eng.gemm_fp8_device("e5m2", "e4m3", "fp32", N, D, T, *at(self.dzT[0]), *at(self.dzT[1]), *at(self.yT[0]), 1,
                            *at(self.yT[1]), *at(self.dW), True, *room)
        eng.add_rms_norm_backward_device("bf16", "fp32", "bf16", T, D, *at(self.dy), *at(self.dh), *at(self.h),
                                         ptr(self.w), ptr(self.rstd), *at(self.dres), *at(self.dx), ptr(self.dw), True,
                                         *room)

    def outputs(self):
        return [m.raw().clone() for m in (self.h, self.z, self.dy, self.dres, self.dx, self.dW)] + [self.dw.clone()]

    def check(self):
        T, D, N = self.T, self.D, self.N

        def value(pair, block_rows=1):
            v = pair[0].f64()
            return v * ref.spread(pair[1].f64(), *v.shape, block_rows)

        h, y64 = self.h.f64(), None
        w, rstd = f64(self.w), f64(self.rstd)
        y64, r64 = ref.rms(h, w, EPS)
        within(rstd, r64, ref.RMS_REL * r64, "rstd")
        e = (ref.RMS_REL + 2 * U) * np.abs(y64)
        check_quantised(*self.q, y64, e, "e4m3", "q")
        # Each product against its operands as they were quantised.
        Wq, WT = value(self.Wq, 128), value(self.WqT, 128)
        assert np.array_equal(Wq, WT.T)
        for got, a, b, t in ((self.z, value(self.q), Wq, "bf16"), (self.dy, value(self.dzq), WT, "bf16"),
                             (self.dW, value(self.dzT), value(self.yT), "fp32")):
            want = a @ b.T
            within(got.f64(), want, ref.gemm_bound(np.abs(a) @ np.abs(b).T, ref.blocks(a.shape[1]), want, t), "product")
        dx, dw = ref.rms_grad(self.dy.f64(), h, w, rstd)
        want = dx + self.dh.f64()
        e, ew = ref.rms_grad_bounds(self.dy.f64(), h, w, rstd, want, "fp32", np.abs(self.dh.f64()))
        within(self.dres.f64(), want, e, "dres")
        within(f64(self.dw), dw, ew + U * np.abs(dw), "dw")
        # And the whole against the unquantised step: what 8 bits cost. An e4m3 operand is off by 2^-4 of an element at
        # most (subnormals apart), e5m2 by 2^-3, so a product of N(0, 1)-like terms by less than their sum's norm
        # times the two together.
        dz, Wf = self.dz.f64(), self.W.f64()
        for got, want, rel in ((self.z, y64 @ Wf.T, 2.0 ** -4 * 2), (self.dy, dz @ Wf, 2.0 ** -4 + 2.0 ** -3),
                               (self.dW, dz.T @ y64, 2.0 ** -4 + 2.0 ** -3)):
            off = got.f64() - want
            assert np.linalg.norm(off) < rel * np.linalg.norm(want), "the 8-bit step"


@pytest.mark.parametrize("T,D,N", [(40, 384, 384), (203, 768, 1152), (1000, 768, 2304), (131, 1000, 300)])
def test_block_step(eng, T, D, N):
    b = Block(np.random.default_rng(T), T, D, N)
    b.step(eng)
    b.check()


def test_equal_calls_give_equal_bits(eng):
    b = Block(np.random.default_rng(5), 600, 768, 384)
    b.step(eng)
    first = b.outputs()
    b.dW.raw().zero_()
    b.dw.zero_()
    b.step(eng)
    assert all(torch.equal(x, y) for x, y in zip(first, b.outputs()))


def test_captured_step(eng):
    """The whole step in a graph: every replay equals the eager step on the same inputs."""
    rng = np.random.default_rng(6)
    b = Block(rng, 600, 768, 384)
    side = torch.cuda.Stream()
    eng.set_stream(side.cuda_stream)
    try:
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            b.step(eng)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.step(eng)
        for k in range(4):
            b.x.raw().copy_(Matrix(600, 768, "bf16", rng.standard_normal((600, 768))).raw())
            b.dW.raw().zero_()
            b.dw.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                b.step(eng)
            torch.cuda.synchronize()
            want = b.outputs()
            b.dW.raw().zero_()
            b.dw.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(want, b.outputs())), k
        b.check()
    finally:
        eng.set_stream(torch.cuda.current_stream().cuda_stream)


def test_two_contexts_at_once(eng):
    """Steps of two contexts on two streams, each with buffers and a workspace of its own."""
    from decide_amd import Engine

    other = Engine(eng.cfg, None, precision="fp32")
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    blocks = [Block(np.random.default_rng(7 + i), 700 + i, 768, 384) for i in range(2)]
    try:
        torch.cuda.synchronize()
        for e, s in zip((eng, other), streams):
            e.set_stream(s.cuda_stream)
        for e, b in zip((eng, other), blocks):
            b.step(e)
        torch.cuda.synchronize()
        for b in blocks:
            b.check()
    finally:
        eng.set_stream(torch.cuda.current_stream().cuda_stream)
        other.close()


def test_refusals_reach_the_caller(eng):
    from decide_amd.native import InvalidArgument, Unsupported

    t = torch.empty(4096, device="cuda")
    p = t.data_ptr()
    with pytest.raises(InvalidArgument, match="overlaps"):
        eng.quantize_blocks_device("fp32", "e4m3", 2, 8, 1, p, 8, p + 4, 8, p + 1024, 2)
    with pytest.raises(Unsupported):
        eng.gemm_fp8_device("e4m3", "e4m3", "bf16", 2, 2, 16, p, 16, p + 64, 2, p + 128, 16, 1, p + 256, 2, p + 512, 2,
                            True)
    with pytest.raises(InvalidArgument, match="NULL"):
        eng.add_rms_norm_device("fp32", "fp32", "fp32", "e4m3", 2, 8, p, 8, None, 0, None, EPS, None, 0, None, 0, None, 0,
                                None, 0)
    for big in (2 ** 31, 2 ** 63, 2 ** 70):
        with pytest.raises((InvalidArgument, Unsupported)):
            eng.gemm_fp8_device("e4m3", "e4m3", "bf16", big, 2, 16, p, 16, p, 2, p, 16, 1, p, 2, p + 512, 2)
        with pytest.raises((InvalidArgument, Unsupported)):
            eng.quantize_blocks_device("fp32", "e4m3", 2, 8, big, p, 8, p + 128, 8, p + 1024, 2)
    with pytest.raises(KeyError):
        eng.gemm_fp8_device("bf16", "e4m3", "bf16", 2, 2, 16, p, 16, p, 2, p, 16, 1, p, 2, p + 512, 2)
