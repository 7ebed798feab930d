"""The 8-bit operators on the GPU at the edges of their ranges: products of many
rows and few columns, and of a last column of tiles that has a launch of its
own; norms of zeros and of values near the ends of fp32. Bounds: fp8_reference.py."""
import numpy as np
import pytest
import torch

import fp8_reference as ref
from fp8_reference import U
from test_gpu_fp8_ops import (TYPES, Matrix, at, check_gemm, check_quantised, eng, f64, ptr, scale_matrix,  # noqa: F401
                              vec, within)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [1, 8, 16, 17, 32, 33])
def test_tall_products_of_few_columns(eng, N):  # noqa: F811
    """65,537 rows (513 tiles of 128) and a head's or a router's few columns."""
    M, K, types = 65537, 2064, ("e4m3", "e4m3")
    gen = torch.Generator(device="cuda").manual_seed(N)
    a, b = Matrix(M, K, types[0], pad=-K % 16), Matrix(N, K, types[1], pad=-K % 16)
    sa, sb = scale_matrix(M, K), scale_matrix(N, K, 128)
    for m in (a, b):
        v = torch.randn(m.rows, K, generator=gen, device="cuda")
        m.raw().copy_(v.to(TYPES[m.dtype]).view(m.bits))
    for s in (sa, sb):
        s.view.copy_(torch.randn(s.view.shape, generator=gen, device="cuda").exp() / 16)  # sums in fp16's range
    blocks, spread = ref.blocks(K), lambda s, rows: s.view.repeat_interleave(128, 0)[:K].t()[:rows]
    a64 = a.raw().contiguous().view(TYPES[types[0]]).double() * spread(sa, M).double()
    b64 = b.raw().contiguous().view(TYPES[types[1]]).double() * spread(sb, 1).double()
    want, size = f64(a64 @ b64.t().contiguous()), f64(a64.abs() @ b64.t().abs().contiguous())
    for ct, c_pad in (("bf16", 0), ("fp16", 3)):
        c = Matrix(M, N, ct, pad=c_pad)
        assert eng.gemm_fp8_workspace(M, N, K) == 0
        eng.gemm_fp8_device(*types, ct, M, N, K, *at(a), *at(sa), *at(b), 128, *at(sb), *at(c))
        within(c.f64(), want, ref.gemm_bound(size, blocks, want, ct), (M, N, K, ct))
        assert c.untouched_outside()


@pytest.mark.parametrize("M,N,K", [(8065, 2048 + 24, 2060), (8065, 2048 + 32, 2064), (16257, 1024 + 17, 1936)])
def test_last_columns_of_17_to_32(eng, M, N, K):  # noqa: F811
    """A last column of tiles of 17 to 32 outputs, in a launch of its own."""
    rng = np.random.default_rng(N)
    check_gemm(eng, rng, M, N, K, ("e5m2", "e4m3"), "bf16", pad=-K % 16, c_pad=3)


def norm_of(eng, v, eps, qt, w=None, y=True):  # noqa: F811
    """(y, q, scale, rstd) of the RMS norm of rows of fp32 values, and y and rstd in 64 bits."""
    rows, cols = v.shape
    x, Y = Matrix(rows, cols, "fp32", v), Matrix(rows, cols, "fp32")
    Q, scale, rstd = Matrix(rows, cols, qt), scale_matrix(rows, cols), torch.empty(rows, device="cuda")
    w = None if w is None else vec(w)
    eng.add_rms_norm_device("fp32", "fp32", "fp32", qt, rows, cols, *at(x), None, 0, ptr(w), eps, None, 0,
                            *(at(Y) if y else (None, 0)), *at(Q), *at(scale), ptr(rstd))
    return Y, Q, scale, rstd, *ref.rms(x.f64(), f64(w), float(np.float32(eps)))


@pytest.mark.parametrize("eps", [1e-5, 4e-8, 1e-8, 1e-12, 1e-20, 1e-30, 1e-38])
@pytest.mark.parametrize("qt", ["e4m3", "e5m2"])
def test_norm_of_zeros_and_tiny_values(eng, qt, eps):  # noqa: F811
    """Rows and blocks of zeros give zeros with the least scale for every eps, whatever rstd = eps^-0.5 is; values so
    small that rstd lifts them, or does not, above the least magnitude of a block keep their relative precision."""
    rng = np.random.default_rng(11)
    for cols in (1, 7, 100, 128, 300, 768, 2900, 9000):
        v = rng.standard_normal((12, cols))
        v[0] = 0.0
        for r, size in enumerate((1e-20, 1e-25, 1e-30, 1e-33, 1e-34, 1e-35, 1e-36, 2.0 ** -100)):
            v[1 + r] *= size
        v[9, cols // 2:] = 0.0
        v[10, cols // 2:] *= 1e-34
        v[11, :cols // 2] *= 1e-37
        Y, Q, scale, rstd, want, r64 = norm_of(eng, v, eps, qt)
        # Squares below fp32's smallest normal lose up to half of its smallest step each, eps's sum one more.
        rel = ref.RMS_REL + 2 * 2.0 ** -149 / np.float32(eps)
        within(f64(rstd), r64, rel * r64, ("rstd", cols))
        e = (rel + 2 * U) * np.abs(want) + 2.0 ** -149
        within(Y.f64(), want, e + U * np.abs(want), ("y", cols))
        check_quantised(Q, scale, want, e, qt, (cols, eps))
        zeros = Q.f64()[0], Q.f64()[9, cols // 2:]
        assert not zeros[0].any() and not zeros[1].any()
        least = np.float32(2.0 ** -100) / np.float32(ref.MOST[qt])
        assert (scale.f64()[:, 0] == least).all()
        assert cols < 512 or (scale.f64()[-1, 9] == least).all()


@pytest.mark.parametrize("y", [True, False])
def test_norm_weights_near_the_ends(eng, y):  # noqa: F811
    """y = (h rstd) w: where h w alone would leave fp32's range, above or below, y does not; a block whose y is
    infinite has an infinite scale, its finite rows and blocks do not see it."""
    rng = np.random.default_rng(12)
    for cols in (1, 7, 100, 300, 768, 2900, 9000):
        for size, weight, eps in ((1e6, 1e34, 1e-5), (1e16, 1e30, 1e-5), (1e-25, 1e-18, 1e-38), (1e-24, 1e-20, 1e-38)):
            v = rng.standard_normal((6, cols)) * size
            w = weight * (0.5 + rng.random(cols))
            Y, Q, scale, rstd, want, r64 = norm_of(eng, v, eps, "e4m3", w, y)
            rel = ref.RMS_REL + 2 * 2.0 ** -149 / np.float32(eps)
            within(f64(rstd), r64, rel * r64, ("rstd", cols))
            # A row's smallest elements times rstd may be below fp32's normal range: half of its step, times w.
            e = (rel + 2 * U) * np.abs(want) + 2.0 ** -150 * (1 + w)
            if y:
                within(Y.f64(), want, e + U * np.abs(want), ("y", cols, size))
            check_quantised(Q, scale, want, e, "e4m3", (cols, size))
    # y past fp32's range in one block: infinite there, in y and in its scale.
    w = np.ones(300)
    w[130] = 1e38
    v = rng.standard_normal((5, 300))
    v[:, 130], v[4, 130] = 10.0, 0.0
    Y, Q, scale, rstd, want, r64 = norm_of(eng, v, 1e-5, "e4m3", w, y)
    over = want[:, 130] > 3.5e38
    assert over[:4].all() and not over[4]
    assert np.array_equal(np.isinf(scale.f64()), np.array([[False] * 5, list(over), [False] * 5]))
    for b, at_columns in enumerate((slice(0, 128), slice(128, 256), slice(256, 300))):
        for r in range(5):
            stands = Q.f64()[r, at_columns] * np.float64(scale.f64()[b, r]) if not (b == 1 and over[r]) else None
            assert stands is None or np.abs(stands - want[r, at_columns]).max() <= np.abs(want[r, at_columns]).max() / 16
    if y:
        assert np.array_equal(np.isinf(Y.f64()), np.abs(want) > 3.5e38)
