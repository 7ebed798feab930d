"""The 8-bit operators on the GPU at the edges of their ranges: products of many
rows and few columns, and of a last column of tiles that has a launch of its
own; norms of zeros and of values near the ends of fp32. Bounds: fp8_reference.py."""
import numpy as np
import pytest
import torch

import block_reference as block
import fp8_reference as ref
from fp8_bounds import gemm_bound
from fp8_reference import U
from test_gpu_fp8_ops import (GEMM_TYPES, TYPES, Matrix, at, check_gemm, check_quantised, eng, f64,  # noqa: F401
                              ptr, scale_matrix, vec, within)

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
            if b == 1 and over[r]:
                continue
            stands, wanted = Q.f64()[r, at_columns] * scale.f64()[b, r], want[r, at_columns]
            assert np.abs(stands - wanted).max() <= np.abs(wanted).max() / 16
    if y:
        assert np.array_equal(np.isinf(Y.f64()), np.abs(want) > 3.5e38)


NAN8 = 0x7F  # a NaN of both 8-bit types


def poisoned(rng, rows, K, dtype, block_rows, lead, pad):
    """An operand and its scales, every byte beside them a NaN."""
    v = rng.standard_normal((rows, K)) * np.exp2(rng.integers(-6, 3, (rows, K)))
    m, s = Matrix(rows, K, dtype, lead=lead, pad=pad), scale_matrix(rows, K, block_rows, pad)
    m.bytes.fill_(NAN8)
    m.raw().copy_(torch.from_numpy(v).cuda().float().to(TYPES[dtype]).view(m.bits))
    s.bytes.view(torch.float32).fill_(float("nan"))
    s.view.copy_(torch.from_numpy(np.exp(rng.standard_normal(tuple(s.view.shape)) - 4)))
    return m, s


# A size for each kernel: 16 x 16, 32 x 32, 64 x 32, 128 x 128 and 128 x 256 outputs, and one split along K.
@pytest.mark.parametrize("M,N,K", [(M, N, K) for M, N in ((40, 50), (500, 400), (64, 8200), (1000, 900), (32641, 385))
                                   for K in (1, 15, 17, 129, 260, 1143)] + [(500, 400, 9001)])
def test_nothing_behind_a_row_takes_part(eng, M, N, K):  # noqa: F811
    """NaNs fill every byte that belongs to no element, of operands and scales. A NaN, an infinity and an infinite
    scale reach their own rows and columns and no others, in every type of C."""
    rng = np.random.default_rng(M + K)
    wide = M > 30000
    for k, ct in enumerate(("bf16", "fp16") if wide else ("bf16", "fp16", "fp32")):
        for lead, pad in ((0, -K % 16), (16, -K % 16 + 16), (1, 3)):
            if wide and lead != 16 * k:  # the 128 x 256 kernel takes aligned rows alone
                continue
            b_rows = 128 if wide or (lead + k) % 2 else 1
            a, sa = poisoned(rng, M, K, "e5m2", 1, lead, pad)
            b, sb = poisoned(rng, N, K, "e4m3", b_rows, lead, pad)
            a.raw()[5, K - 1], a.raw()[12, 0], b.raw()[7, K // 2] = 0x7C, 0x7E, 0x7F  # inf, NaN, NaN
            sa.view[0, 20] = float("inf")
            b.raw()[30] = 0
            c = Matrix(M, N, ct, lead=lead, pad=pad)
            work = torch.empty(max(1, eng.gemm_fp8_workspace(M, N, K)), dtype=torch.uint8, device="cuda")
            eng.gemm_fp8_device("e5m2", "e4m3", ct, M, N, K, *at(a), *at(sa), *at(b), b_rows, *at(sb), *at(c), False,
                                ptr(work), work.numel())
            what, got = (M, N, K, ct, lead, pad), c.f64()
            bad = np.zeros((M, N), bool)
            bad[[5, 12, 20]], bad[:, 7] = True, True
            assert np.array_equal(~np.isfinite(got), bad), what
            assert np.isnan(got[12]).all() and np.isnan(got[:, 7]).all() and np.isnan(got[[5, 20], 30]).all(), what
            assert c.untouched_outside(), what
            if not wide or K < 300:
                va, vs = a.f64(), sa.f64()
                va[[5, 12]], vs[0, 20] = 0.0, 0.0
                vb = b.f64()
                vb[7] = 0.0
                want = ref.gemm(va, vs, vb, sb.f64(), b_rows)[0]
                bound = gemm_bound(va, vs, vb, sb.f64(), b_rows, ("e5m2", "e4m3"), want, ct)
                within(np.where(bad, 0.0, got), np.where(bad, 0.0, want), bound, what)


@pytest.mark.parametrize("dtype", ["e4m3", "e5m2"])
@pytest.mark.parametrize("ct", ["fp32", "bf16", "fp16"])
def test_every_value_of_a_type(eng, dtype, ct):  # noqa: F811
    """Each 8-bit value, subnormals among them, times 1 (and times the least subnormal) is itself: it has at most four
    significant bits."""
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes = codes[torch.isfinite(codes.view(TYPES[dtype]).float())]
    n = codes.numel()
    for M in (n, 4 * n, 40 * n):
        a = codes.repeat(M // n)[:, None].expand(M, 128).contiguous()
        eye = torch.zeros(128, 128, dtype=torch.uint8, device="cuda")
        ones = torch.tensor([1.0], device="cuda").to(TYPES[dtype]).view(torch.uint8)
        for code, by in ((ones, 1.0), (torch.tensor([1], dtype=torch.uint8), 2.0 ** (-9 if dtype == "e4m3" else -16))):
            b = eye.clone()
            b.fill_diagonal_(int(code))
            sa, sb = torch.ones(1, M, device="cuda"), torch.full((1, 128), 1 / by, device="cuda")
            c = torch.empty(M, 128, dtype=TYPES[ct], device="cuda")
            work = torch.empty(max(1, eng.gemm_fp8_workspace(M, 128, 128)), dtype=torch.uint8, device="cuda")
            eng.gemm_fp8_device(dtype, dtype, ct, M, 128, 128, ptr(a), 128, ptr(sa), M, ptr(b), 128, 1, ptr(sb), 128,
                                ptr(c), 128, False, ptr(work), work.numel())
            want = codes.view(TYPES[dtype]).float().repeat(M // n)[:, None].expand(M, 128).to(TYPES[ct])
            assert torch.equal(c.float(), want.float()), (dtype, ct, M, by)


def test_more_rows_than_a_launch_takes(eng):  # noqa: F811
    """2^22 tiles of 128 rows and more, 2^20 workgroups of rows of the norm, 2^20 tiles of the quantiser."""
    M, K = (1 << 29) + 200, 16
    for lda, M in ((16, M), (1, M)):
        K = lda
        a = torch.full((M, lda), 0x38, dtype=torch.uint8, device="cuda")  # 1
        b, sb = torch.full((1, 16), 0x38, dtype=torch.uint8, device="cuda"), torch.ones(1, 1, device="cuda")
        sa = (torch.arange(M, dtype=torch.int32, device="cuda") % 251).float()  # at most 8 bits
        c = torch.zeros(M, dtype=torch.bfloat16, device="cuda")
        eng.gemm_fp8_device("e4m3", "e4m3", "bf16", M, 1, K, ptr(a), lda, ptr(sa), M, ptr(b), 16, 128, ptr(sb), 1,
                            ptr(c), 1)
        torch.cuda.synchronize()
        del a
        for r in range(0, M, 1 << 26):
            assert torch.equal(c[r:r + (1 << 26)].float(), sa[r:r + (1 << 26)] * K), (lda, r)
        del c, sa
    rows = (1 << 20) * 32 + 41
    x = torch.randn(rows, 8, device="cuda").bfloat16()
    q, s = torch.zeros(rows, 8, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    y = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    eng.add_rms_norm_device("bf16", "bf16", "bf16", "e4m3", rows, 8, ptr(x), 8, None, 0, None, 1e-5, None, 0, ptr(y), 8,
                            ptr(q), 8, ptr(s), rows)
    want = x.float() / (x.float().square().mean(1, keepdim=True) + 1e-5).sqrt()
    rel = 2.0 ** -8 + 2.0 ** -18  # bf16's rounding; fp32's of both sides
    assert bool(((y.float() - want).abs() <= want.abs() * rel + 2.0 ** -60).all())
    off = (q.view(torch.float8_e4m3fn).float() * s[:, None] - want).abs()
    assert bool((off <= want.abs() * (2.0 ** -4 + 2.0 ** -18) + s[:, None] * 2.0 ** -10).all())
    del x, y, q, s, want, off
    rows = (1 << 20) * 128 + 77
    x = torch.randn(rows, 1, device="cuda")
    q, qt = torch.zeros(rows, dtype=torch.uint8, device="cuda"), torch.zeros(rows, dtype=torch.uint8, device="cuda")
    nb = ref.blocks(rows)
    s, st = torch.zeros(nb, device="cuda"), torch.zeros(nb, device="cuda")
    eng.quantize_blocks_device("fp32", "e4m3", rows, 1, 128, ptr(x), 1, ptr(q), 1, ptr(s), nb, ptr(qt), rows, ptr(st),
                               1)
    assert torch.equal(q, qt) and torch.equal(s, st)
    tall = torch.zeros(nb * 128, device="cuda")
    tall[:rows] = x[:, 0]
    assert torch.equal(s, (tall.view(nb, 128).abs().amax(1).double() / 448).float())
    off = (q.view(torch.float8_e4m3fn).float() * s.repeat_interleave(128)[:rows] - x[:, 0]).abs()
    assert bool((off <= x[:, 0].abs() * (2.0 ** -4 + 2.0 ** -20) + s.repeat_interleave(128)[:rows] * 2.0 ** -10).all())


@pytest.mark.parametrize("types", GEMM_TYPES)
@pytest.mark.parametrize("M,N", [(300, 200), (1500, 776)])
def test_subnormal_operands(eng, types, M, N):  # noqa: F811
    """Products of subnormals by large values beside smaller ones: an fp32 C keeps fp32's bits, a 16-bit C the 8-bit
    instruction's, whose cut lies higher for them, and stays within 2^-7 (e5m2 alone: 2^-8) of the terms' magnitudes."""
    rng = np.random.default_rng(M)
    worst = 7 * 2.0 ** -10 if "e4m3" in types else 7 * 2.0 ** -11
    for K in (2, 3, 8, 9, 40, 300):
        pair = []
        for rows, t in ((M, types[0]), (N, types[1])):
            low, high = (-9, 8) if t == "e4m3" else (-16, 14)
            v = rng.choice([-1.0, 1.0], (rows, K)) * np.exp2(rng.uniform(low, high, (rows, K)))
            v[rng.random((rows, K)) < 0.5] *= 2.0 ** low  # half of them subnormal or zero
            s = scale_matrix(rows, K)
            s.view.copy_(torch.from_numpy(np.exp2(rng.integers(-8, -4, tuple(s.view.shape)) - (high - 8.0))))
            pair += [Matrix(rows, K, t, v, pad=-K % 16), s]
        a, sa, b, sb = pair
        want, terms = ref.gemm(a.f64(), sa.f64(), b.f64(), sb.f64(), 1)
        for ct in ("fp32", "bf16", "fp16"):
            c = Matrix(M, N, ct)
            work = torch.empty(max(1, eng.gemm_fp8_workspace(M, N, K)), dtype=torch.uint8, device="cuda")
            eng.gemm_fp8_device(*types, ct, M, N, K, *at(a), *at(sa), *at(b), 1, *at(sb), *at(c), False, ptr(work),
                                work.numel())
            within(c.f64(), want, gemm_bound(a.f64(), sa.f64(), b.f64(), sb.f64(), 1, types, want, ct), (K, ct))
            if ct != "fp32":  # as decide_hip.h says it
                e = (worst + 2.0 ** -15) * terms
                within(c.f64(), want, e + block.rounding(np.abs(want) + e, ct), (K, ct))
