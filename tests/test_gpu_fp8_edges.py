"""The 8-bit operators on the GPU at the edges of their ranges: products of many
rows and few columns, and of a last column of tiles that has a launch of its
own. Bounds: fp8_reference.py."""
import numpy as np
import pytest
import torch

import fp8_reference as ref
from test_gpu_fp8_ops import TYPES, Matrix, at, check_gemm, eng, f64, ptr, scale_matrix, within  # noqa: F401

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
