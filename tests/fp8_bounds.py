"""Error bound of the block-scaled product for every operand, subnormals too."""
import numpy as np

import block_reference as block
import fp8_reference as ref

LEAST_NORMAL = {"e4m3": 2.0 ** -6, "e5m2": 2.0 ** -14}


def lifted(v, dtype):
    """|v| with subnormals at the type's least normal value, whose exponent they have."""
    return np.where(v == 0, 0.0, np.maximum(np.abs(v), LEAST_NORMAL[dtype]))


def gemm_bound(a, sa, b, sb, b_rows, types, want, dtype):
    """fp32 C: as fp8_reference.gemm_bound. 16-bit C: the 8-bit matrix instruction cuts the products of eight at
    2^-13 of two to the largest sum of two operands' exponents, where a subnormal has the exponent of the least normal
    value: that power of two is at most the product of the lifted operands, and seven products may lose up to the cut
    each."""
    size = ref.gemm(a, sa, b, sb, b_rows)[1]
    e = (128 * 2 + 2 + ref.blocks(a.shape[1]) + 32 + 1) * ref.U * size
    if dtype != "fp32":
        e = e + 7 * 2.0 ** -13 * ref.gemm(lifted(a, types[0]), sa, lifted(b, types[1]), sb, b_rows)[1]
    return e + block.rounding(np.abs(want) + e, dtype)
