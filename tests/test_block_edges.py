"""CPU checks of the training-block operators' arguments at the edges of their
types."""
import ctypes

import numpy as np
import pytest

import block_reference as ref
from test_block_ops import OK, checks  # noqa: F401


@pytest.mark.parametrize("halves,threshold", [(1, 0), (2, 1), (3, 2), (5, 2), (7, 4), (131069, 65534), (131071, 65536)])
def test_thresholds_between_two_steps(checks, halves, threshold):  # noqa: F811
    """p = an odd number of half steps of 2^-16: the even threshold, as the plain form rounds."""
    out, scale, p = (ctypes.c_uint32 * 5)(), ctypes.c_float(), halves / 131072
    assert checks.mask_of(ctypes.c_float(p), ctypes.c_uint64(1), ctypes.c_uint64(2), out, ctypes.byref(scale)) == OK
    assert out[0] == threshold == round(65536 * float(np.float32(p)))
    keep, want = ref.keep_scale(1, 8, p, 1, 2)
    assert scale.value == np.float32(want)
