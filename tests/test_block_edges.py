"""CPU checks of the training-block operators' arguments at the edges of their
types."""
import ctypes

import numpy as np
import pytest

import block_reference as ref
from test_block_ops import OK, checks  # noqa: F401


@pytest.mark.parametrize("halves,threshold", [(1, 0), (3, 2), (5, 2), (7, 4), (131069, 65534), (131071, 65536)])
def test_thresholds_between_two_steps(checks, halves, threshold):  # noqa: F811
    """p = an odd number of half steps of 2^-16: the even threshold, as the plain form rounds."""
    out, scale, p = (ctypes.c_uint32 * 5)(), ctypes.c_float(), halves / 131072
    assert checks.mask_of(ctypes.c_float(p), ctypes.c_uint64(1), ctypes.c_uint64(2), out, ctypes.byref(scale)) == OK
    assert out[0] == threshold == round(65536 * float(np.float32(p)))
    keep, want = ref.keep_scale(1, 8, p, 1, 2)
    assert scale.value == np.float32(want)


class Recorder:
    """A library whose calls keep their arguments and answer status."""

    def __init__(self, status):
        self.status, self.args = status, None

    def __getattr__(self, name):
        def call(*args):
            self.args = args
            return self.status
        return call


def block_calls(eng, rows, cols, ld):
    at, p = 1 << 20, 0.1
    yield lambda: eng.layer_norm_device("fp32", "fp32", rows, cols, at, ld, None, None, 1e-5, at, ld)
    yield lambda: eng.layer_norm_backward_device("fp32", "fp32", rows, cols, at, ld, at, ld, None, at, at, at, ld)
    yield lambda: eng.dropout_device("fp32", "fp32", rows, cols, at, ld, at, ld, p, 1, 2, at, ld)
    yield lambda: eng.dropout_add_norm_device("fp32", "fp32", "fp32", rows, cols, at, ld, at, ld, p, 1, 2, None, None,
                                              1e-5, at, ld, at, ld)
    yield lambda: eng.dropout_add_norm_backward_device("fp32", "fp32", "fp32", rows, cols, at, ld, at, ld, at, ld, p, 1, 2,
                                                       None, at, at, at, ld, at, ld)


@pytest.mark.parametrize("rows,cols,ld", [(2 ** 64 + 4, 64, 64), (4, 2 ** 32 + 64, 64), (4, 2 ** 64 + 64, 64),
                                          (4, 64, 2 ** 64 + 64), (-2 ** 64 + 4, 64, 64), (4, -2 ** 32 + 64, 64),
                                          (4, 64, -2 ** 64 + 64), (4, 64, 2 ** 63), (2 ** 63 - 1, 2 ** 31 - 1, 2 ** 63 - 1),
                                          (-1, -1, -1), (4, 64, 2 ** 40)])
def test_sizes_past_their_type_are_not_wrapped(monkeypatch, rows, cols, ld):
    """ctypes drops the bits that an integer's C type does not hold: 2^32 + 64 columns would be 64."""
    from decide_amd import nn

    eng = nn.Engine.__new__(nn.Engine)
    eng._h = None
    lib = Recorder(0)
    monkeypatch.setattr(nn, "lib", lib)

    def ends(v, bits):
        return max(-2 ** (bits - 1), min(v, 2 ** (bits - 1) - 1))

    for k, call in enumerate(block_calls(eng, rows, cols, ld)):
        call()
        passed = [v for v in lib.args if isinstance(v, int)]
        dropout = k == 2
        assert ends(rows, 64) in passed and ends(cols, 64 if dropout else 32) in passed
        strides = {0: 2, 1: 3, 2: 3, 3: 4, 4: 5}[k]
        assert passed.count(ends(ld, 64)) >= strides
        assert all(-2 ** 63 <= v < 2 ** 63 for v in passed)
    eng._h = None  # nothing to close


def test_workspace_of_sizes_past_their_type():
    from decide_amd.nn import Engine

    for rows, cols in ((2 ** 64 + 8, 8), (600, 2 ** 32 + 8), (600, -2 ** 32 + 8)):
        with pytest.raises(ValueError):
            Engine.norm_backward_workspace(rows, cols)
