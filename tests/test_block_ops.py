"""CPU checks of the training-block operators: the generator against its
published answers, the mask's definition, and every refusal of a call's
arguments (the host code that runs before any kernel)."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

import block_reference as ref
from conftest import ROOT

OK, INVALID, UNSUPPORTED = 0, 2, 5
FP32, BF16, FP16 = 0, 1, 2


class NormCall(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int) for n in ("a_type", "stream_type", "b_type", "cols")]
                + [("rows", ctypes.c_int64), ("p", ctypes.c_float), ("eps", ctypes.c_float)]
                + [(n, ctypes.c_size_t) for n in ("x", "res", "h", "y", "dy", "dh", "dres", "dx", "w", "b", "mean",
                                                  "rstd", "dw", "db", "work")]
                + [(n, ctypes.c_int64) for n in ("ldx", "ldres", "ldh", "ldy", "lddy", "lddh", "lddres", "lddx",
                                                 "drop_cols", "work_floats", "work_bytes")])


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("needs g++")
    so = str(tmp_path_factory.mktemp("block") / "block_check.so")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", so,
                    os.path.join(ROOT, "tests", "block_check.cpp")], check=True)
    return ctypes.CDLL(so)


# Arrays of 40 rows and 24 columns, each in a megabyte of its own.
NAMES = ("x", "res", "h", "y", "dy", "dh", "dres", "dx", "w", "b", "mean", "rstd", "dw", "db", "work")
OPS = ("norm", "boundary", "norm_grad", "boundary_grad", "dropout")
USES = {"norm": ("x", "y", "w", "b", "mean", "rstd"),
        "boundary": ("x", "res", "h", "y", "w", "b", "mean", "rstd"),
        "norm_grad": ("dy", "h", "w", "mean", "rstd", "dres", "dw", "db", "work"),
        "boundary_grad": ("dy", "dh", "h", "w", "mean", "rstd", "dres", "dx", "dw", "db", "work"),
        "dropout": ("x", "res", "y")}
REQUIRED = {"norm": ("x", "y"), "boundary": ("x", "res", "h", "y"),
            "norm_grad": ("dy", "h", "mean", "rstd", "dres", "work"),
            "boundary_grad": ("dy", "h", "mean", "rstd", "dres", "dx", "work"), "dropout": ("x", "y")}
OUT = ("h", "y", "dres", "dx")  # matrices that calls write (h: the forward's)


def call(checks, op, **kw):
    c = NormCall(a_type=FP32, stream_type=FP32, b_type=FP32, cols=24, rows=40, p=0.1, eps=1e-5, drop_cols=24,
                 work_floats=480, work_bytes=1920)
    for i, n in enumerate(NAMES):
        setattr(c, n, (i + 1) << 20)
    for n in ("ldx", "ldres", "ldh", "ldy", "lddy", "lddh", "lddres", "lddx"):
        setattr(c, n, 24)
    for k, v in kw.items():
        setattr(c, k, v)
    msg = ctypes.create_string_buffer(300)
    rc = getattr(checks, "check_" + op)(ctypes.byref(c), msg, 300)
    assert bool(msg.value) == (rc != OK)
    return rc, msg.value.decode()


def test_philox_known_answers():
    """The published known answers of Philox4x32-10 (zeros, ones, digits of pi)."""
    for ctr, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in ref.philox(*ctr, *key)) == want


def test_mask_is_a_function_of_row_and_column():
    """A mask's element depends on seed, offset, row and column alone, and as many are kept as p says:
    the share of 65,536 independent draws lies within 5 standard deviations."""
    keep, scale = ref.keep_scale(256, 256, 0.25, 7 << 40, 9 << 33)
    assert scale == 65536 / (65536 - 16384)
    assert abs(keep.mean() - 0.75) < 5 * (0.25 * 0.75 / 65536) ** 0.5
    wide, _ = ref.keep_scale(256, 261, 0.25, 7 << 40, 9 << 33)
    assert np.array_equal(wide[:, :256], keep)
    other, _ = ref.keep_scale(256, 256, 0.25, 7 << 40, (9 << 33) + 1)
    assert 0.3 < (other == keep).mean() < 0.75


@pytest.mark.parametrize("p,threshold", [(0.0, 0), (1e-6, 0), (0.1, 6554), (0.5, 32768), (1.0, 65536)])
def test_mask_words(checks, p, threshold):
    out, scale = (ctypes.c_uint32 * 5)(), ctypes.c_float()
    seed, offset = 0x0123456789ABCDEF, 0xFEDCBA9876543210
    rc = checks.mask_of(ctypes.c_float(p), ctypes.c_uint64(seed), ctypes.c_uint64(offset), out, ctypes.byref(scale))
    assert rc == OK
    assert list(out) == [threshold, seed & 0xFFFFFFFF, seed >> 32, offset & 0xFFFFFFFF, offset >> 32]
    want = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    assert scale.value == np.float32(want)


@pytest.mark.parametrize("op", OPS)
def test_ordinary_calls_pass(checks, op):
    assert call(checks, op) == (OK, "")
    assert call(checks, op, rows=0, x=0, y=0, h=0, dy=0, dres=0, dx=0, res=0)[0] == OK
    optional = [n for n in USES[op] if n not in REQUIRED[op]]
    assert call(checks, op, **{n: 0 for n in optional})[0] == OK
    if "dw" in USES[op]:
        assert call(checks, op, dw=0, db=0, work=0, work_bytes=0)[0] == OK  # no sums, no workspace
    assert call(checks, op, rows=1, ldx=0, ldres=0, ldh=0, ldy=0, lddy=0, lddh=0, lddres=0, lddx=0)[0] == OK
    if op == "dropout":
        assert call(checks, op, drop_cols=0, x=0, y=0)[0] == OK


@pytest.mark.parametrize("op", OPS)
def test_null_misaligned_and_narrow_arrays(checks, op):
    for n in REQUIRED[op]:
        rc, msg = call(checks, op, **{n: 0})
        assert rc == INVALID and "is NULL" in msg, n
    for n in USES[op]:
        rc, msg = call(checks, op, **{n: (NAMES.index(n) + 1 << 20) + 2})
        assert rc == INVALID and "not aligned" in msg, n
        ld = "ld" + n
        if hasattr(NormCall, ld):
            for bad in (23, 0, -24):
                rc, msg = call(checks, op, **{ld: bad})
                assert rc == INVALID and "row stride" in msg, n
            assert call(checks, op, **{ld: 1 << 60})[0] == INVALID


@pytest.mark.parametrize("op", OPS)
def test_a_single_row_has_any_stride(checks, op):
    for ld in (0, 1, 23, -1, -(1 << 63), (1 << 63) - 1):
        strides = {n: ld for n in dir(NormCall) if n.startswith("ld")}
        assert call(checks, op, rows=1, **strides)[0] == OK
        # A gradient's h is an input: two inputs may overlap.
        inputs = ("h",) if op.endswith("grad") else ()
        for o in [n for n in USES[op] if hasattr(NormCall, "ld" + n) and n in OUT and n not in inputs]:
            other = next(n for n in USES[op] if n != o)
            assert call(checks, op, rows=1, **strides, **{o: (NAMES.index(other) + 1 << 20) + 4})[0] == INVALID


@pytest.mark.parametrize("op", OPS)
def test_sizes(checks, op):
    assert call(checks, op, rows=-1)[0] == INVALID
    assert call(checks, op, rows=1 << 31)[0] == UNSUPPORTED
    if op == "dropout":
        assert call(checks, op, drop_cols=-1)[0] == INVALID
        assert call(checks, op, rows=1, drop_cols=(1 << 34) - 7)[0] == UNSUPPORTED
        return
    assert call(checks, op, cols=0)[0] == INVALID
    assert call(checks, op, cols=16385)[0] == UNSUPPORTED


@pytest.mark.parametrize("op", OPS)
def test_values(checks, op):
    nan = float("nan")
    if op in ("boundary", "boundary_grad", "dropout"):
        for p in (-0.01, 1.01, nan, float("inf")):
            rc, msg = call(checks, op, p=p)
            assert rc == INVALID and "probability" in msg
    if op in ("norm", "boundary"):
        for eps in (0.0, -1e-5, nan, float("inf")):
            rc, msg = call(checks, op, eps=eps)
            assert rc == INVALID and "eps" in msg
    if op.endswith("grad"):
        rc, msg = call(checks, op, work_bytes=1919)
        assert rc == INVALID and "workspace" in msg


def test_types(checks):
    built = {
        # (x or dy, stream or x, y or dx)
        "norm": lambda a, s, b: s == FP32 or s == b,
        "norm_grad": lambda a, s, b: s == FP32 or s == a,
        "boundary": lambda a, s, b: (a == b == s) if s != FP32 else (a == b or (a == FP32 and b != FP32)),
        "dropout": lambda a, s, b: a == b or FP32 in (a, b)}
    built["boundary_grad"] = built["boundary"]
    for op in OPS:
        for a in (FP32, BF16, FP16):
            for s in (FP32, BF16, FP16):
                for b in (FP32, BF16, FP16):
                    rc, msg = call(checks, op, a_type=a, stream_type=s, b_type=b)
                    want = OK if built[op](a, s, b) else UNSUPPORTED
                    assert rc == want, (op, a, s, b, msg)
        assert call(checks, op, a_type=3, stream_type=3, b_type=3)[0] == INVALID
        assert call(checks, op, a_type=-1, stream_type=-1, b_type=-1)[0] == INVALID


@pytest.mark.parametrize("op", OPS)
def test_overlaps(checks, op):
    """An output may be an input's very array; every other overlap with an output is refused."""
    uses = USES[op]
    outs = [n for n in uses if n in OUT and not (n == "h" and op.endswith("grad"))]
    ins = [n for n in uses if n not in outs and hasattr(NormCall, "ld" + n)]
    at = {n: NAMES.index(n) + 1 << 20 for n in NAMES}
    size = 40 * 24 * 4
    for o in outs:
        for i in ins:
            assert call(checks, op, **{o: at[i]})[0] == OK, (o, i)
            for delta in (4, -4, size - 4, 4 - size):
                rc, msg = call(checks, op, **{o: at[i] + delta})
                assert rc == INVALID and "overlaps" in msg, (o, i, delta)
            for delta in (size, -size):
                assert call(checks, op, **{o: at[i] + delta})[0] == OK
            # the same address with another stride is another array
            rc, msg = call(checks, op, **{o: at[i], "ld" + o: 25})
            assert rc == INVALID and "overlaps" in msg
            # columns of one buffer side by side, in either order; one column shared is refused
            both = {"ld" + o: 64, "ld" + i: 64}
            for delta, want in ((24, OK), (40, OK), (-24, OK), (-40, OK), (23, INVALID), (41, INVALID), (-23, INVALID),
                                (64 * 3 + 30, OK), (-64 * 3 - 30, OK), (64, INVALID)):
                assert call(checks, op, **both, **{o: at[i] + 4 * delta})[0] == want, (o, i, delta)
        for o2 in outs:
            if o2 != o:
                assert call(checks, op, **{o: at[o2]})[0] == INVALID  # two outputs in one array
        for v in [n for n in uses if n in ("w", "b", "mean", "rstd", "dw", "db", "work")]:
            assert call(checks, op, **{v: at[o] + 8})[0] == INVALID, (o, v)
    for v in ("dw", "db", "work"):
        if v in uses:
            assert call(checks, op, **{v: at["w"]})[0] == INVALID
            assert call(checks, op, **{v: at["rstd"]})[0] == INVALID


def test_exported_and_null_context():
    from decide_amd import native

    lib = native.lib
    z = (None,) * 30
    assert lib.dn_layer_norm_device(None, 0, 0, 1, 8, None, 8, None, None, 1e-5, None, 8, None, None) == INVALID
    assert lib.dn_layer_norm_backward_device(None, 0, 0, 1, 8, None, 8, None, 8, *z[:4], 8, None, None, 0, None,
                                             0) == INVALID
    assert lib.dn_dropout_device(None, 0, 0, 1, 8, None, 8, None, 8, 0.1, 1, 2, None, 8) == INVALID
    assert lib.dn_dropout_add_norm_device(None, 0, 0, 0, 1, 8, None, 8, None, 8, 0.1, 1, 2, None, None, 1e-5, None, 8,
                                          None, 8, None, None) == INVALID
    assert lib.dn_dropout_add_norm_backward_device(None, 0, 0, 0, 1, 8, None, 8, None, 8, None, 8, 0.1, 1, 2, None,
                                                   None, None, None, 8, None, 8, None, None, 0, None, 0) == INVALID


def test_workspace_sizes():
    from decide_amd.nn import Engine

    for rows, cols in ((0, 1), (1, 1), (7, 768), (12288, 768), (2 ** 31 - 1, 16384)):
        n = Engine.norm_backward_workspace(rows, cols)
        assert 0 <= n <= 768 * 2 * cols * 4 and n % 4 == 0
    for rows, cols in ((-1, 8), (8, 0), (8, 16385), (2 ** 31, 8)):
        with pytest.raises(ValueError):
            Engine.norm_backward_workspace(rows, cols)
