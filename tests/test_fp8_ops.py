"""CPU checks of the 8-bit operators: every refusal of a call's arguments (the
host code that runs before any kernel), and the plain forms that the kernels
are tested against."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import fp8_reference as ref
from conftest import ROOT

OK, INVALID, UNSUPPORTED = 0, 2, 5
FP32, BF16, FP16, E4M3, E5M2 = 0, 1, 2, 3, 4
ARRAYS = ("x", "res", "h", "y", "q", "qt", "scale", "scalet", "w", "rstd", "dy", "dh", "dres", "dx", "dw", "work", "A",
          "B", "sa", "sb", "C")
STRIDES = ("ldx", "ldres", "ldh", "ldy", "ldq", "ldqt", "ldscale", "ldscalet", "lddy", "lddh", "lddres", "lddx", "ldA",
           "ldB", "ldsa", "ldsb", "ldC")


class Fp8Call(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int) for n in ("x_type", "stream_type", "y_type", "q_type", "b_type", "block_rows",
                                             "accumulate")]
                + [("eps", ctypes.c_float)] + [(n, ctypes.c_int64) for n in ("rows", "cols", "depth")]
                + [(n, ctypes.c_size_t) for n in ARRAYS] + [(n, ctypes.c_int64) for n in STRIDES]
                + [("work_floats", ctypes.c_int64), ("work_bytes", ctypes.c_int64)])


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("needs g++")
    so = str(tmp_path_factory.mktemp("fp8") / "fp8_check.so")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", so,
                    os.path.join(ROOT, "tests", "fp8_check.cpp")], check=True)
    return ctypes.CDLL(so)


# Calls of 40 rows, 200 columns (two blocks) and a depth of 300 (three), each array in a megabyte of its own.
OPS = ("rms", "rms_grad", "quantise", "gemm")
R, C, K = 40, 200, 300
# op -> {array: (rows, columns, element size)}
SHAPES = {"rms": {"x": (R, C, 4), "res": (R, C, 4), "h": (R, C, 4), "y": (R, C, 4), "q": (R, C, 1),
                  "scale": (2, R, 4), "w": (1, C, 4), "rstd": (1, R, 4)},
          "rms_grad": {"dy": (R, C, 4), "dh": (R, C, 4), "h": (R, C, 4), "w": (1, C, 4), "rstd": (1, R, 4),
                       "dres": (R, C, 4), "dx": (R, C, 4), "dw": (1, C, 4), "work": (1, 480, 4)},
          "quantise": {"x": (R, C, 4), "q": (R, C, 1), "scale": (2, R, 4), "qt": (C, R, 1), "scalet": (1, C, 4)},
          "gemm": {"A": (R, K, 1), "sa": (3, R, 4), "B": (C, K, 1), "sb": (3, C, 4), "C": (R, C, 4),
                   "work": (1, 480, 4)}}
REQUIRED = {"rms": ("x", "h", "scale"), "rms_grad": ("dy", "h", "rstd", "dres", "work"),
            "quantise": ("x", "scale", "scalet"), "gemm": ("A", "sa", "B", "sb", "C", "work")}
OUT = {"rms": ("h", "y", "q", "scale", "rstd"), "rms_grad": ("dres", "dx", "dw", "work"),
       "quantise": ("q", "scale", "qt", "scalet"), "gemm": ("C", "work")}
# Outputs that may be an input's very array.
IN_PLACE = {"rms": {"h": ("x", "res"), "y": ("x", "res")}, "rms_grad": {"dres": ("dy", "dh", "h"), "dx": ("dy", "dh", "h")},
            "quantise": {}, "gemm": {}}
AT = {n: (i + 1) << 20 for i, n in enumerate(ARRAYS)}


def call(checks, op, **kw):
    c = Fp8Call(x_type=FP32, stream_type=FP32, y_type=FP32, q_type=E4M3, b_type=E5M2, block_rows=1, accumulate=0,
                eps=1e-5, rows=R, cols=C, depth=K, work_floats=480, work_bytes=1920)
    for n in ARRAYS:
        setattr(c, n, AT[n])
    for n in STRIDES:
        shape = SHAPES[op].get(n[2:])
        setattr(c, n, shape[1] if shape else 0)
    for k, v in kw.items():
        setattr(c, k, v)
    msg = ctypes.create_string_buffer(300)
    rc = getattr(checks, "check_" + op)(ctypes.byref(c), msg, 300)
    assert bool(msg.value) == (rc != OK)
    return rc, msg.value.decode()


@pytest.mark.parametrize("op", OPS)
def test_ordinary_calls_pass(checks, op):
    assert call(checks, op) == (OK, "")
    assert call(checks, op, rows=0, **{n: 0 for n in ARRAYS if n != "work"})[0] == OK
    for n in SHAPES[op]:
        if n not in REQUIRED[op]:
            assert call(checks, op, **{n: 0})[0] == OK, n
    strides = {n: -7 for n in STRIDES if n[2:] in SHAPES[op] and n not in ("ldscale", "ldsa", "ldsb", "ldqt", "ldB")}
    if op != "gemm":
        assert call(checks, op, rows=1, **strides, **({"ldqt": 1} if op == "quantise" else {}))[0] == OK
    if op in ("quantise", "gemm"):
        assert call(checks, op, cols=0, **{n: 0 for n in ARRAYS if n != "work"})[0] == OK
        assert call(checks, op, block_rows=128)[0] == OK
    if op == "gemm":
        assert call(checks, op, depth=0, A=0, B=0, sa=0, sb=0)[0] == OK
        assert call(checks, op, work_floats=0, work_bytes=0, work=0)[0] == OK
    if op == "rms_grad":
        assert call(checks, op, dw=0, work=0, work_bytes=0)[0] == OK
    if op == "rms":
        assert call(checks, op, res=0, h=0)[0] == OK
        assert call(checks, op, q=0, scale=0)[0] == OK
        assert call(checks, op, y=0, y_type=99)[0] == OK
    if op == "rms_grad":
        assert call(checks, op, dx=0, y_type=99)[0] == OK


@pytest.mark.parametrize("op", OPS)
def test_null_misaligned_and_narrow_arrays(checks, op):
    for n in REQUIRED[op]:
        rc, msg = call(checks, op, **{n: 0})
        assert rc == INVALID and "is NULL" in msg, n
    for n, (rows, cols, es) in SHAPES[op].items():
        if es > 1:
            rc, msg = call(checks, op, **{n: AT[n] + 2})
            assert rc == INVALID and "not aligned" in msg, n
        else:
            assert call(checks, op, **{n: AT[n] + 1})[0] == OK, n
        if rows > 1:
            for bad in (cols - 1, 0, -cols):
                rc, msg = call(checks, op, **{"ld" + n: bad})
                assert rc == INVALID and "row stride" in msg, n
            assert call(checks, op, **{"ld" + n: 1 << 60})[0] == INVALID
            assert call(checks, op, **{"ld" + n: cols + 1})[0] == OK


def test_nothing_to_write(checks):
    rc, msg = call(checks, "rms", y=0, q=0)
    assert rc == INVALID and "both NULL" in msg
    rc, msg = call(checks, "quantise", qt=0, q=0)
    assert rc == INVALID and "both NULL" in msg


def test_scales_have_the_blocks_sizes(checks):
    """128 x 128 blocks have a scale each: fewer rows of scales side by side."""
    assert call(checks, "quantise", block_rows=128, ldscale=1)[0] == OK
    assert call(checks, "quantise", block_rows=1, ldscale=R - 1)[0] == INVALID
    assert call(checks, "gemm", block_rows=128, ldsb=2)[0] == OK
    assert call(checks, "gemm", block_rows=128, ldsb=1)[0] == INVALID
    assert call(checks, "gemm", block_rows=1, ldsb=C - 1)[0] == INVALID


@pytest.mark.parametrize("op", OPS)
def test_sizes(checks, op):
    assert call(checks, op, rows=-1)[0] == INVALID
    assert call(checks, op, rows=1 << 31)[0] == UNSUPPORTED
    if op in ("quantise", "gemm"):
        assert call(checks, op, cols=-1)[0] == INVALID
        assert call(checks, op, cols=1 << 31)[0] == UNSUPPORTED
        for bad in (0, 2, 64, 127, 256, -128):
            assert call(checks, op, block_rows=bad)[0] == INVALID
    else:
        assert call(checks, op, cols=0)[0] == INVALID
        assert call(checks, op, cols=16385)[0] == UNSUPPORTED
    if op == "gemm":
        assert call(checks, op, depth=-1)[0] == INVALID
        assert call(checks, op, depth=1 << 31)[0] == UNSUPPORTED


def test_values(checks):
    for eps in (0.0, -1e-5, float("nan"), float("inf")):
        rc, msg = call(checks, "rms", eps=eps)
        assert rc == INVALID and "eps" in msg
    for op in ("rms_grad", "gemm"):
        rc, msg = call(checks, op, work_bytes=1919)
        assert rc == INVALID and "workspace" in msg


def test_types(checks):
    types = (FP32, BF16, FP16)

    def boundary(a, s, b):
        return (a == b == s) if s != FP32 else (a == b or (a == FP32 and b != FP32))

    for a in types:
        for s in types:
            for b in types:
                for op in ("rms", "rms_grad"):
                    assert call(checks, op, x_type=a, stream_type=s, y_type=b)[0] == (OK if boundary(a, s, b)
                                                                                      else UNSUPPORTED), (op, a, s, b)
                want = OK if a == s and boundary(a, s, b) else UNSUPPORTED
                assert call(checks, "rms", x_type=a, stream_type=s, y_type=b, res=0)[0] == want
            assert call(checks, "rms", x_type=a, stream_type=s, y=0)[0] == (OK if boundary(a, s, a) else UNSUPPORTED)
    for t in (E4M3, E5M2, 5, -1):
        for op in ("rms", "rms_grad", "quantise"):
            assert call(checks, op, x_type=t, stream_type=t, y_type=t)[0] == INVALID
        assert call(checks, "gemm", y_type=t)[0] == INVALID
    for t in (FP32, BF16, FP16, 5, -1):
        for op in ("rms", "quantise", "gemm"):
            assert call(checks, op, q_type=t)[0] == INVALID
        assert call(checks, "gemm", b_type=t)[0] == INVALID
    for t in types:
        assert call(checks, "gemm", y_type=t)[0] == OK
        assert call(checks, "gemm", y_type=t, accumulate=1)[0] == (OK if t == FP32 else UNSUPPORTED)


@pytest.mark.parametrize("op", OPS)
def test_overlaps(checks, op):
    """An output may be an input's very array where the element sizes agree; every other overlap with an output is
    refused."""
    shapes = SHAPES[op]
    for o in OUT[op]:
        for other in shapes:
            if other == o:
                continue
            size = shapes[other][0] * shapes[other][1] * shapes[other][2]
            fine = other in IN_PLACE[op].get(o, ())
            rc, msg = call(checks, op, **{o: AT[other]})
            assert rc == (OK if fine else INVALID), (o, other, msg)
            for delta in (8, size - 4):
                rc, msg = call(checks, op, **{o: AT[other] + delta})
                assert rc == INVALID and "overlaps" in msg, (o, other, delta)
            assert call(checks, op, **{o: AT[other] + (size + 3) // 4 * 4})[0] == OK, (o, other)


def test_existing_operators_refuse_8_bit_types(checks):
    from decide_amd import native

    assert set(native.PRECISIONS) == {"fp32", "bf16", "fp16"}
    assert native.FP8_TYPES == {"e4m3": 3, "e5m2": 4}


def test_null_context_and_workspaces():
    from decide_amd import native
    from decide_amd.nn import Engine

    lib = native.lib
    assert lib.dn_add_rms_norm_device(None, 0, 0, 0, 3, 1, 8, None, 8, None, 8, None, 1e-5, None, 8, None, 8, None, 8,
                                      None, 1, None) == INVALID
    assert lib.dn_add_rms_norm_backward_device(None, 0, 0, 0, 1, 8, None, 8, None, 8, None, 8, None, None, None, 8,
                                               None, 8, None, 0, None, 0) == INVALID
    assert lib.dn_quantize_blocks_device(None, 0, 3, 1, 8, 1, None, 8, None, 8, None, 1, None, 1, None, 8) == INVALID
    assert lib.dn_gemm_fp8_device(None, 3, 3, 0, 1, 1, 8, None, 8, None, 1, None, 8, 1, None, 1, None, 1, 0, None,
                                  0) == INVALID
    for m, n, k in ((0, 0, 0), (1, 1, 1), (1, 2304, 768), (2304, 768, 12288), (32768, 768, 2304), (100, 100, 100000),
                    (2 ** 31 - 1, 1, 1)):
        assert 0 <= Engine.gemm_fp8_workspace(m, n, k) <= 1 << 30
        assert Engine.gemm_fp8_workspace(m, n, k) % 4 == 0
    for bad in ((-1, 1, 1), (1, -1, 1), (1, 1, -1), (2 ** 31, 1, 1), (1, 2 ** 31, 1), (1, 1, 2 ** 70)):
        with pytest.raises(ValueError):
            Engine.gemm_fp8_workspace(*bad)


@pytest.mark.parametrize("dtype,t", [("e4m3", torch.float8_e4m3fn), ("e5m2", torch.float8_e5m2)])
def test_half_steps(dtype, t):
    """rounding8 is half of the distance to the type's neighbours: every value of the type, moved by a little less
    than that, rounds back to itself."""
    v = torch.arange(128, dtype=torch.uint8).view(t).double().numpy()
    v = v[np.isfinite(v)]
    assert v.max() == ref.MOST[dtype]
    for w in (v[:-1] + np.diff(v) * 0.499, v[1:] - np.diff(v) * 0.499):
        r = torch.from_numpy(w).float().to(t).double().numpy()
        assert (np.abs(r - w) <= ref.rounding8(w, dtype)).all()
        assert (np.abs(r - w) >= 0.49 * np.diff(v)).all()


def test_plain_forms():
    """The scales' layout and the product of blocks, element by element."""
    rng = np.random.default_rng(1)
    v = rng.standard_normal((130, 257))
    s1, s2 = ref.scales(v, "e4m3"), ref.scales(v, "e4m3", 128)
    assert s1.shape == (3, 130) and s2.shape == (3, 2)
    assert s1[1, 5] == np.abs(v[5, 128:256]).max() / 448 and s1[2, 129] == np.abs(v[129, 256]) / 448
    assert s2[1, 0] == np.abs(v[:128, 128:256]).max() / 448 and s2[2, 1] == np.abs(v[128:, 256:]).max() / 448
    assert ref.spread(s1, 130, 257)[5, 200] == s1[1, 5] and ref.spread(s2, 130, 257, 128)[129, 10] == s2[0, 1]
    b = rng.standard_normal((5, 257))
    got, size = ref.gemm(v, s1, b, ref.scales(b, "e4m3"), 1)
    want = sum(v[7, k] * s1[k // 128, 7] * b[3, k] * ref.scales(b, "e4m3")[k // 128, 3] for k in range(257))
    assert abs(got[7, 3] - want) <= 1e-12 * size[7, 3]
