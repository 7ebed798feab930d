"""The launches of the block-scaled product (host code, no GPU): every output
belongs to one tile of one launch, every block of K to one part, no launch is
empty or past its limits, and the workspace holds the parts."""
import ctypes
import os
import random
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

SMALL11, SMALL22, SMALL42, TILE, WIDE = range(5)
CAP = 4096


class Fp8Launch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("kind", "m", "M", "n", "N", "tiles_m", "tiles_n", "each", "parts")]


def load(so):
    lib = ctypes.CDLL(so)
    i64 = ctypes.c_int64
    lib.launches.argtypes = [i64] * 3 + [ctypes.c_int] * 3 + [ctypes.POINTER(Fp8Launch), ctypes.c_int]
    lib.work_floats.argtypes, lib.work_floats.restype = [i64] * 3, i64
    lib.takes_direct.argtypes = [ctypes.c_uint64, i64, i64, i64]
    return lib


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("needs g++")
    so = str(tmp_path_factory.mktemp("fp8") / "fp8_plan.so")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", so,
                    os.path.join(ROOT, "tests", "fp8_plan.cpp")], check=True)
    return so


@pytest.fixture(scope="module")
def plan(built):
    return load(built)


def launches(plan, M, N, K, exact=False, square=True, direct=True):
    out = (Fp8Launch * CAP)()
    n = plan.launches(M, N, K, exact, square, direct, out, CAP)
    assert n >= 0, (M, N, K)
    return out[:n]


def check(plan, M, N, K, exact=False, square=True, direct=True):
    got, what = launches(plan, M, N, K, exact, square, direct), (M, N, K, exact, square, direct)
    blocks, bands = -(-K // 128), {}
    for l in got:
        bm, bn = plan.tile_rows(l.kind), plan.tile_cols(l.kind)
        assert l.M > 0 and l.N > 0 and l.tiles_m == -(-l.M // bm) and l.tiles_n == -(-l.N // bn), what
        threads = 256 if l.kind in (TILE, WIDE) else 512
        assert l.tiles_m * l.tiles_n * l.parts * threads < 1 << 32 and l.parts < 1 << 16, what
        # Every part has blocks of its own, the last one what is left.
        assert l.parts == 1 and l.each >= blocks or (l.parts - 1) * l.each < blocks <= l.parts * l.each, what
        assert l.kind == TILE or l.parts == 1, what
        # The 128 x 256 kernel is built for a 16-bit C, square scales and direct loads.
        assert l.kind != WIDE or not exact and square and direct, what
        # A launch's scales of 128 x 128 blocks begin at a block.
        assert l.n % 128 == 0, what
        if l.parts > 1:
            assert len(got) == 1 and l.parts * M * N <= plan.work_floats(M, N, K), what
        bands.setdefault((l.n, l.N), []).append((l.m, l.M))
    at = 0
    for n, count in sorted(bands):
        assert n == at, what
        at += count
        row = 0
        for m, rows in sorted(bands[n, count]):
            assert m == row, what
            row += rows
        assert row == M, what
    assert at == N, what
    return [l.kind for l in got]


def test_tall_products_of_few_columns(built):
    """512 tiles of 128 rows and more, 1 to 32 columns, 16 blocks of K and more: nothing is left beside the last
    column of tiles. In a process of its own, which a division by zero would end."""
    code = ("import sys; sys.path[:0] = [%r, %r]\nimport test_fp8_plan as t\nplan = t.load(%r)\n"
            "for M in (65408, 65409, 65536, 70000, 1 << 20):\n"
            "    for N in (1, 2, 8, 16, 17, 31, 32, 33, 256, 257, 288):\n"
            "        for K in (1920, 1921, 2048, 4096, 8192):\n"
            "            t.check(plan, M, N, K)\n" % (os.path.join(ROOT, "tests"), ROOT, built))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stderr[-2000:])


def test_a_last_column_of_tiles(plan):
    """A last column of up to 32 outputs that would cost a round of the CUs has a launch of its own."""
    assert check(plan, 4001, 4099, 8200) == [SMALL11, WIDE]
    assert check(plan, 8065, 2051, 2060) == [SMALL11, WIDE]
    assert check(plan, 4001, 4096 + 32, 8200) == [SMALL22, WIDE]
    assert check(plan, 4001, 4096 + 33, 8200) == [WIDE]
    assert check(plan, 4001, 4099, 1920) == [WIDE]
    assert check(plan, 32768, 2304, 768) == [WIDE]


def test_sizes(plan):
    rng = random.Random(1)

    def size(top):
        n = int(round(2 ** rng.uniform(0, top)))
        return max(1, rng.choice([n, n, -(-n // 128) * 128, -(-n // 128) * 128 + rng.choice([-1, 1, 16, 32])]))

    kinds = set()
    for _ in range(40000):
        M, N, K = size(20), size(16), rng.choice([0, size(16), size(16), size(23)])
        kinds.update(check(plan, M, N, K, rng.random() < 0.5, rng.random() < 0.7, rng.random() < 0.7))
    assert kinds == {SMALL11, SMALL22, SMALL42, TILE, WIDE}
    for M, N in ((2 ** 31 - 1, 1), (2 ** 31 - 1, 16), (2 ** 31 - 1, 300), (64, 2 ** 26), (1, 2 ** 26), (129, 2 ** 26)):
        for K in (0, 1, 128, 2048, 2 ** 31 - 1):
            for direct in (False, True):
                check(plan, M, N, K, direct=direct and K <= 1 << 23)


def test_direct_loads(plan):
    """Offsets inside a tile's buffers stay below 2^31 bytes: 256 rows of an operand, a scale's blocks."""
    top = 1 << 23
    assert plan.takes_direct(1 << 20, top, (1 << 13) - 1, top) and 255 * top + (top - 128) + 7 * 16 + 16 <= 1 << 31
    for p, ld, ld_scale, K in ((8, 16, 1, 128), (16, 24, 1, 128), (16, top + 16, 1, 128), (16, top, 1, top + 1),
                               (16, -16, 1, 128), (16, 1024, 1 << 28, 256), (16, 1024, (1 << 28) + 1, 256),
                               (16, top, 1 << 13, top)):
        assert not plan.takes_direct(p, ld, ld_scale, K), (p, ld, ld_scale, K)
    assert plan.takes_direct(16, 1024, 1 << 40, 128)  # a single block: its stride is any number
