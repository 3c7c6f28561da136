"""The rules that the 8-bit products' kernels go by, without a GPU: which bytes a
load of a tile's rows may read."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("f8") / "f8_rules.so")
    subprocess.run(["/opt/rocm/bin/amdclang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "f8_rules_stub.cpp"),
                    "-Wl,-Bsymbolic", "-o", out], check=True, capture_output=True)
    return ctypes.CDLL(out)


def readable(nbytes, scalar, at):
    """Whether a lane at `at` reads memory: the range check of a raw buffer, which takes the scalar offset from the bytes
    in unsigned arithmetic."""
    return at < (nbytes - scalar) % 2 ** 32


@pytest.mark.parametrize("most", [16, 32, 64])  # rows of one load: of a stream's wave, of four and eight waves of a tile
@pytest.mark.parametrize("rows,pitch", [(1, 128), (7, 256), (33, 640), (200, 384), (2 ** 12, 2 ** 21)])
def test_loads_stay_in_the_matrix(rules, most, rows, pitch):
    """Rows that are there are read whole, at their column block, and what lies past the matrix's end is not: for loads
    partly and wholly behind it, and for a workgroup past its last tile (none left, wherever it stands)."""
    last, to = pitch // 128 - 1, (ctypes.c_int * 2)()
    for first in sorted({0, 1, most - 1, most, max(rows - most, 0), max(rows - 1, 0), rows, rows + 1, rows + 255}):
        for left in {rows - first, min(rows - first, 0) - 5, min(rows - first, 0)}:
            rules.rule_piece(first, left, rows, most, to)
            base, nbytes = to[0], to[1] * pitch
            assert 0 <= base and base + to[1] <= rows
            assert left < 1 or base == first
            for block in {0, last // 2, last}:
                for row in range(most):
                    for column in (0, 16, 112):
                        at = row * pitch + column
                        if readable(nbytes, block * 128, at):
                            assert base * pitch + block * 128 + at + 16 <= rows * pitch
                            assert row < max(left, 1)
                        else:
                            assert row >= left
    assert readable(0, 128, 0)  # what a scalar offset does to a buffer of no rows
