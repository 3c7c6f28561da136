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


def piece(rules, left, most, pitch, block):
    b, o = ctypes.c_uint32(), ctypes.c_uint32()
    rules.rule_piece(left, most, pitch, block, ctypes.byref(b), ctypes.byref(o))
    return b.value, o.value


def readable(bytes_, offset, at):
    """Whether a lane at `at` reads memory: the range check of a raw buffer, which takes the scalar offset from the bytes
    in unsigned arithmetic."""
    return at < (bytes_ - offset) % 2 ** 32


@pytest.mark.parametrize("most", [8, 16, 32, 64])  # rows that one load brings: of a stream's wave 8 and 16, of a tile 32 and 64
@pytest.mark.parametrize("pitch", [128, 256, 640, 2 ** 21])
def test_pieces_stay_in_the_matrix(rules, most, pitch):
    """Rows that are there are read whole, at their column block; none past the matrix's end, where a tile is
    partly or wholly behind it too."""
    last = pitch // 128 - 1
    for left in (-2 ** 21, -300, -1, 0, 1, 2, most - 1, most, most + 1, 300, 2 ** 21):
        for block in {0, last // 2, last}:
            bytes_, offset = piece(rules, left, most, pitch, block)
            assert bytes_ <= max(left, 0) * pitch
            for row in range(most):
                for column in (0, 16, 112):
                    at = row * pitch + column
                    assert readable(bytes_, offset, at) == (row < left), (left, block, row)
                    if row < left:
                        assert offset + at == row * pitch + block * 128 + column
                        assert offset + at + 16 <= bytes_
    # a buffer of no rows at any other offset would be read
    assert readable(0, 128, 0) and not readable(0, 0, 0)
