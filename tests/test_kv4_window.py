"""What window sm_kv4_attention gives its kernels, without a GPU: they take the
difference of a position, which may lie before 0, and the window in 32 bits."""
import ctypes
import os
import subprocess

import pytest

import test_kv4_refusals as entries
from conftest import ROOT


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("kv4") / "kv4_window.so")
    subprocess.run(["/opt/rocm/bin/amdclang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "kv4_window_stub.cpp"),
                    os.path.join(ROOT, "stratacuda_amd", "csrc", "kv4.cpp"), "-Wl,-Bsymbolic", "-o", out], check=True,
                   capture_output=True)
    import stratacuda_amd as sm
    L = ctypes.CDLL(out)
    L.sm_kv4_attention.argtypes = sm.lib().sm_kv4_attention.argtypes
    L.stub_context.restype = ctypes.c_void_p
    L.stub_free.argtypes = [ctypes.c_void_p]
    L.stub_buffer.argtypes = [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_uint64]
    L.stub_error.argtypes, L.stub_error.restype = [ctypes.c_void_p], ctypes.c_char_p
    return L


def test_no_difference_of_a_position_and_a_window_leaves_32_bits(lib):
    big = {n: 1 << 50 for n in entries.ATTENTION.need}
    for table_pages in (1, 18, (1 << 24) // 3):
        reach = 64 * table_pages
        for window in (0, 1, reach - 1, reach, reach + 1, 2 ** 30, 2 ** 31 - 100, 2 ** 31 - 1):
            change = {"table_pages": table_pages, "window": window, "bytes": 1 << 40}
            assert entries.ATTENTION.run(lib, change=change, sizes=big) == 0
            kept = lib.stub_window()
            # no position of the tables lies before any window that reaches past them
            assert kept == (window if window < reach else 0)
            for position in (-(1 << 24), -1, reach - 1):  # a row's; the kernels have position - window + 1
                assert -2 ** 31 <= position - kept < 2 ** 31 - 1
