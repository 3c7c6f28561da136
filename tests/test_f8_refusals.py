"""What the C entries of the 8-bit floating-point operators refuse, without a GPU:
csrc/f8.cpp over stand-ins for the launchers (f8_entries_stub.cpp). Each entry's
call is right as it stands; one thing at a time is made wrong."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

ARG, BOUNDS, HANDLE = -2, -3, -4
u64, i32, i64, vp = ctypes.c_uint64, ctypes.c_int, ctypes.c_int64, ctypes.c_void_p


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("f8") / "f8_entries.so")
    subprocess.run(["/opt/rocm/bin/amdclang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "f8_entries_stub.cpp"),
                    os.path.join(ROOT, "stratacuda_amd", "csrc", "f8.cpp"), "-Wl,-Bsymbolic", "-o", out], check=True,
                   capture_output=True)
    import stratacuda_amd as sm
    L, real = ctypes.CDLL(out), sm.lib()
    for name in ("sm_f8_bytes", "sm_f8_quantize", "sm_f8_norm", "sm_f8_project", "sm_f8_gate_up_workspace", "sm_f8_gate_up"):
        getattr(L, name).argtypes = getattr(real, name).argtypes
    L.stub_context.restype = vp
    L.stub_free.argtypes = [vp]
    L.stub_buffer.argtypes = [vp, u64, u64]
    L.stub_error.argtypes, L.stub_error.restype = [vp], ctypes.c_char_p
    return L


class Call:
    """An entry's arguments by name, and the bytes that its buffers need by handle."""

    def __init__(self, entry, names, values, need):
        self.entry, self.names, self.values, self.need = entry, names.split(), dict(values), need

    def run(self, lib, change=(), sizes=()):
        ctx = lib.stub_context()
        try:
            for name, nbytes in {**self.need, **dict(sizes)}.items():
                if nbytes is not None:
                    lib.stub_buffer(ctx, self.values[name], nbytes)
            before, args = lib.stub_launches(), {**self.values, **dict(change)}
            rc = getattr(lib, self.entry)(ctx, *[args[n] for n in self.names])
            assert lib.stub_launches() - before == (rc == 0)
            assert rc == 0 or lib.stub_error(ctx)
            return rc
        finally:
            lib.stub_free(ctx)


QUANTIZE = Call("sm_f8_quantize", "X type rows cols block codes scales",
                dict(X=0x100, type=0, rows=130, cols=300, block=128, codes=0x200, scales=0x300),
                dict(X=130 * 300 * 4, codes=130 * 384, scales=2 * 4))
NORM = Call("sm_f8_norm", "X type R gamma eps rows cols H codes scales",
            dict(X=0x100, type=0, R=0x400, gamma=0x500, eps=1e-6, rows=3, cols=600, H=0x600, codes=0x200, scales=0x300),
            dict(X=7200, R=7200, gamma=2400, H=7200, codes=3 * 640, scales=3 * 8))
PROJECT = Call("sm_f8_project", "X Xs tokens cols W Ws rows R Y type stride offset",
               dict(X=0x100, Xs=0x200, tokens=5, cols=129, W=0x300, Ws=0x400, rows=200, R=0x500, Y=0x600, type=0, stride=210,
                    offset=7),
               dict(X=5 * 256, Xs=5 * 4, W=200 * 256, Ws=2 * 4, R=(4 * 210 + 207) * 4, Y=(4 * 210 + 207) * 4))
GATE_UP = Call("sm_f8_gate_up", "X Xs tokens cols Wg Wgs Wu Wus ff codes scales ws bytes",
               dict(X=0x100, Xs=0x200, tokens=5, cols=129, Wg=0x300, Wgs=0x400, Wu=0x500, Wus=0x600, ff=200, codes=0x700,
                    scales=0x800, ws=0x900, bytes=4000),
               dict(X=5 * 256, Xs=5 * 4, Wg=200 * 256, Wgs=2 * 4, Wu=200 * 256, Wus=2 * 4, codes=5 * 256, scales=5 * 4, ws=4000))
CALLS = [QUANTIZE, NORM, PROJECT, GATE_UP]


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c.entry)
def test_right_calls_run(lib, call):
    assert call.run(lib) == 0


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c.entry)
def test_buffers(lib, call):
    """One byte short, not a buffer, none."""
    for name, nbytes in call.need.items():
        assert call.run(lib, sizes={name: nbytes - 1}) == BOUNDS, name
        assert call.run(lib, sizes={name: None}) == HANDLE, name
        if name not in ("R", "H"):
            assert call.run(lib, change={name: 0}) == HANDLE, name
    assert getattr(lib, call.entry)(None, *[call.values[n] for n in call.names]) == ARG


@pytest.mark.parametrize("call,dims", [(QUANTIZE, ("rows", "cols")), (NORM, ("rows", "cols")),
                                       (PROJECT, ("tokens", "cols", "rows")), (GATE_UP, ("tokens", "cols", "ff"))],
                         ids=lambda v: getattr(v, "entry", ""))
def test_dimensions(lib, call, dims):
    for d in dims:
        for v in (0, -1, -2 ** 31, 2 ** 21 + 1, 2 ** 31 - 1):
            assert call.run(lib, change={d: v}) == ARG, (d, v)
    for a in dims:  # a product past 2^33
        for b in dims:
            if a != b:
                assert call.run(lib, change={a: 2 ** 21, b: 2 ** 13}) == ARG, (a, b)


@pytest.mark.parametrize("call,outputs,inputs", [
    (QUANTIZE, ("codes", "scales"), ("X",)), (NORM, ("codes", "scales"), ("X", "R", "gamma")), (NORM, ("H",), ("gamma",)),
    (PROJECT, ("Y",), ("X", "Xs", "W", "Ws")),
    (GATE_UP, ("codes", "scales", "ws"), ("X", "Xs", "Wg", "Wgs", "Wu", "Wus"))], ids=lambda v: getattr(v, "entry", ""))
def test_one_buffer_twice(lib, call, outputs, inputs):
    big = {n: 1 << 20 for n in call.need}
    for o in outputs:
        for other in inputs + tuple(x for x in outputs if x != o):
            assert call.run(lib, change={o: call.values[other]}, sizes=big) == ARG, (o, other)


def test_kinds(lib):
    for call in (QUANTIZE, NORM, PROJECT):
        for t in (-1, 2):
            assert call.run(lib, change={"type": t}) == ARG
    for b in (0, 2, 64, 256, -1):
        assert QUANTIZE.run(lib, change={"block": b}) == ARG
    assert QUANTIZE.run(lib, change={"type": 1}, sizes={"X": 130 * 300 * 2}) == 0
    assert QUANTIZE.run(lib, change={"block": 1}) == BOUNDS  # 130 rows of scales


def test_norm_arguments(lib):
    for eps in (-1e-9, float("nan")):
        assert NORM.run(lib, change={"eps": eps}) == ARG
    assert NORM.run(lib, change={"eps": 0.0}) == 0
    assert NORM.run(lib, change={"R": 0, "H": 0}) == 0
    assert NORM.run(lib, change={"H": NORM.values["R"]}) == 0
    assert NORM.run(lib, change={"H": NORM.values["X"]}) == 0
    assert NORM.run(lib, change={"type": 1}, sizes={"X": 3600}) == 0
    assert NORM.run(lib, change={"H": NORM.values["X"], "type": 1}) == ARG


def test_project_slots(lib):
    assert PROJECT.run(lib, change={"R": PROJECT.values["Y"]}) == 0
    assert PROJECT.run(lib, change={"R": 0}) == 0
    assert PROJECT.run(lib, change={"type": 1}) == ARG  # a residual
    assert PROJECT.run(lib, change={"type": 1, "R": 0}, sizes={"Y": (4 * 210 + 207) * 2}) == 0
    for change in ({"stride": 199}, {"stride": 0}, {"stride": -210}, {"offset": -1}, {"stride": 2 ** 62}, {"offset": 2 ** 62},
                   {"stride": 2 ** 33 // 5 + 1}):
        assert PROJECT.run(lib, change=change) == ARG, change
    assert PROJECT.run(lib, change={"stride": 211}) == BOUNDS
    assert PROJECT.run(lib, change={"offset": 8}) == BOUNDS


def test_gate_up_arguments(lib):
    assert GATE_UP.run(lib, change={"bytes": 3999}) == ARG
    assert GATE_UP.run(lib, change={"Wu": GATE_UP.values["Wg"], "Wus": GATE_UP.values["Wgs"]}) == 0


def test_sizes():
    import stratacuda_amd as sm
    B = sm.Backend
    assert B.f8_bytes(130, 300, 128) == (130 * 384, 8)
    assert B.f8_bytes(130, 300) == (130 * 384, 130 * 4)
    assert B.f8_bytes(1, 640) == (640, 8)
    assert B.f8_gate_up_workspace_bytes(5, 200) >= 0
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 2), (1, 1, 0), (2 ** 21 + 1, 1, 1), (2 ** 21, 2 ** 13, 1), (-1, 5, 128)):
        with pytest.raises(sm.ArgumentError):
            B.f8_bytes(*bad)
    for bad in ((0, 1), (1, 0), (2 ** 21, 2 ** 13)):
        with pytest.raises(sm.ArgumentError):
            B.f8_gate_up_workspace_bytes(*bad)
    with pytest.raises(sm.ArgumentError):
        B._f8_type("f16")
