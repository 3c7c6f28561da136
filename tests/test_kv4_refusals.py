"""What the C entries of attention over a 4-bit cache refuse, without a GPU:
csrc/kv4.cpp over stand-ins for the launchers (kv4_entries_stub.cpp). Each
entry's call is right as it stands; one thing at a time is made wrong."""
import ctypes
import os
import subprocess

import pytest

from conftest import ROOT

ARG, BOUNDS, HANDLE = -2, -3, -4
u64, vp = ctypes.c_uint64, ctypes.c_void_p
ENTRIES = ("sm_qk_norm_rope", "sm_kv4_bytes", "sm_kv4_write", "sm_kv4_read", "sm_kv4_attention_workspace", "sm_kv4_attention")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("kv4") / "kv4_entries.so")
    subprocess.run(["/opt/rocm/bin/amdclang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "kv4_entries_stub.cpp"),
                    os.path.join(ROOT, "stratacuda_amd", "csrc", "kv4.cpp"), "-Wl,-Bsymbolic", "-o", out], check=True,
                   capture_output=True)
    import stratacuda_amd as sm
    L, real = ctypes.CDLL(out), sm.lib()
    for name in ENTRIES:
        getattr(L, name).argtypes = getattr(real, name).argtypes
    L.stub_context.restype = vp
    L.stub_free.argtypes = [vp]
    L.stub_buffer.argtypes = [vp, u64, u64]
    L.stub_error.argtypes, L.stub_error.restype = [vp], ctypes.c_char_p
    return L


def view(*v):
    return (ctypes.c_int64 * 3)(*v)


class Call:
    """An entry's arguments by name, and the bytes that its buffers need by handle."""

    def __init__(self, entry, names, values, need, outputs):
        self.entry, self.names, self.values, self.need, self.outputs = entry, names.split(), dict(values), need, outputs

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
            assert lib.stub_device() == 0  # the caller's device is current again
            return rc
        finally:
            lib.stub_free(ctx)


SEQ = dict(tokens=5, count=3, longest=4, starts=0x10, lengths=0x20, table=0x30, table_pages=18)
SEQ_NEED = dict(starts=16, lengths=12, table=216)
TILE = 68 * 128  # bytes of a page's tile of dim 72 to 128
ROPE = Call("sm_qk_norm_rope", "Q qv K kv type tokens heads kv_heads dim qg kg eps Cos Sin rotary context positions Yq Yk",
            dict(Q=0x100, qv=view(2000, 200, 72), K=0x200, kv=None, type=0, tokens=5, heads=6, kv_heads=2, dim=72, qg=0x300, kg=0x400,
                 eps=1e-6, Cos=0x500, Sin=0x600, rotary=36, context=100, positions=0x700, Yq=0x800, Yk=0x900),
            dict(Q=(4 * 2000 + 5 * 200 + 72 + 72) * 4, K=5 * 144 * 4, qg=288, kg=288, Cos=100 * 18 * 4, Sin=100 * 18 * 4, positions=20,
                 Yq=5 * 6 * 72 * 4, Yk=5 * 144 * 4), ("Yq", "Yk"))
WRITE = Call("sm_kv4_write", "K kv V vv type tokens count longest starts lengths table table_pages kv_heads dim pool pages",
             dict(SEQ, K=0x100, kv=None, V=0x200, vv=view(300, 100, 7), type=1, kv_heads=2, dim=72, pool=0x300, pages=9),
             dict(SEQ_NEED, K=5 * 144 * 2, V=(4 * 300 + 100 + 7 + 72) * 2, pool=9 * 2 * TILE), ("pool",))
READ = Call("sm_kv4_read", "pool pages kv_heads dim tokens count longest starts lengths table table_pages K kv V vv type",
            dict(SEQ, K=0x100, kv=None, V=0x200, vv=view(300, 100, 7), type=0, kv_heads=2, dim=72, pool=0x300, pages=9),
            dict(SEQ_NEED, K=5 * 144 * 4, V=(4 * 300 + 100 + 7 + 72) * 4, pool=9 * 2 * TILE), ("K", "V"))
# 15 pieces of 4 pages and one more a sequence, of 2 heads' 16 rows: 128 sums and two statistics; 2 words a sequence
WORKSPACE = (15 + 3) * 2 * 16 * (128 + 2) * 4 + 3 * 8
ATTENTION = Call("sm_kv4_attention", "Q qv type tokens count longest starts lengths table table_pages pool pages heads kv_heads dim scale "
                 "window G gv Y ws bytes",
                 dict(SEQ, Q=0x100, qv=None, type=0, pool=0x300, pages=9, heads=6, kv_heads=2, dim=72, scale=0.1, window=0, G=0x400,
                      gv=view(2000, 200, 72), Y=0x500, ws=0x600, bytes=WORKSPACE),
                 dict(SEQ_NEED, Q=5 * 432 * 4, G=(4 * 2000 + 5 * 200 + 144) * 4, pool=9 * 2 * TILE, Y=5 * 432 * 4, ws=WORKSPACE),
                 ("Y", "ws"))
CALLS = [ROPE, WRITE, READ, ATTENTION]


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c.entry)
def test_right_calls_run(lib, call):
    assert call.run(lib) == 0
    assert call.run(lib, change={"type": 0}, sizes={k: 2 * v for k, v in call.need.items()}) == 0


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c.entry)
def test_buffers(lib, call):
    """One byte short, not a buffer, none."""
    for name, nbytes in call.need.items():
        assert call.run(lib, sizes={name: nbytes - 1}) == BOUNDS, name
        assert call.run(lib, sizes={name: None}) == HANDLE, name
        if name != "G":
            assert call.run(lib, change={name: 0}) == HANDLE, name
    assert getattr(lib, call.entry)(None, *[call.values[n] for n in call.names]) == ARG


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c.entry)
def test_outputs_are_no_inputs(lib, call):
    for out in call.outputs:
        for name in call.need:
            if name != out:
                large = {n: 1 << 20 for n in call.need}
                assert call.run(lib, change={out: call.values[name]}, sizes=large) == ARG, (out, name)


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c.entry)
def test_numbers(lib, call):
    wrong = dict(type=[-1, 2], tokens=[0, -1], kv_heads=[0, -2, 4, 1025], dim=[0, 4, 68, 264, -8], heads=[0, 1, 5, 1026, -6],
                 count=[0, -1, 32769], longest=[0, 6, -1], table_pages=[0, -1], pages=[0, -1, (1 << 24) + 1], rotary=[0, 1, 35, 74, -2],
                 context=[0, -1], eps=[-1.0, float("nan")], scale=[0.0, -1.0, float("nan"), float("inf"), 1e30], window=[-1], bytes=[WORKSPACE - 1])
    big = {n: 1 << 50 for n in call.need}
    for name, values in wrong.items():
        if name not in call.values or (name == "kv_heads" and call in (WRITE, READ)):
            continue
        for v in values:
            assert call.run(lib, change={name: v}, sizes=big) == ARG, (name, v)
    if call in (WRITE, READ):
        for v in (0, -1, 1025):
            assert call.run(lib, change={"kv_heads": v}, sizes=big) == ARG
    assert call.run(lib, change={"tokens": 1 << 24}, sizes=big) == ARG
    if "table_pages" in call.values:
        assert call.run(lib, change={"table_pages": (1 << 24) // 3 + 1}, sizes=big) == ARG
        most = {"table_pages": (1 << 24) // 3, **({"bytes": 1 << 40} if call is ATTENTION else {})}
        assert call.run(lib, change=most, sizes=big) == 0


@pytest.mark.parametrize("call", CALLS, ids=lambda c: c.entry)
def test_views(lib, call):
    big = {n: 1 << 50 for n in call.need}
    for name in ("qv", "kv", "vv", "gv"):
        if name not in call.values:
            continue
        for at in range(3):
            for v in (-1, (1 << 40) + 1, -2 ** 63, 2 ** 63 - 1):
                w = [5000, 500, 3]
                w[at] = v
                assert call.run(lib, change={name: view(*w)}, sizes=big) == ARG, (name, w)
        assert call.run(lib, change={name: view(1 << 40, 0, 0)}, sizes=big) == ARG  # 5 rows of it
        if call is READ:  # an output's rows and heads do not overlap
            assert call.run(lib, change={name: view(300, 71, 0)}, sizes=big) == ARG
            assert call.run(lib, change={name: view(171, 100, 0)}, sizes=big) == ARG
            assert call.run(lib, change={name: view(172, 100, 0)}, sizes=big) == 0
        else:  # an input's may
            assert call.run(lib, change={name: view(0, 0, 0)}, sizes=big) == 0


def test_no_gate_takes_no_view(lib):
    assert ATTENTION.run(lib, change={"G": 0, "gv": view(-1, -1, -1)}) == 0


def test_no_workspace_where_none_is_needed(lib):
    """Eight pages are one piece in either type."""
    assert ATTENTION.run(lib, change={"table_pages": 8, "ws": 0, "bytes": 0}) == 0
    assert ATTENTION.run(lib, change={"table_pages": 9, "ws": 0, "bytes": 0}) == ARG


def test_bytes_and_workspace(lib):
    n = u64()
    assert lib.sm_kv4_bytes(7, 3, 200, ctypes.byref(n)) == 0 and n.value == 7 * 3 * 68 * 256
    for args in ((0, 3, 200), (7, 0, 200), (7, 3, 201), (7, 3, 0), ((1 << 24) + 1, 3, 200)):
        assert lib.sm_kv4_bytes(*args, ctypes.byref(n)) == ARG
    assert lib.sm_kv4_bytes(7, 3, 200, None) == ARG
    good = (5, 3, 4, 18, 6, 2, 72)
    assert lib.sm_kv4_attention_workspace(*good, ctypes.byref(n)) == 0 and n.value == WORKSPACE
    assert lib.sm_kv4_attention_workspace(*good, None) == ARG
    for at in range(7):
        bad = list(good)
        bad[at] = 0
        assert lib.sm_kv4_attention_workspace(*bad, ctypes.byref(n)) == ARG


def test_python_types():
    import stratacuda_amd as sm
    with pytest.raises(sm.ArgumentError):
        sm.Backend.kv4_bytes(1, 1, 7)
    q = sm.Sequences(count=1, tokens=1, longest=2, starts=None, lengths=None, table=None, table_pages=1)
    with pytest.raises(sm.ArgumentError):
        sm.Backend.kv4_attention_workspace_bytes(q, 2, 1, 64)
