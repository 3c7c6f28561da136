"""Which kernel a product of 8-bit matrices takes, by the library's own rules
(f8_rules_stub.cpp) for the 256 compute units of an MI355X."""
import ctypes
import os
import subprocess

from conftest import ROOT

CUS = 256
OUT = {"f32": 0, "bf16": 1, "hidden": 2}


def build(directory):
    out = os.path.join(str(directory), "f8_rules.so")
    subprocess.run(["/opt/rocm/bin/amdclang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "f8_rules_stub.cpp"),
                    "-Wl,-Bsymbolic", "-o", out], check=True, capture_output=True)
    return ctypes.CDLL(out)


class Way:
    """The kernel of one product: `tokens` and `rows` of a workgroup (of a gated pair, of each matrix), whether it is
    persistent, the most tiles that one of its workgroups goes through, and its steps."""

    def __init__(self, kind, tokens, rows, persistent, tiles, steps):
        self.kind, self.tokens, self.rows, self.persistent, self.tiles, self.steps = kind, tokens, rows, persistent, tiles, steps

    def __repr__(self):
        return "%s %d x %d%s" % (self.kind, self.tokens, self.rows,
                                 ", %d tiles of %d steps" % (self.tiles, self.steps) if self.persistent else "")


def most_tiles(lib, n, kb, resident):
    """Tiles of the busiest workgroup: each of eight XCDs takes an eighth of them."""
    return -(-(-(-n // 8)) // (lib.rule_grid(n, kb, CUS, resident) // 8))


def way(lib, type, tokens, cols, rows):
    """type: f32, bf16 or gated"""
    kb = -(-cols // 128)
    if type == "gated":
        tile = lib.rule_gated(tokens, rows, kb, CUS)
        if tile:
            n = -(-tokens // tile) * -(-rows // 128)
            return Way("gated", tile, 128, True, most_tiles(lib, n, kb, 1), kb)
        type = "hidden"
    to = (ctypes.c_int * 4)()
    lib.rule_shape(OUT[type], tokens, rows, kb, CUS, to)
    t, r, resident, blocks = to
    if blocks > 1:
        return Way(type, t, r, False, 1, -(-kb // blocks))
    return Way(type, t, r, True, most_tiles(lib, -(-tokens // t) * -(-rows // r), kb, resident), kb)
