"""Which kernel attention over a 4-bit cache runs and what workspace it asks
for (csrc/kv4_shapes.h), without a GPU."""
import ctypes
import os
import random
import subprocess
from collections import namedtuple

import pytest

import kv4_batches as batches
from conftest import ROOT

Shape = namedtuple("Shape", "prompt tile_rows tiles pieces least slots bytes units")


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("kv4") / "kv4_rules.so")
    subprocess.run(["/opt/rocm/bin/amdclang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "kv4_rules_stub.cpp"),
                    "-o", out], check=True, capture_output=True)
    L = ctypes.CDLL(out)
    L.rule_workspace.restype = ctypes.c_uint64

    def shape(count, tokens, longest, width, heads, kv, dim, window, bf16):
        to = (ctypes.c_longlong * 8)()
        L.rule_shape(count, tokens, longest, width, heads, kv, dim, window, bf16, to)
        return Shape(*to)
    L.shape = shape
    return L


def of(rules, batch, dim, type, window=0):
    n = batch["sequences"]
    return rules.shape(len(n), sum(r for r, _ in n) + 2, max(1, max(r for r, _ in n)), batch["width"], batch["heads"], batch["kv"], dim, window, type == "bf16")


def test_the_gpu_tests_reach_every_kernel(rules):
    for type, dim in batches.TYPES:
        for window in (0,) + batches.WINDOWS:
            s = of(rules, batches.WHOLE, dim, type, window)
            assert s.prompt and s.pieces == 1
        s = of(rules, batches.PIECES, dim, type)
        assert s.prompt and s.pieces > 1
        assert -(-sum(-(-length // 64) for _, length in batches.PIECES["sequences"]) // s.pieces) > s.least
        s = of(rules, batches.LONG, dim, type)
        assert s.prompt and s.pieces == 1 and batches.LONG["sequences"][0][1] > 64 * 64
    for dim in (192, 256):  # f32 has no kernel of many rows there
        assert not of(rules, batches.WHOLE, dim, "f32").prompt
    for type, dim in batches.TYPES:
        for name in ("FEW", "SOME"):
            for window in (0,) + batches.LONG_WINDOWS:
                s = of(rules, getattr(batches, name), dim, type, window)
                assert not s.prompt and (s.pieces > 4 if window in (0, 1000) else s.pieces == 1)
    for type, dim in (("bf16", 128), ("bf16", 256), ("f32", 64), ("f32", 256)):
        s = of(rules, batches.MIXED, dim, type)
        assert not s.prompt and s.pieces == 1 and s.units < len(batches.MIXED["sequences"]) * s.tiles // 10
    for type in ("bf16", "f32"):
        s = of(rules, batches.LONG_ROWS, 64, type)
        assert not s.prompt and sum(-(-length // 64) for _, length in batches.LONG_ROWS["sequences"]) > 64 * s.pieces
        s = of(rules, batches.FAR_ROWS, 64, type)
        assert not s.prompt and s.pieces > 128


def test_shapes_and_workspace(rules):
    """Whatever the window and the type, the workspace is enough, tiles hold the rows and parts of a row have slots."""
    rng = random.Random(1)
    for _ in range(20000):
        kv = rng.choice([1, 2, 3, 4, 8, 16, 1024])
        heads = kv * rng.choice([1, 2, 5, 8, 12, 64, 1024 // kv])
        count, longest = rng.choice([1, 2, 3, 8, 64, 1000, 32768]), int(2 ** rng.uniform(0, 24)) // heads + 1
        width = int(2 ** rng.uniform(0, 24)) // count + 1
        dim, window = 8 * rng.randint(1, 32), rng.choice([0, 1, 64, 4096, 2 ** 31 - 1, rng.randint(1, 1 << 20)])
        some = [int(rng.uniform(0, 1) ** rng.choice([0.1, 1, 5]) * longest) for _ in range(min(count, 64) - 1)] + [longest]
        tokens = sum(some) + rng.choice([0, 3])
        least = rules.rule_workspace(count, tokens, longest, width, heads, kv, dim)
        for bf16 in (0, 1):
            s = rules.shape(count, tokens, longest, width, heads, kv, dim, window, bf16)
            assert s.bytes <= least < 1 << 40
            rows = longest * (heads // kv)
            assert s.tiles * s.tile_rows >= rows > (s.tiles - 1) * s.tile_rows
            assert s.units >= sum(-(-n * (heads // kv) // s.tile_rows) for n in some)
            if s.pieces == 1:
                assert s.bytes == 0 and s.slots == count and s.least > width
            else:
                # a sequence's last piece may be a part of one
                assert s.slots == s.pieces + count <= 65535
                assert s.bytes == s.slots * kv * s.tiles * s.tile_rows * (-(-dim // 64) * 64 + 2) * 4 + 8 * count


def test_no_workspace_for_short_tables(rules):
    for width in range(1, 20):
        assert (rules.rule_workspace(3, 5, 4, width, 6, 2, 72) == 0) == (width <= 8)
        for bf16, most in ((0, 8), (1, 12)):
            assert (rules.shape(3, 5, 4, width, 6, 2, 72, 0, bf16).pieces == 1) == (width <= most)


def test_more_work_never_returns_to_sixteen_rows(rules):
    """The kernel changes once as tokens grow, and once as the window does."""
    for bf16, dim in ((0, 64), (1, 64), (0, 128), (1, 128), (1, 256)):
        for count, width in ((1, 64), (8, 64), (2, 2048)):
            seen = [rules.shape(count, count * n, n, width, 32, 8, dim, 0, bf16).prompt for n in range(1, 64 * min(width, 64), 7)]
            assert seen == sorted(seen)
            seen = [rules.shape(count, count * 512, 512, width, 32, 8, dim, w, bf16).prompt for w in range(1, 1 << 17, 999)]
            assert seen == sorted(seen)
