"""How attention over a 4-bit cache cuts the contexts of batches whose
sequences' rows differ (csrc/kv4_shapes.h), without a GPU."""
import ctypes
import os
import random
import subprocess
from collections import namedtuple

import pytest

import kv4_batches as batches
from conftest import ROOT

Shape = namedtuple("Shape", "prompt tile_rows tiles pieces budget units workspace least")


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("kv4") / "kv4_unlike.so")
    subprocess.run(["/opt/rocm/bin/amdclang++", "-x", "c++", "-std=c++17", "-O1", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "kv4_unlike_stub.cpp"),
                    "-o", out], check=True, capture_output=True)
    L = ctypes.CDLL(out)
    L.rule_workspace.restype = ctypes.c_uint64

    def shape(sequences, width, heads, kv, dim, bf16, window=0):
        to = (ctypes.c_longlong * 8)()
        rows = [n for n, _ in sequences]
        L.rule_unlike(len(rows), max(1, sum(rows)), max(1, max(rows)), width, heads, kv, dim, window, bf16, to)
        return Shape(*to)
    L.shape = shape
    return L


def pieces(s, sequences, group):
    """(tiles, pieces) of each sequence as the kernels cut them, by their formula, and the pages of a piece."""
    tiles = [-(-n * group // s.tile_rows) for n, _ in sequences]
    pages = [-(-length // 64) for _, length in sequences]
    each = max(s.least, -(-sum(t * p for t, p in zip(tiles, pages)) // s.budget))
    return [(t, max(1, -(-p // each)) if t else 0) for t, p in zip(tiles, pages)], each


# 24 heads on 2 of dimension 256, bf16: a chunk and single tokens over long contexts
@pytest.mark.parametrize("sequences,width,prompt", [
    ([(512, 32768), (1, 32768)], 512, True), ([(512, 32768)] + [(1, 32768)] * 2, 512, True), ([(512, 32768)] + [(1, 32768)] * 8, 512, True),
    ([(64, 64)] + [(1, 131072)] * 4, 2048, False), ([(64, 131072)] + [(1, 131072)] * 4, 2048, False)])
def test_single_tokens_beside_a_chunk_are_cut(rules, sequences, width, prompt):
    s = rules.shape(sequences, width, 24, 2, 256, True)
    assert s.prompt == prompt
    many, each = pieces(s, sequences, 12)
    # no workgroup walks a context of many thousand positions alone, and the pieces fill the CUs
    assert all(each <= width // 2 for _, length in sequences if length == 64 * width)
    assert 128 <= 2 * sum(t * p for t, p in many) <= (256 if prompt else 512)
    assert s.workspace < 140 << 20


def test_the_gpu_tests_reach_both(rules):
    for type, dim in batches.TYPES:
        s = rules.shape(batches.UNLIKE["sequences"], batches.UNLIKE["width"], batches.UNLIKE["heads"], batches.UNLIKE["kv"], dim, type == "bf16")
        assert not s.prompt and s.budget and s.pieces == 1
        s = rules.shape(batches.UNLIKE_PROMPT["sequences"], batches.UNLIKE_PROMPT["width"], batches.UNLIKE_PROMPT["heads"],
                        batches.UNLIKE_PROMPT["kv"], dim, type == "bf16")
        assert s.prompt and s.budget and s.pieces == 1
        for which in (batches.UNLIKE, batches.UNLIKE_PROMPT):
            s = rules.shape(which["sequences"], which["width"], which["heads"], which["kv"], dim, type == "bf16")
            many, _ = pieces(s, which["sequences"], which["heads"] // which["kv"])
            assert max(p for _, p in many) > 1


def test_alike_sequences_and_short_tables_are_not(rules):
    for width in (1, 64, 128, 512, 4096):
        for sequences in ([(1, 1)], [(1, 1)] * 8, [(512, 600)], [(64, 100)] * 4):
            assert rules.shape(sequences, width, 24, 2, 256, True).budget == 0
    for width in (1, 16, 127):
        assert rules.shape([(64, 64)] + [(1, 99)] * 4, width, 24, 2, 256, True).budget == 0


def test_workspace(rules):
    """Every tile's pieces have a place, whatever the window, the type and the lengths."""
    rng = random.Random(2)
    seen = 0
    for _ in range(20000):
        kv = rng.choice([1, 2, 4, 8])
        heads, dim = kv * rng.choice([1, 2, 4, 8, 12, 16]), 8 * rng.randint(1, 32)
        count, longest, width = rng.randint(2, 40), int(2 ** rng.uniform(0, 10)), int(2 ** rng.uniform(6, 14))
        sequences = [(int(rng.random() ** 4 * longest), rng.randint(0, 64 * width)) for _ in range(count - 1)] + [(longest, 64 * width)]
        least = rules.rule_workspace(count, max(1, sum(n for n, _ in sequences)), longest, width, heads, kv, dim)
        for bf16 in (False, True):
            for window in (0, 1, 4000, 2 ** 30):
                s = rules.shape(sequences, width, heads, kv, dim, bf16, window)
                assert s.workspace <= least < 1 << 40
                if not s.budget:
                    continue
                seen += 1
                held = kv * (s.units + s.budget) * s.tile_rows
                assert s.workspace == held * (-(-dim // 64) * 64 + 2) * 4 + 8 * count
                assert sum(t for t, _ in pieces(s, sequences, heads // kv)[0]) <= s.units
                assert sum(t * p for t, p in pieces(s, sequences, heads // kv)[0]) <= s.units + s.budget
                assert kv * (s.units + s.budget) <= (256 if s.prompt else 2 * 384)
    assert seen > 1000
