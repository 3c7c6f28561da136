"""The 8-bit floating-point operators through the JavaScript host (backend.js and
the Node-API addon): its checks and argument order on the CPU, a feed-forward
block on the GPU."""
import json
import os

import numpy as np
import pytest

import f8_plain as p
from test_js_host import run_node


def test_js_f8_cpu():
    assert "FAIL" not in run_node("f8.test.js", "cpu", timeout=120)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 70])
def test_js_f8_gpu(tmp_path, tokens):
    width, ff = 256, 300
    rng = np.random.default_rng(tokens)
    w = {k: rng.normal(0, s[1] ** -0.5, s).astype(np.float32) for k, s in (("wg", (ff, width)), ("wu", (ff, width)), ("wd", (width, ff)))}
    x, r = (rng.normal(0, 1, (tokens, width)).astype(np.float32) for _ in range(2))
    gamma = rng.normal(1, 0.1, width).astype(np.float32)
    h = (x + r).astype(np.float64)
    f8 = lambda m, block: (lambda v, s: v * 2.0 ** (s[:, : v.shape[1] // 128].astype(np.float64) - 127).repeat(block, 0)[: m.shape[0]].repeat(128, 1))(*p.quantize(m, block))[:, : m.shape[1]]  # noqa: E731,E501
    n = f8(h / np.sqrt((h * h).mean(-1, keepdims=True) + 1e-6) * gamma, 1)
    a = f8(p.silu(n @ f8(w["wg"], 128).T) * (n @ f8(w["wu"], 128).T), 1)
    y = h + a @ f8(w["wd"], 128).T
    for name, v in {**w, "x": x, "r": r, "gamma": gamma, "y": y}.items():
        np.ascontiguousarray(v, np.float32).tofile(os.path.join(str(tmp_path), name + ".bin"))
    # A code that falls to the other side of its rounding in f32 is a step off (2^-3 of it at most). Of 256 and 300
    # columns one or two in a thousand tokens do; a whole token's worth of them would still be under 1e-3 of y.
    json.dump({"tokens": tokens, "width": width, "ff": ff, "bound": 1e-3}, open(os.path.join(str(tmp_path), "shape.json"), "w"))
    assert "FAIL" not in run_node("f8.test.js", "gpu", str(tmp_path), timeout=300)
