"""Attention over a 4-bit cache through the JavaScript host (backend.js and the
Node-API addon): its checks and argument order on the CPU, a layer's prompt and
one more token on the GPU. No counterpart in the reference."""
import json
import os

import numpy as np
import pytest

import kv4_plain as plain
from test_js_host import run_node


def test_js_kv4_cpu():
    assert "FAIL" not in run_node("kv4.test.js", "cpu", timeout=120)


@pytest.mark.gpu
def test_js_kv4_gpu(tmp_path):
    heads, kv, dim, rotary, context, tokens, scale = 12, 2, 128, 64, 400, 300, 128 ** -0.5
    rng = np.random.default_rng(1)
    n = tokens + 1
    full, k, v = (rng.normal(0, 1, s).astype(np.float32) for s in ((n, heads, 2 * dim), (n, kv, dim), (n, kv, dim)))
    qg, kg = (rng.normal(1, 0.1, dim).astype(np.float32) for _ in range(2))
    angles = np.arange(context)[:, None] * 10000.0 ** (-np.arange(rotary // 2) * 2 / rotary)
    cos, sin = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    at = np.arange(n)
    q = plain.norm_rope(full[..., :dim], qg, 1e-6, cos, sin, rotary, at)[0]
    turned = plain.norm_rope(k, kg, 1e-6, cos, sin, rotary, at)[0]
    held, vv = (plain.numbers(*plain.quantize(np.asarray(x, np.float64))) for x in (turned, v))
    y = plain.attention(q, at, held, vv, scale, gate=full[..., dim:].astype(np.float64))[0]
    for name, x in dict(q=full, k=k, v=v, qg=qg, kg=kg, cos=cos, sin=sin, y0=y[:tokens], y1=y[tokens:], v0=vv[:tokens], v1=vv[tokens:]).items():
        np.ascontiguousarray(x, np.float32).tofile(os.path.join(str(tmp_path), name + ".bin"))
    # A key's code that falls to the other side of its rounding in f32 is a step off (a third of it at most). One or two in a
    # million do (2^-21 of the key, where a step is a fifth): of the keys here none or one, of 128 in a score; all scores off by
    # 2^-10 would still be under 2e-3 of y.
    json.dump(dict(heads=heads, kvHeads=kv, dim=dim, rotary=rotary, context=context, tokens=tokens, scale=scale, pages=6,
                   table=[4, 0, 5, 2, 1], bound=2e-3), open(os.path.join(str(tmp_path), "shape.json"), "w"))
    assert "FAIL" not in run_node("kv4.test.js", "gpu", str(tmp_path), timeout=300)
