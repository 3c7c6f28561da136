"""The 8-bit norm on the GPU at both ends of f32's range, against 64 bits (f8_plain)."""
import numpy as np
import pytest

import f8_plain as p
from f8_plain import HALF24
from test_gpu_f8 import F8, get, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [4, 300, 2560, 20000])  # in registers of one wave and of several, and read twice
@pytest.mark.parametrize("eps", [0.0, 1e-38])
def test_norm_of_tiny_and_huge_rows(backend, cols, eps):
    """Rows whose root-mean-square is subnormal, so that one over it passes f32's range, and rows of 1e38, so that one
    over it is subnormal: finite, and as exact as any other row."""
    rng = np.random.default_rng(cols)
    size = np.array([1e-44, 1e-42, 1e-40, 1e-39, 1e-37, 1e30, 3e37, 1e38])
    x = (rng.uniform(0.5, 1, (len(size), cols)) * rng.choice([-1, 1], (len(size), cols)) * size[:, None]).astype(np.float32)
    gamma = rng.normal(1, 0.1, cols).astype(np.float32)
    out, H = F8(backend, len(size), cols), put(backend, np.zeros(x.shape, np.float32))
    backend.f8_norm(put(backend, x), put(backend, gamma), eps, len(size), cols, out.codes, out.scales, H=H)
    assert np.array_equal(get(backend, H, np.float32, x.shape).view(np.uint32), x.view(np.uint32))
    h = x.astype(np.float64)
    y = h / np.sqrt((h * h).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * gamma.astype(np.float64)
    # 1 / sqrt rounded to f32, times h, times gamma
    p.check_f8(*out.read(), y, 4 * HALF24)
