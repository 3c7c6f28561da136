"""The comparison of the 4-bit cache's GPU tests (kv4_compare), on the CPU:
results that are no numbers, or off by more than their bound, fail it."""
import numpy as np
import pytest

import kv4_compare
import kv4_plain as plain


class Held:
    """Two sequences' keys and values as a batch of the GPU tests gives them, and a row of none."""

    def __init__(self, rng, kv=2, dim=8):
        self.sequences, self.starts, self.rows, self.dim = [(3, 5), (2, 1)], np.array([0, 3, 5]), 5, dim
        self.both = [tuple(rng.integers(-4, 5, (length, kv, dim)) / 2 for _ in range(2)) for _, length in self.sequences]

    def held(self, s):
        return self.both[s]


@pytest.fixture
def case():
    rng = np.random.default_rng(1)
    b = Held(rng)
    q = rng.integers(-2, 3, (6, 4, 8)).astype(np.float32)
    got = np.full((6, 4, 8), 9.0)
    for s, (n, length) in enumerate(b.sequences):
        a = b.starts[s]
        got[a:a + n] = plain.attention(q[a:a + n].astype(np.float64), length - n + np.arange(n), *b.held(s), 0.1)[0]
    return b, q, got


def test_right_results_pass(case):
    b, q, got = case
    kv4_compare.expect(b, q, got, 0.1, "f32")
    got[3:5] = 9
    kv4_compare.expect(b, q, got, 0.1, "f32", left=[1])


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("row", [0, 2, 3, 4, 5])  # 3 lies before position 0, 5 belongs to no sequence
@pytest.mark.parametrize("wrong", [np.nan, np.inf, -np.inf, 30.0])
def test_one_wrong_value_fails(case, wrong, row, type):
    b, q, got = case
    got[row, 1, 7] = wrong
    with pytest.raises(AssertionError):
        kv4_compare.expect(b, q, got, 0.1, type)


def test_what_is_no_number_is_outside():
    x = np.array([1.0, np.nan, 1.0, 1.0, np.nan, np.inf, 1.0])
    y = np.array([1.0, 1.0, np.nan, 1.0, np.nan, np.inf, 1.5])
    off = np.array([0.1, 0.1, 0.1, np.nan, 0.1, 0.1, 0.1])
    assert list(kv4_compare.outside(x, y, off)) == [False, True, True, True, True, True, True]
