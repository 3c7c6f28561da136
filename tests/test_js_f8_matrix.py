"""HipBackend.f8Matrix over the stand-in addon."""
from test_js_host import run_node


def test_js_f8_matrix():
    assert "FAIL" not in run_node("f8_matrix.test.js", timeout=120)
