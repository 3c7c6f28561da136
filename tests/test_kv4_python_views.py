"""Views that the Python methods of the 4-bit cache refuse before any call: not
three whole numbers."""
import numpy as np
import pytest

import stratacuda_amd as sm


def test_views():
    assert sm.Backend._view(None) is None
    for view in ((4, 5, 6), [4, 5, 6], np.array([4, 5, 6])):
        assert list(sm.Backend._view(view)) == [4, 5, 6]
    for wrong in ((), (1,), (4, 5), (4, 5, 6, 7)):
        with pytest.raises(sm.ArgumentError):
            sm.Backend._view(wrong)
    for wrong in ((1.5, 2, 3), ("1", 2, 3), (1, None, 3)):
        with pytest.raises(TypeError):
            sm.Backend._view(wrong)
