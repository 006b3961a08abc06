"""`rotate` refuses axes that are no whole numbers, which would be cut to another axis."""
import numpy as np
import pytest

from anima_hip import rope_axes
from test_fp8_classes_cpu import lib  # noqa: F401


@pytest.mark.parametrize("axis", [[0.0, 1.0, 1.9, 2.0], [0, 1, float("nan"), 2],
                                  ["0", "1", "2", "0"]])
def test_axes_that_are_no_whole_numbers(lib, axis):  # noqa: F811
    q = np.zeros((1, 5, 2, 8), np.float32)
    with pytest.raises(ValueError, match="pair_axis"):
        rope_axes.rotate(q, None, np.zeros((1, 5, 3), int), np.ones(4), axis)
    assert not lib.seen
    for good in ([0, 1, 2, 0], np.array([2, 2, 1, 0], np.uint64), np.array([True, False] * 2)):
        rope_axes.rotate(q, None, np.zeros((1, 5, 3), int), np.ones(4), good)
    assert len(lib.seen) == 3
