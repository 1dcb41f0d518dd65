# SPDX-License-Identifier: BSD-3-Clause
"""4-bit codes of what no scale of its own would be given, in numpy."""

from __future__ import annotations

import numpy as np
import pytest

from xtc_amd.utils.mx4 import mx4_codes, mx4_values


@pytest.mark.parametrize("scale", [0, 1, 127, 254, 255])
def test_codes_of_nan_and_infinity_for_given_scales(scale):
    x = np.zeros((1, 32), np.float32)
    x[0, :4] = np.array([0x7FC00000, 0xFFC00000, 0x7F800000, 0xFF800000], np.uint32).view(np.float32)
    s = np.array([[scale]], np.uint8)
    codes = mx4_codes(x, s)
    assert codes[0, :2].tolist() == ([0, 0] if scale == 255 else [0x80, 0xF7]) and not codes[0, 2:].any()
    values = mx4_values(codes, s, dtype=np.float64)[0]
    if scale == 255:
        assert np.isnan(values).all()
    else:
        assert np.signbit(values[:4]).tolist() == [False, True] * 2
        np.testing.assert_array_equal(values[:4], np.array([0, -0.0, 6, -6]) * 2.0 ** (scale - 127))
