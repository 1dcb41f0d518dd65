# SPDX-License-Identifier: BSD-3-Clause
"""The expert layer's activations between its products are kept in fp32 or in x's type, as
the caller has it: types, numpy semantics, plans and launches, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest

import xtc_amd.graphs.xtc.op as O
from test_dispatch import pytestmark, run  # noqa: F401
from test_expert_graphs import build, forward
from test_layer_dispatch import CALLS
from test_layer_graphs import B, F, compiled
from xtc_amd.utils.bf16 import round_to_bf16


def graph(dtype=B, T=2, E=1, K=3, H=5, **attrs):
    return build(lambda *a: O.expert_layer(*a, top_k=1, activation="relu", **attrs), ((T, K), dtype), ((E, K), dtype), ((E, H, K), dtype),
                 ((E, K, H), dtype))


def test_types():
    for dtype, hidden in ((B, F), (B, B), (F, F)):
        assert graph(dtype, hidden_dtype=hidden).outputs_types[0].constant_shape == (2, 3)
    for dtype, hidden in ((F, B), (B, "float64"), (F, "float16")):
        with pytest.raises(ValueError, match="neither float32 nor x's type"):
            graph(dtype, hidden_dtype=hidden).outputs_types


def test_semantics():
    """257 needs nine bits, one more than bf16 has."""
    x, router = np.array([[1, 1, 0], [1, 0, 0]], np.float32), np.zeros((1, 3), np.float32)
    up, down = np.zeros((1, 5, 3), np.float32), np.zeros((1, 3, 5), np.float32)
    up[0, 0], down[0, :, 0] = (256, 1, 0), (1, 2, 0)
    up[0, 1, :2], down[0, 1, 1] = 256, -1  # 512 for the first token, 256 for the second
    for attrs, first in (({}, 257), (dict(hidden_dtype=F), 257), (dict(hidden_dtype=B), 256)):
        (y,) = forward(graph(**attrs), x, router, up, down)
        want = np.array([[first, 2 * first - 512, 0], [256, 256, 0]], np.float32)
        np.testing.assert_array_equal(y, round_to_bf16(want))


def test_plans():
    """What the generated call asks for, after the row strides."""
    for dtype, attrs, want in ((B, {}, 1), (B, dict(hidden_dtype=F), 1), (B, dict(hidden_dtype=B), 0), (F, {}, 1)):
        assert f", 1, 0, 0, {want}, 0}};" in compiled(graph(dtype, **attrs))


def test_launches(run):  # noqa: F811
    """Rows of the down matrices by three planes of tokens for bf16 alone."""
    got = run(CALLS + """
for weights, dtype in ((0, 0), (0, 1), (1, 1), (2, 1)):
    for hidden in (0, 1):
        for H, K in ((32, 64), (64, 2048), (8192, 2048)):
            out.append(layer(weights=weights, dtype=dtype, hidden_f32=hidden, H=H, K=K)[-1][0])
out.append([layer(room=2**40, hidden_f32=v) for v in (-1, 2)])
""")
    names, refused = got[:-1], got[-1]
    planes = [name.rstrip(">").rsplit(", ", 1)[1] for name in names]
    assert planes == ["1"] * 6 + (["1"] * 3 + ["3"] * 3) * 3, names
    assert all("hidden_f32" in m for m in refused)
    # by depth and rows: every instance of the three planes is reached
    assert {n for n in names if n.endswith("3>")} == {f"layer_down<{f}, {how}, 3>" for f in (1, 2, 3) for how in ("1, 4", "2, 4", "2, 2")
                                                      if (f, how) != (1, "2, 2")}, names
