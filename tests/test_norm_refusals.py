# SPDX-License-Identifier: BSD-3-Clause
"""Layer norm's gradients refuse rows that are too long to sum over before they launch
anything, on the CPU."""

from __future__ import annotations

from test_dispatch import pytestmark, run  # noqa: F401
from test_layer_dispatch import CALLS

MOST = 65535 * 2048


def test_sums_over_long_rows(run):  # noqa: F811
    got = run(CALLS + f"""
G = "xtc_hip_layer_norm_grad"
for K in ({MOST}, {MOST} + 1, 2**30):
    for rows in (0, 4):
        out.append(norm(G, K=K, rows=rows))
# x's gradient alone has no such bound
out.append(norm(G, (256, 256, 256, 256, None, None, None), K=2**30))
""")
    names = [[g[0].split("<")[0] for g in one] if isinstance(one, list) else one for one in got]
    assert names[0] == ["layer_norm_grad_sum"] and names[1] == ["layer_norm_long", "layer_norm_grad_columns", "layer_norm_grad_sum"]
    assert all(isinstance(one, str) and "too many to sum over" in one for one in names[2:6]), names
    assert names[6] == ["layer_norm_long"]


def test_large_gradients_are_stored_past_the_caches(run):  # noqa: F811
    """fp32 rows past 4096 elements, from 128 MB on."""
    got = run(CALLS + """
G = "xtc_hip_layer_norm_grad"
for dtype, rows, K in ((0, 4096, 8192), (0, 4095, 8192), (0, 2048, 16384), (0, 32768, 4096), (1, 65536, 8192)):
    out.append(norm(G, dtype=dtype, rows=rows, K=K)[0][0])
# no dx, nothing to store
out.append(norm(G, (256, 256, 256, None, 256, 256, 256), dtype=0, rows=4096, K=8192)[0][0])
""")
    assert [name.split("<")[1].split(",")[0] in ("true", "1") for name in got] == [True, False, True, False, False, False], got
