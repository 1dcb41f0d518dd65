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
