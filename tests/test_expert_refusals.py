# SPDX-License-Identifier: BSD-3-Clause
"""What the expert and 4-bit entry points refuse past what test_expert_dispatch
asks of them, on the CPU: libxtc_hip.so against the stand-in for the HIP runtime."""

from __future__ import annotations

import pytest

from test_dispatch import pytestmark, run  # noqa: F401
from test_expert_dispatch import CALLS


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("fn", ["grouped_matmul", "grouped_matmul_grad_w"])
def test_too_many_workgroups_are_refused_by_name(run, fn, dtype):  # noqa: F811
    (message,) = run(CALLS + f"""
out.append(grouped("xtc_hip_{fn}", dtype={dtype}, E=1, T=2**31 - 2000, N=2**31 - 2000, K=2**21))
""")
    assert message.startswith(f"{fn}: ") and message.endswith("workgroups are too many"), message
