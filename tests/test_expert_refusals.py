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


@pytest.mark.parametrize("fn,args", [("quantize", 4), ("encode", 3), ("dequantize", 3)])
def test_rows_past_64_bits_of_bytes_are_refused(run, fn, args):  # noqa: F811
    got = run(CALLS + f"""
for kw in (dict(K=32), dict(K=64), dict(K=33), dict(K=1, ld=2**31 - 1)):
    out.append(mx4("xtc_hip_mx4_{fn}", (256,) * {args}, rows=2**61, **kw))
""")
    assert all(isinstance(m, str) and "too many" in m for m in got), got
