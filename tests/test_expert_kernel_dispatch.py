# SPDX-License-Identifier: BSD-3-Clause
"""That the GPU tests of the expert and 4-bit kernels reach the kernels that they
name: on the CPU, libxtc_hip.so against
the stand-in for the HIP runtime."""

from __future__ import annotations

import pytest

import expert_cases as cases
from test_dispatch import pytestmark, run  # noqa: F401
from test_expert_dispatch import CALLS

IDS = {"float32": 0, "bfloat16": 1}


def names(run, script):  # noqa: F811
    """The kernels of each call."""
    got = run(CALLS + script)
    assert all(isinstance(g, list) for g in got), got
    return [[name for name, _ in g] for g in got]


@pytest.fixture(scope="module")
def launched(run):  # noqa: F811
    forward = cases.GROUPED_SMALL + cases.GROUPED_ANY + cases.GROUPED_DMA
    gradients = cases.GRAD_SMALL + cases.GRAD_ANY
    calls = [("", dict(dtype=IDS[d], out_dtype=IDS[o], trans_w=int(t), T=T, K=K, N=N, E=len(s)))
             for _, d, o, t, T, K, N, s in forward]
    calls += [("_grad_w", dict(dtype=IDS[d], out_dtype=IDS[o], T=T, K=K, N=N, E=len(s))) for _, _, d, o, T, K, N, s in gradients]
    mx4 = [((256, 256 + u, 256, 256 + v, 256 if s else None, 256), dict(out_dtype=IDS[o], M=M, N=N, blocks=nb, E=len(s or [])))
           for _, o, M, N, nb, s, (u, v) in cases.MX4]
    got = names(run, f"""
for fn, kw in {calls!r}:
    out.append(grouped("xtc_hip_grouped_matmul" + fn, **kw))
for args, kw in {mx4!r}:
    out.append(mx4_matmul(args, **kw))
""")
    want = [[c[0]] for c in forward] + [[c[0], *(["grouped_grad_sum"] if c[1] else [])] for c in gradients]
    want += [[c[0]] for c in cases.MX4]
    return list(zip([*forward, *gradients, *cases.MX4], got, want, strict=True))


def test_cases_reach_their_kernels(launched):
    for case, got, want in launched:
        assert got == want, case
