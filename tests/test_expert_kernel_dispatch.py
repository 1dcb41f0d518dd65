# SPDX-License-Identifier: BSD-3-Clause
"""That the GPU tests of the expert and 4-bit kernels reach the kernels that they
name, and that together they reach all of them: on the CPU, libxtc_hip.so against
the stand-in for the HIP runtime."""

from __future__ import annotations

from itertools import product

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
    gradients = cases.GRAD_SMALL + cases.GRAD_ANY + cases.GRAD_DMA
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


def test_all_kernels_are_reached(launched):
    types = [("float", "float"), ("__bf16", "float"), ("__bf16", "__bf16")]
    want = {f"grouped_any<{t}, {u}, {w}>" for (t, u), w in product(types, ("false, false", "true, false", "false, true"))}
    want |= {f"grouped_small<{t}, {u}, {w}>" for (t, u), w in product(types, (
        "true, false, 1, 1", "false, false, 1, 2", "true, false, 1, 2", "false, false, 1, 4", "true, false, 1, 4", "false, true, 2, 2"))}
    want |= {f"grouped_dma<false, {w}, {tile}>" for w, tile in product(
        ("false, false", "false, true", "true, false"), (cases.TILE64, cases.TILE128, cases.TILE256))}
    want |= {f"grouped_dma<true, false, true, {tile}>" for tile in ("2, 2, 2, 2, 4, false", "2, 2, 4, 4, 2, false", "2, 4, 8, 4, 2, true")}
    want |= {f"mx4_any<{u}>" for u in ("float", "__bf16")} | {"grouped_grad_sum"}
    want |= {f"mx4_rows<{u}, {m}, 2, false>" for u, m in product(("float", "__bf16"), (1, 2))}
    assert {name for _, got, _ in launched for name in got} == want


def test_far_operands_reach_their_kernels(run):  # noqa: F811
    calls = [("", dict(trans_w=int(cases.transposed(k)), T=T, K=K, N=N, E=len(s), ldx=ldx, ldy=ldy, stride_w=sw))
             for k, T, K, N, s, ldx, ldy, sw in cases.FAR]
    calls += [("_grad_w", dict(T=T, K=K, N=N, E=len(s), ldx=ldx, ldy=ldy, stride_w=sw)) for _, T, K, N, s, ldx, ldy, sw in cases.FAR_GRAD]
    mx4 = [((256,) * 4 + (256 if s else None, 256), dict(M=M, N=N, blocks=nb, E=len(s or []), ldc=ldc))
           for _, M, N, nb, s, ldc in cases.FAR_MX4]
    got = names(run, f"""
for fn, kw in {calls!r}:
    out.append(grouped("xtc_hip_grouped_matmul" + fn, **kw))
for args, kw in {mx4!r}:
    out.append(mx4_matmul(args, **kw))
""")
    assert got == [[c[0]] for c in cases.FAR + cases.FAR_GRAD + cases.FAR_MX4]
