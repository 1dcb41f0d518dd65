# SPDX-License-Identifier: BSD-3-Clause
"""How an 8-bit product adds up is its caller's choice: what the entry point launches for
it and refuses, and what the graph operator asks for, on the CPU."""

from __future__ import annotations

import pytest

import xtc_amd.graphs.xtc.op as O
from fp8_cases import CASES, FP8
from test_dispatch import pytestmark, run  # noqa: F401
from test_expert_graphs import build
from test_layer_dispatch import CALLS
from test_layer_graphs import B, F, U8, compiled

TILE = {"fp8_rows<float, 1, 2>": "rows16", "fp8_rows<__bf16, 1, 2>": "rows16", "fp8_rows<float, 2, 2>": "rows32",
        "fp8_rows<__bf16, 2, 2>": "rows32", "2, 4, 4, 2": "256", "2, 2, 4, 4": "256", "2, 2, 2, 2": "128", "2, 2, 1, 1": "64"}


def kernel(name):
    return next(v for k, v in TILE.items() if k in name)


def test_every_kernel_of_either_sums_is_reached(run):  # noqa: F811
    got = run(CALLS + f"""
for sums, out_dtype, _, (M, N, blocks) in {CASES!r}:
    out.append(product(out_dtype=int(out_dtype == "bfloat16"), sums=sums, M=M, N=N, blocks=blocks))
""")
    for (sums, _, want, _), ((name, _),) in zip(CASES, got, strict=True):
        assert kernel(name) == want, (name, want)
        assert "rows" in want or ("<true" in name or "<1" in name) == (sums == FP8), name


def test_the_choice_holds_at_every_number_of_rows(run):  # noqa: F811
    """One kind of sums from one row to many, for either result."""
    sizes = [(M, N, 64) for M in (1, 16, 17, 40, 300, 2000, 8192) for N in (64, 2048, 8192)]
    got = run(CALLS + f"""
for out_dtype in (0, 1):
    for sums in (1, 2):
        out.append([product(out_dtype=out_dtype, sums=sums, M=M, N=N, blocks=b)[0][0] for M, N, b in {sizes!r}])
out.append([product(sums=s) for s in (-1, 3)])
""")
    for i, names in enumerate(got[:4]):
        fast = ["fp8_dma" in n and ("<true" in n or "<1" in n) for n in names]
        assert fast == [i % 2 == 1] * len(sizes), names
    assert all(isinstance(m, str) and "unsupported sums" in m for m in got[4])


def test_few_rows_of_wide_matrices(run):  # noqa: F811
    """Two rounds of tiles take the kernels of few rows, three do not; tiles of 32 rows give
    way to 8-bit sums, where those are wanted, past one."""
    sizes = [(16, 8192), (16, 8224), (16, 11008), (16, 16384), (16, 16416), (17, 8192), (17, 8224), (32, 16384), (32, 16416), (512, 1024), (1, 28672)]
    got = run(CALLS + f"""
for sums in (1, 0):
    out.append([product(out_dtype=1, sums=sums, M=M, N=N, blocks=64)[0][0] for M, N in {sizes!r}])
""")
    want = ["rows16"] * 4 + ["64", "rows32", "rows32", "rows32", "64", "rows32", "64"]
    assert [kernel(n) for n in got[0]] == want, got[0]
    assert [kernel(n) for n in got[1]] == [w if w != "rows32" or i == 5 else "64" for i, w in enumerate(want)], got[1]


def test_the_operator_sums_in_fp32_unless_asked():
    types = [((200, 256), U8), ((200, 2), U8), ((300, 256), U8), ((3, 2), U8)]
    for out in (F, B):
        assert "XTC_HIP_SUMS_FP32, 0}" in compiled(build(lambda *a: O.fp8_matmul(*a, out_dtype=out), *types))
        for sums in ("fp32", "fp8", "any"):
            assert f"XTC_HIP_SUMS_{sums.upper()}, 0}}" in compiled(build(lambda *a: O.fp8_matmul(*a, out_dtype=out, sums=sums), *types))
    with pytest.raises(ValueError, match="are none of"):
        build(lambda *a: O.fp8_matmul(*a, sums="fp16"), *types).outputs_types
