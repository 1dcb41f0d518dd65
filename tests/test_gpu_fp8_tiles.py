# SPDX-License-Identifier: BSD-3-Clause
"""8-bit products by every kernel with a random scale for each block of each row: a kernel
that took another row's scale would be off by powers of two.  Results in rows of their own
stride and off every boundary too.

Bounds as in test_gpu_fp8_sums: K 2^-23 sum|a||b| for fp32 sums, 2^-12 sum|a||b| more for
those of the 8-bit instructions, and half a step of a bf16 result."""

from __future__ import annotations

import functools

import numpy as np
import pytest

from fp8_cases import CASES, FP8
from test_gpu_fp8_sums import product, random_rows
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.fp8 import fp8_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


@functools.lru_cache(maxsize=1)
def operands(size, block_rows):
    """a, b, their product and that of their magnitudes."""
    M, N, nb = size
    a, b = random_rows(M, M, nb), random_rows(N, N, nb, block_rows)
    av, bv = (fp8_values(*v, dtype=np.float64) for v in (a, b))
    return a, b, av @ bv.T, np.abs(av) @ np.abs(bv).T


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("sums,out,kernel,size", sorted(CASES, key=lambda c: c[3]))
def test_every_row_has_its_scales(sums, out, kernel, size, block_rows):
    a, b, want, magnitudes = operands(size, block_rows)
    bound = (128 * size[2] * 2.0**-23 + (2.0**-12 if sums == FP8 else 0)) * magnitudes
    if out == "bfloat16":
        bound += 2.0**-8 * (np.abs(want) + bound)
    first = None
    for pad, shift in ((0, 0), (8, 0), (7, 3), (4, 1)):
        got = product(a, b, sums, out, pad, shift)
        assert np.all(np.abs(got - want) <= bound), (pad, shift, np.unravel_index(np.argmax(np.abs(got - want) - bound), got.shape))
        first = got if first is None else first
        np.testing.assert_array_equal(got, first)
