# SPDX-License-Identifier: BSD-3-Clause
"""8-bit products and the expert layer at the ends of the scales' range and with NaN among
codes and scales, by every kernel.  A product of two codes has eight significant bits, and
rows with one element each make results of single products: compared for equality."""

from __future__ import annotations

import numpy as np
import pytest

from fp8_cases import CASES, FP8, FP32
from test_gpu_fp8_sums import coded, ones, product
from test_gpu_layer_hidden import layer
from expert_calls import ints, rounded
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.fp8 import fp8_codes, fp8_scales, fp8_values
from xtc_amd.utils.mx4 import mx4_values

pytestmark = pytest.mark.gpu

KERNELS = [c for c in CASES if c[1] == "float32"]


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def single(seed, rows, nb):
    """Codes of one finite element a row, the same one of each."""
    codes = np.zeros((rows, 128 * nb), np.uint8)
    codes[:, 5] = np.arange(rows) % 127 | (np.arange(rows) // 127 % 2) << 7
    return codes


@pytest.mark.parametrize("sums,out,kernel,size", KERNELS)
def test_scales_at_the_ends_of_their_range(sums, out, kernel, size):
    M, N, nb = size
    a, b = single(1, M, nb), single(2, N, nb)
    pairs = [(3, 246), (246, 3), (3, 131), (246, 107), (10, 244)]
    if sums == FP8:  # the instructions take every scale
        pairs += [(0, 254), (254, 0), (1, 250), (247, 2)]
    for sa, sb in pairs:
        sa, sb = np.full((M, nb), sa, np.uint8), np.full((N, nb), sb, np.uint8)
        want = fp8_values(a, sa, dtype=np.float64)[:, 5:6] @ fp8_values(b, sb, dtype=np.float64)[:, 5:6].T
        assert np.abs(want).max() < 2.0**128 and np.abs(want[want != 0]).min() >= 2.0**-149
        np.testing.assert_array_equal(product((a, sa), (b, sb), sums), want.astype(np.float32))


@pytest.mark.parametrize("sums,out,kernel,size", CASES)
def test_nan_codes_and_scales(sums, out, kernel, size):
    """A NaN code makes its row or column NaN, a scale of 255 those of its block, in results
    that are exact otherwise."""
    M, N, nb = size
    x, y = ints(1, (M, 128 * nb), 1), ints(2, (N, 128 * nb), 1)
    (ac, asc), (bc, _) = coded(x), coded(y)
    bsc = ones(-(-N // 128), nb)  # blocks of 128 x 128
    want = rounded(x @ y.T, out)
    np.testing.assert_array_equal(product((ac, asc), (bc, bsc), sums, out), want)
    ac[M // 2, 7], ac[0, -1] = 0x7F, 0xFF
    bc[N - 1, 64] = 0x7F
    asc[M - 1, nb - 1] = 255
    if N > 128:
        bsc[0, 0] = 255
    got = product((ac, asc), (bc, bsc), sums, out)
    rows, columns = np.isin(np.arange(M), (M // 2, 0, M - 1)), np.isin(np.arange(N), (N - 1,))
    if N > 128:
        columns[:128] = True
    assert np.isnan(got[rows]).all() and np.isnan(got[:, columns]).all()
    np.testing.assert_array_equal(got[~rows][:, ~columns], want[~rows][:, ~columns])


@pytest.mark.parametrize("weights,first,second", [("fp8", 3, 246), ("fp8", 246, 3), ("mx4", 0, 252), ("mx4", 252, 0), ("mx4", 130, 120)])
def test_layer_with_scales_at_the_ends(weights, first, second):
    """Two matrices with one element a row: relu of one product, then another."""
    n = 128
    # y = code code x 2^(first + second - 254), with x bringing the activations into range
    x = np.zeros((2, n), np.float32)
    x[:, 3] = 2.0 ** min(127 - first + 10, 100) * np.array([1, -1])
    pair = []
    for i, s in enumerate((first, second)):
        codes = np.zeros((1, n, n if weights == "fp8" else n // 2), np.uint8)
        if weights == "fp8":
            codes[0, :, 3] = np.arange(n) % 127 if i else 0x38
            scales = np.full((1, 1, 1), s, np.uint8)
        else:
            codes[0, :, 1] = (np.arange(n) % 16 if i else 2) << 4
            scales = np.full((1, n, n // 32), s, np.uint8)
        pair.append((codes, scales))
    up, down = ((fp8_values if weights == "fp8" else mx4_values)(*p, n, np.float64)[0] for p in pair)
    want = np.maximum(x.astype(np.float64) @ up.T, 0) @ down.T
    assert np.isfinite(want).all() and want.any() and np.abs(want).max() < 2.0**127
    for hidden in (0, 1):
        np.testing.assert_array_equal(layer(x, np.zeros((1, n), np.float32), *pair, 1, weights, "relu", hidden=hidden), rounded(want, "bfloat16"))
