# SPDX-License-Identifier: BSD-3-Clause
"""4-bit codes for given scales and values in strided rows, against their
definition in numpy."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from expert_calls import IDS, Mem, encode, padded, rounded
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.mx4 import mx4_codes, mx4_values

pytestmark = pytest.mark.gpu

NANS = np.array([0x7FC00000, 0xFFC00000, 0x7F800001, 0xFF800001, 0x7FFFFFFF, 0xFFFFFFFF], np.uint32).view(np.float32)


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def test_codes_of_fp32_for_given_scales():
    """NaN of both signs, infinities, zeros, subnormals and numbers of every exponent,
    under every scale: a NaN's code is a zero of its sign, all codes are 0 under 255."""
    rng = np.random.default_rng(71)
    bits = rng.integers(0, 2**32, (256, 90), np.uint64).astype(np.uint32)
    x = bits.view(np.float32)
    x[:, 1:7] = NANS
    x[:, 30:36] = np.float32([np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45])
    # ties, and their neighbours, of the second block's scales
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 3, 1)
    with np.errstate(over="ignore"):
        ties = np.ldexp(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]), np.arange(256)[:, None] - 127).astype(np.float32)
    x[:, 64:72], x[:, 72:80], x[:, 80:88] = ties, np.nextafter(ties, np.float32(0)), -ties
    got = encode(x, scales, "float32")
    np.testing.assert_array_equal(got, mx4_codes(x, scales))
    nan = np.stack((got[:, :16] & 15, got[:, :16] >> 4), -1).reshape(256, 32)[:, 1:7]
    assert (nan[:255] == [0, 8, 0, 8, 0, 8]).all() and not got[255].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("K", [1, 32, 45, 100, 256])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (8, 0), (5, 3)])
def test_dequantize_strides_and_alignment(dtype, K, pad, shift):
    nb = -(-K // 32)
    rng = np.random.default_rng(K)
    codes = rng.integers(0, 256, (300, 16 * nb)).astype(np.uint8)
    scales = rng.integers(0, 256, (300, nb)).astype(np.uint8)
    d = capi.Mx4Desc(dtype=IDS[dtype], rows=300, K=K, ld=K + pad)
    mems = [Mem(codes, "uint8"), Mem(scales, "uint8", shift), Mem(padded(np.full((300, K), 7.0), K + pad), dtype, shift)]
    print(f"[mx4 dequantize strides] {dtype} {K} pad {pad} shift {shift}", flush=True)
    capi.check(capi.lib().xtc_hip_mx4_dequantize(ctypes.byref(d), *[m.ptr for m in mems]))
    capi.check(capi.lib().xtc_hip_synchronize())
    got = mems[2].numpy()
    for m in mems:
        m.free()
    assert np.isnan(got[:, K:]).all(), "written past the columns"
    np.testing.assert_array_equal(got[:, :K], rounded(mx4_values(codes, scales, K), dtype))
