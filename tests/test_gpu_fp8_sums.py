# SPDX-License-Identifier: BSD-3-Clause
"""Sums of 8-bit products on the GPU, fp32 ones and those of the 8-bit matrix
instructions, by every kernel.

Bounds: K additions in fp32 change a partial sum, at most sum|a||b|, by at most a unit of
24 bits each, K 2^-23 sum|a||b|.  The 8-bit instructions add up eight products at a time and
keep 16 bits below the largest: each is off by less than 2^-15 of it, all by 8 2^-15
sum|a||b| = 2^-12 sum|a||b| besides.  A bf16 result is off by half a step, 2^-8 |c|, of what
was summed."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import xtc_amd.graphs.xtc.op as O
from expert_calls import IDS, Mem, ints, padded, rounded
from fp8_cases import CASES, FP8, FP32, TILES
from layer_calls import finish
from test_gpu_layer_graphs import payload
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.fp8 import fp8_codes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def product(a, b, sums, out="float32", pad=0, shift=0):
    """a, b: (codes, scales)."""
    (M, nb), N = a[1].shape, len(b[0])
    print(f"[fp8 sums] {M}x{N}x{nb} sums {sums} {out}", flush=True)
    d = capi.Fp8MatmulDesc(out_dtype=IDS[out], M=M, N=N, blocks=nb, b_block_rows=1 if len(b[1]) == N else 128, ldc=N + pad, sums=sums)
    mems = [Mem(a[0], "uint8"), Mem(a[1], "uint8", 1), Mem(b[0], "uint8"), Mem(b[1], "uint8", 1)]
    res = Mem(padded(np.full((M, N), 7.0), N + pad), out, shift)
    capi.check(capi.lib().xtc_hip_fp8_matmul(ctypes.byref(d), *[m.ptr for m in mems], res.ptr))
    (got,) = finish(mems, [res])
    assert np.isnan(got[:, N:]).all(), "written past the columns"
    return got[:, :N]


def ones(rows, nb):
    return np.full((rows, nb), 127, np.uint8)


def coded(x):
    """Rows of numbers that 8 bits hold, for scales of 1."""
    s = ones(len(x), x.shape[1] // 128)
    return fp8_codes(x, s), s


def cancelling(rows, nb, negative):
    """Rows with 2^8 and 1 among eight neighbours and 2^8 again in the next eight."""
    x = np.zeros((rows, 128 * nb), np.float32)
    x[:, [0, 1, 8]] = 256, 1, -256 if negative else 256
    return x


@pytest.mark.parametrize("sums,out,kernel,size", CASES)
def test_sums_that_cancel(sums, out, kernel, size):
    """2^16 + 1 - 2^16: 1 in fp32, anything within the bound for the 8-bit instructions."""
    M, N, nb = size
    got = product(coded(cancelling(M, nb, True)), coded(cancelling(N, nb, False)), sums, out)
    if sums == FP32:
        np.testing.assert_array_equal(got, 1)
    else:
        assert np.abs(got - 1).max() <= 2.0**-12 * (2.0**17 + 1) * (1 + 2.0**-8)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,N,nb", [(40, 256, 3), (600, 640, 3)])
def test_the_operator_sums_in_fp32(M, N, nb, out):
    a, b = coded(cancelling(M, nb, True)), coded(cancelling(N, nb, False))
    given = [O.tensor(t.shape, "uint8") for t in (*a, *b)]
    with O.graph(name="sums") as gb:
        O.fp8_matmul(*given, out_dtype=out)
    (got,) = payload(gb.graph, [*a, *b], [np.empty((M, N), np.float32)])
    np.testing.assert_array_equal(got, 1)


def random_rows(seed, rows, nb, block_rows=1):
    rng = np.random.default_rng(seed)
    codes = (rng.integers(0, 127, (rows, 128 * nb)) | rng.integers(0, 2, (rows, 128 * nb)) << 7).astype(np.uint8)
    return codes, (127 + rng.integers(-4, 5, (-(-rows // block_rows), nb))).astype(np.uint8)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_a_row_keeps_its_bits_beside_others(out):
    """Sums of the 8-bit instructions: the first rows of calls of more and more rows, by
    each of the tiles."""
    (_, N, _), nb = TILES["256"], 3
    b = random_rows(1, N, nb, 128)
    codes, scales = random_rows(2, 4000, nb)
    most = product((codes, scales), b, FP8, out)
    for M in (1, 16, 40, 300, 2000):
        np.testing.assert_array_equal(product((codes[:M], scales[:M]), b, FP8, out), most[:M])


@pytest.mark.parametrize("sums", [FP32, FP8])
@pytest.mark.parametrize("M", [16, 300, 2000])
def test_whole_numbers(M, sums):
    """Sums of whole numbers within 15 bits: exact either way."""
    a, b = ints(3, (M, 640), 3), ints(4, (1100, 640), 3)
    for out in ("float32", "bfloat16"):
        np.testing.assert_array_equal(product(coded(a), coded(b), sums, out, 3, 1), rounded(a @ b.T, out))
