# SPDX-License-Identifier: BSD-3-Clause
"""Every kernel of the expert and 4-bit products at sizes that reach it
(expert_cases; test_expert_kernel_dispatch checks on the CPU that they do).

Whole numbers whose sums stay below 2^24 are compared for equality, after the one
rounding of a bf16 result.  On fractions the bounds are those of test_gpu_experts
and test_gpu_mx4: (d + 2) 2^-24 sum|a||b| of d terms, K 2^-23 sum|a||b| of 4-bit
operands, and 2^-8 |c| more for a bf16 result.  What no sum may see is NaN: the
rows of nobody, the matrices of empty groups and the columns between the rows.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import numpy as np
import pytest

import expert_cases as cases
from expert_calls import IDS, Mem, bounds, grad_w, grouped, ints, padded, plain_grad_w, plain_grouped, rounded
from test_gpu_experts import within
from test_gpu_mx4 import check_product, operand, plain
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def frozen(*arrays):
    for a in arrays:
        a.flags.writeable = False
    return arrays


@lru_cache(maxsize=2)
def forward_data(T, K, N, sizes):
    x, w = ints(51, (T, K)), ints(52, (len(sizes), K, N))
    want = plain_grouped(x, w, sizes)
    x[sum(sizes):] = np.nan
    w[[e for e, n in enumerate(sizes) if not n]] = np.nan
    return frozen(x, w, want)


@lru_cache(maxsize=2)
def gradient_data(T, K, N, sizes):
    x, dy = ints(53, (T, K), 3), ints(54, (T, N), 3)
    want = plain_grad_w(x, dy, sizes)
    x[sum(sizes):], dy[sum(sizes):] = np.nan, np.nan
    return frozen(x, dy, want)


FORWARD = cases.GROUPED_SMALL + cases.GROUPED_ANY + cases.GROUPED_DMA
GRADIENTS = cases.GRAD_SMALL + cases.GRAD_ANY + cases.GRAD_DMA


# by size, so that calls of one size share their data
@pytest.mark.parametrize("kernel,dtype,out,trans,T,K,N,sizes", sorted(FORWARD, key=lambda c: c[4:]))
def test_grouped(kernel, dtype, out, trans, T, K, N, sizes):
    x, w, want = forward_data(T, K, N, tuple(sizes))
    pad = (8, 16, 8) if "dma" in kernel else (1, 3, 5)
    print(f"[grouped kernels] {kernel} {T}x{K}x{N} {sizes}", flush=True)
    np.testing.assert_array_equal(grouped(x, w, sizes, dtype, out, trans, pad), rounded(want, out))


@pytest.mark.parametrize("kernel,parts,dtype,out,T,K,N,sizes", sorted(GRADIENTS, key=lambda c: c[4:]))
def test_gradients(kernel, parts, dtype, out, T, K, N, sizes):
    x, dy, want = gradient_data(T, K, N, tuple(sizes))
    pad, shift = ((8, 16, 8), (0, 0, 1)) if "dma" in kernel else ((1, 3, 5), (0, 0, 0))
    print(f"[gradient kernels] {kernel} parts {parts} {T}x{K}x{N} {sizes}", flush=True)
    for s in {(0, 0, 0), shift}:  # the gradient on and off its vectors
        np.testing.assert_array_equal(grad_w(x, dy, sizes, dtype, out, pad, s), rounded(want, out))


def one_of(cs):
    """The last case of each kernel with fp32 results."""
    return list({c[0]: c for c in cs if "float32" in c}.values())


@pytest.mark.parametrize("kernel,dtype,out,trans,T,K,N,sizes", one_of(cases.GROUPED_ANY + cases.GROUPED_DMA))
def test_fractions(kernel, dtype, out, trans, T, K, N, sizes):
    rng = np.random.default_rng(55)
    x, w = (rounded(rng.uniform(-1, 1, s), dtype) for s in ((T, K), (len(sizes), K, N)))
    print(f"[grouped fractions] {kernel} {T}x{K}x{N}", flush=True)
    got = grouped(x, w, sizes, dtype, out, trans)
    within(got, plain_grouped(x, w, sizes), plain_grouped(abs(x), abs(w), sizes), K, out)
    np.testing.assert_array_equal(grouped(x, w, sizes, dtype, out, trans), got)


@pytest.mark.parametrize("kernel,parts,dtype,out,T,K,N,sizes", one_of(cases.GRAD_ANY + cases.GRAD_DMA))
def test_gradients_of_fractions(kernel, parts, dtype, out, T, K, N, sizes):
    rng = np.random.default_rng(56)
    x, dy = (rounded(rng.uniform(-1, 1, s), dtype) for s in ((T, K), (T, N)))
    print(f"[gradient fractions] {kernel} {T}x{K}x{N}", flush=True)
    got = grad_w(x, dy, sizes, dtype, out)
    within(got, plain_grad_w(x, dy, sizes), plain_grad_w(abs(x), abs(dy), sizes), max(sizes), out)
    np.testing.assert_array_equal(grad_w(x, dy, sizes, dtype, out), got)


def mx4_call(ac, asc, bc, bsc, sizes, out, shifts, pad=3):
    """The product, scales `shifts` bytes past a boundary."""
    M, nb = asc.shape
    N = bsc.shape[-2]
    d = capi.Mx4MatmulDesc(out_dtype=IDS[out], E=len(sizes) if sizes else 0, M=M, N=N, blocks=nb, ldc=N + pad)
    mems = [Mem(ac, "uint8"), Mem(asc, "uint8", shifts[0]), Mem(bc, "uint8"), Mem(bsc, "uint8", shifts[1])]
    sz = Mem(np.asarray(sizes), "int32") if sizes else None
    c = Mem(padded(np.full((M, N), 7.0), N + pad), out)
    capi.check(capi.lib().xtc_hip_mx4_matmul(ctypes.byref(d), *[m.ptr for m in mems], sz.ptr if sz else None, c.ptr))
    capi.check(capi.lib().xtc_hip_synchronize())
    got = c.numpy()
    for m in (*mems, c, *([sz] if sz else [])):
        m.free()
    assert np.isnan(got[:, N:]).all(), "written past the columns"
    return got[:, :N]


@lru_cache(maxsize=2)
def mx4_data(M, N, nb, sizes):
    a, b = operand(57, (M,), nb), operand(58, (len(sizes), N) if sizes else (N,), nb)
    return frozen(*a, *b, *plain(*a, *b, sizes))


@pytest.mark.parametrize("kernel,out,M,N,nb,sizes,shifts", sorted(cases.MX4, key=lambda c: (c[2:5], c[5] or [])))
def test_mx4(kernel, out, M, N, nb, sizes, shifts):
    sizes = tuple(sizes) if sizes else None
    ac, asc, bc, bsc, want, spread = mx4_data(M, N, nb, sizes)
    print(f"[mx4 kernels] {kernel} {M}x{N} blocks {nb} {sizes} scales at {shifts}", flush=True)
    got = mx4_call(ac, asc, bc, bsc, sizes, out, shifts)
    check_product(got, want, spread, 32 * nb, out)
    np.testing.assert_array_equal(mx4_call(ac, asc, bc, bsc, sizes, out, shifts), got)


@pytest.mark.parametrize("kernel,out,M,N,nb,sizes,shifts", [c for c in cases.MX4 if c[1] == "float32"])
def test_mx4_nan_blocks(kernel, out, M, N, nb, sizes, shifts):
    """NaN blocks make their rows and columns NaN and no others: at a row's first and
    last block, beside the edges of runs and slabs, in rows of nobody and in the
    matrices of empty groups.  Scales of 1, so that the rest is exact."""
    (ac, _), (bc, _) = operand(59, (M,), nb), operand(60, (len(sizes), N) if sizes else (N,), nb)
    asc, bsc = np.full((M, nb), 127, np.uint8), np.full((*bc.shape[:-1], nb), 127, np.uint8)
    want, _ = plain(ac, asc, bc, bsc, sizes)
    used = sum(sizes) if sizes else M
    asc[2::3, 0], asc[1::7, nb - 1] = 255, 255
    asc[used:] = 255
    bsc[..., 4::5, nb - 1], bsc[..., 3::11, 0] = 255, 255
    bad = np.zeros((M, N), bool)
    bad[2::3], bad[1::7], bad[:, 4::5], bad[:, 3::11] = True, True, True, True
    bad[used:] = False  # zeros, whatever the rows hold
    for e, (lo, hi) in enumerate(bounds(sizes, M) if sizes else []):
        if lo == hi:
            bsc[e] = 255
    print(f"[mx4 kernels nan] {kernel} {M}x{N} blocks {nb} {sizes}", flush=True)
    got = mx4_call(ac, asc, bc, bsc, sizes, out, shifts)
    np.testing.assert_array_equal(np.isnan(got), bad)
    np.testing.assert_array_equal(got[~bad], want[~bad])
