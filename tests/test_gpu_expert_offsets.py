# SPDX-License-Identifier: BSD-3-Clause
"""Operands of the expert and 4-bit kernels more than 2^32 bytes long: rows and
matrices far apart, and 4-bit operands of so many rows.  Whole numbers, exact."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import expert_cases as cases
from expert_calls import ints, plain_grad_w, plain_grouped
from test_gpu_mx4 import operand, plain
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.runtimes.hip.device import HipDevice
from xtc_amd.utils.bf16 import bf16_bits_to_f32, f32_to_bf16_bits, round_to_bf16
from xtc_amd.utils.mx4 import mx4_codes, mx4_scales, mx4_values

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    """memory(bytes): zeroed device memory that the test's end frees."""
    ensure_device(0)
    dev, held = HipDevice(), []

    def take(nbytes):
        held.append(dev.memory_allocate(nbytes))
        dev.memory_fill_zero(held[-1], nbytes)
        return held[-1]

    yield take
    for p in held:
        dev.memory_free(p)


def put(at, array):
    a = np.ascontiguousarray(array)
    HipDevice().memory_copy_to(at, a.ctypes.data_as(ctypes.c_void_p), a.nbytes)


def get(at, shape, dtype):
    a = np.empty(shape, dtype)
    HipDevice().memory_copy_from(at, a.ctypes.data_as(ctypes.c_void_p), a.nbytes)
    return a


def spread(memory, a, stride):
    """Device memory with the bf16 arrays a[i] `stride` elements apart."""
    base = memory((len(a) - 1) * stride * 2 + a[0].size * 2)
    for i, v in enumerate(a):
        put(base + i * stride * 2, f32_to_bf16_bits(np.ascontiguousarray(v)))
    return base


@pytest.mark.parametrize("kernel,T,K,N,sizes,ldx,ldy,stride_w", cases.FAR)
def test_grouped(memory, kernel, T, K, N, sizes, ldx, ldy, stride_w):
    E, trans = len(sizes), cases.transposed(kernel)
    x, w = ints(61, (T, K)), ints(62, (E, K, N))
    print(f"[far] {kernel}", flush=True)
    xb, wb = spread(memory, x, ldx), spread(memory, w.swapaxes(1, 2) if trans else w, stride_w)
    yb, sb = memory(((T - 1) * ldy + N) * 4), memory(64)
    put(sb, np.array(sizes, np.int32))
    d = capi.GroupedMatmulDesc(dtype=1, out_dtype=0, E=E, T=T, N=N, K=K, ldx=ldx, ldy=ldy, trans_w=int(trans), stride_w=stride_w)
    capi.check(capi.lib().xtc_hip_grouped_matmul(ctypes.byref(d), xb, wb, sb, yb))
    capi.check(capi.lib().xtc_hip_synchronize())
    got = np.stack([get(yb + r * ldy * 4, N, np.float32) for r in range(T)])
    np.testing.assert_array_equal(got, plain_grouped(x, w, sizes))


@pytest.mark.parametrize("kernel,T,K,N,sizes,ldx,ldy,stride_w", cases.FAR_GRAD)
def test_gradients(memory, kernel, T, K, N, sizes, ldx, ldy, stride_w):
    E = len(sizes)
    x, dy = ints(63, (T, K)), ints(64, (T, N))
    print(f"[far gradients] {kernel}", flush=True)
    xb, yb = spread(memory, x, ldx), spread(memory, dy, ldy)
    wb, sb = memory(((E - 1) * stride_w + K * N) * 4), memory(64)
    put(sb, np.array(sizes, np.int32))
    d = capi.GroupedMatmulDesc(dtype=1, out_dtype=0, E=E, T=T, N=N, K=K, ldx=ldx, ldy=ldy, stride_w=stride_w)
    capi.check(capi.lib().xtc_hip_grouped_matmul_grad_w(ctypes.byref(d), xb, yb, sb, wb))
    capi.check(capi.lib().xtc_hip_synchronize())
    got = np.stack([get(wb + e * stride_w * 4, (K, N), np.float32) for e in range(E)])
    np.testing.assert_array_equal(got, plain_grad_w(x, dy, sizes))


def some_rows(rows, row_bytes):
    """Rows at both ends and around multiples of 2^32 bytes."""
    at = {0, 1, rows // 2, rows - 2, rows - 1}
    for k in range(1, rows * row_bytes // 2**32 + 1):
        at |= {min(k * 2**32 // row_bytes + i, rows - 1) for i in (-1, 0, 1)}
    return sorted(at)


def sparse_operand(memory, seed, rows, nb):
    """A 4-bit operand whose rows are zeros of scale 2^-127 but for some: its codes and
    scales on the device, those rows, and their codes and scales."""
    at = some_rows(rows, 16 * nb)
    codes, scales = operand(seed, (len(at),), nb, 0)
    cb, sb = memory(rows * 16 * nb), memory(rows * nb)
    for i, r in enumerate(at):
        put(cb + r * 16 * nb, codes[i])
        put(sb + r * nb, scales[i])
    return cb, sb, at, codes, scales


@pytest.mark.parametrize("kernel,M,N,nb,sizes,ldc", cases.FAR_MX4)
def test_mx4(memory, kernel, M, N, nb, sizes, ldc):
    E = len(sizes) if sizes else 1
    print(f"[far mx4] {kernel} {M}x{N} blocks {nb}", flush=True)
    ac, asc, am, a_codes, a_scales = sparse_operand(memory, 65, M, nb)
    bc, bsc, bn, b_codes, b_scales = sparse_operand(memory, 66, E * N, nb)
    part, _ = plain(a_codes, a_scales, b_codes, b_scales, None)
    want = np.zeros((M, N), np.float32)
    for i, m in enumerate(am):
        for j, n in enumerate(bn):
            if not sizes or sum(sizes[: n // N]) <= m < sum(sizes[: n // N + 1]):
                want[m, n % N] = part[i, j]
    ldc = ldc or N
    c, sb = memory(((M - 1) * ldc + N) * 4), None
    if sizes:
        sb = memory(64)
        put(sb, np.array(sizes, np.int32))
    d = capi.Mx4MatmulDesc(out_dtype=0, E=E if sizes else 0, M=M, N=N, blocks=nb, ldc=ldc)
    capi.check(capi.lib().xtc_hip_mx4_matmul(ctypes.byref(d), ac, asc, bc, bsc, sb, c))
    capi.check(capi.lib().xtc_hip_synchronize())
    got = get(c, (M, N), np.float32) if ldc == N else np.stack([get(c + m * ldc * 4, N, np.float32) for m in range(M)])
    assert want[0].any() and want[-1, -1]  # both ends of the operands
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("ld", [0, 32776])
def test_formats(memory, ld):
    """Codes of more than 2^32 bytes and values of four times as many, dense and not."""
    rows, K = 264000, 32768
    nb, stride = K // 32, ld or K
    at = some_rows(rows, K // 2)
    x = round_to_bf16(np.random.default_rng(67).normal(size=(len(at), K)).astype(np.float32))
    print(f"[far formats] row stride {stride}", flush=True)
    xb, cb, sb, vb = memory(rows * stride * 2), memory(rows * K // 2), memory(rows * nb), memory(rows * stride * 2)
    for i, r in enumerate(at):
        put(xb + r * stride * 2, f32_to_bf16_bits(x[i]))
    L, d = capi.lib(), capi.Mx4Desc(dtype=1, rows=rows, K=K, ld=ld)
    scales = mx4_scales(x)
    codes = mx4_codes(x, scales)
    values = mx4_values(codes, scales)

    def compare(values_at, values_stride):
        for i, r in enumerate(at):
            np.testing.assert_array_equal(get(sb + r * nb, nb, np.uint8), scales[i])
            np.testing.assert_array_equal(get(cb + r * K // 2, K // 2, np.uint8), codes[i])
            got = bf16_bits_to_f32(get(values_at + r * values_stride * 2, K, np.uint16))
            np.testing.assert_array_equal(got, values[i])

    capi.check(L.xtc_hip_mx4_quantize(ctypes.byref(d), xb, cb, sb, vb))
    capi.check(L.xtc_hip_synchronize())
    compare(vb, K)  # quantised values are dense
    HipDevice().memory_fill_zero(vb, rows * stride * 2)
    capi.check(L.xtc_hip_mx4_dequantize(ctypes.byref(d), cb, sb, vb))
    capi.check(L.xtc_hip_synchronize())
    compare(vb, stride)
