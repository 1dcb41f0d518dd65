# SPDX-License-Identifier: BSD-3-Clause
"""Operands of layer norm, of the 8-bit entry points and of the expert layer more than
2^32 bytes long: rows and matrices far apart, or so many of them."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from expert_calls import IDS, ints, rounded
from layer_calls import check_close, plain_norm, plain_norm_grad
from test_gpu_expert_offsets import get, memory, put, spread  # noqa: F401
from xtc_amd.runtimes.hip import capi
from xtc_amd.utils.bf16 import bf16_bits_to_f32, f32_to_bf16_bits
from xtc_amd.utils.fp8 import fp8_codes, fp8_scales, fp8_values
from xtc_amd.utils.mx4 import mx4_codes, mx4_scales

pytestmark = pytest.mark.gpu

FAR = 1_100_000_000  # elements from a row to the next: the third starts past 2^32 bytes


def call(fn, desc, *args):
    capi.check(getattr(capi.lib(), fn)(ctypes.byref(desc), *args))
    capi.check(capi.lib().xtc_hip_synchronize())


@pytest.mark.parametrize("K", [300, 3000, 9000, 20000])
def test_layer_norm(memory, K):  # noqa: F811
    rng = np.random.default_rng(K)
    x, dy = (rounded(rng.normal(size=(3, K)), "bfloat16") for _ in range(2))
    w, b = (rng.normal(size=K).astype(np.float32) for _ in range(2))
    print(f"[far norm] {K}", flush=True)
    xb, dyb = spread(memory, x, FAR), spread(memory, dy, FAR)
    wb, bb, yb, dxb = memory(4 * K), memory(4 * K), memory((2 * FAR + K) * 2), memory((2 * FAR + K) * 2)
    put(wb, w)
    put(bb, b)
    d = capi.LayerNormDesc(dtype=1, param_dtype=0, rows=3, K=K, ldx=FAR, ldy=FAR, eps=1e-5)
    call("xtc_hip_layer_norm", d, xb, wb, bb, yb)
    rows = [bf16_bits_to_f32(get(yb + r * FAR * 2, K, np.uint16)) for r in range(3)]
    check_close(np.stack(rows), *plain_norm(x, w, b, 1e-5), "bfloat16")
    dwb, dbb, ws = memory(4 * K), memory(4 * K), memory(4 * (2 * 3 * K + 6))
    call("xtc_hip_layer_norm_grad", d, xb, wb, dyb, dxb, dwb, dbb, ws)
    want, off = plain_norm_grad(x, w, dy, 1e-5)
    rows = [bf16_bits_to_f32(get(dxb + r * FAR * 2, K, np.uint16)) for r in range(3)]
    check_close(np.stack(rows), want[0], off[0], "bfloat16")
    check_close(get(dwb, K, np.float32), want[1], off[1], "float32")
    check_close(get(dbb, K, np.float32), want[2], off[2], "float32")


@pytest.mark.parametrize("rows,transpose", [(1, 0), (128, 0), (1, 1), (128, 1)])
def test_quantize(memory, rows, transpose):  # noqa: F811
    """Three matrices of two rows, the rows far apart."""
    x = rounded(np.random.default_rng(rows).normal(size=(3, 2, 300)), "bfloat16")
    base = spread(memory, x.reshape(6, 300), FAR)
    src = x.swapaxes(1, 2) if transpose else x
    want_s = fp8_scales(src, rows)
    want_c = fp8_codes(src, want_s, rows)
    cb, sb = memory(want_c.size), memory(want_s.size)
    d = capi.Fp8Desc(dtype=1, matrices=3, rows=2, K=300, ld=FAR, block_rows=rows, transpose=transpose)
    print(f"[far quantize] {rows} {transpose}", flush=True)
    call("xtc_hip_fp8_quantize", d, base, cb, sb, None)
    np.testing.assert_array_equal(get(sb, want_s.shape, np.uint8), want_s)
    np.testing.assert_array_equal(get(cb, want_c.shape, np.uint8), want_c)


def test_dequantize(memory):  # noqa: F811
    x = rounded(np.random.default_rng(9).normal(size=(3, 300)), "float32")
    s = fp8_scales(x)
    c = fp8_codes(x, s)
    cb, sb, vb = memory(c.size), memory(s.size), memory((2 * FAR + 300) * 4)
    put(cb, c)
    put(sb, s)
    d = capi.Fp8Desc(dtype=0, matrices=1, rows=3, K=300, ld=FAR, block_rows=1)
    call("xtc_hip_fp8_dequantize", d, cb, sb, vb)
    got = np.stack([get(vb + r * FAR * 4, 300, np.float32) for r in range(3)])
    np.testing.assert_array_equal(got, fp8_values(c, s, 300))


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("swap,M,N,blocks", [(False, 16, 2**20 + 40, 33), (True, 16, 2**20 + 40, 33), (True, 5, 8190, 4200)])
def test_products(memory, swap, M, N, blocks, out):  # noqa: F811
    """One operand of more than 2^32 bytes, whole numbers in its last rows: a's (swap)
    rows, b's, and b's for the kernel of few tiles."""
    few, far, near, last = N < 10000, N, M, 30
    big, small = ints(1, (last, 128 * blocks), 2), ints(2, (near, 128 * blocks), 2)
    print(f"[far products] {M}x{N}x{blocks} {swap} {out}", flush=True)
    cb, sb = memory(far * 128 * blocks), memory(far * blocks)
    s = np.full((far, blocks), 127, np.uint8)
    put(sb, s)
    ones = np.full((last, blocks), 127, np.uint8)
    put(cb + (far - last) * 128 * blocks, fp8_codes(big, ones))
    mc, ms = memory(near * 128 * blocks), memory(near * blocks)
    put(ms, np.full((near, blocks), 127, np.uint8))
    put(mc, fp8_codes(small, np.full((near, blocks), 127, np.uint8)))
    a_is_big = swap and not few
    rows, cols = (far, near) if a_is_big else (near, far)
    esz = 4 if out == "float32" else 2
    yb = memory(rows * cols * esz)
    d = capi.Fp8MatmulDesc(out_dtype=IDS[out], M=rows, N=cols, blocks=blocks, b_block_rows=1)
    operands = (cb, sb, mc, ms) if a_is_big else (mc, ms, cb, sb)
    call("xtc_hip_fp8_matmul", d, *operands, yb)
    got = get(yb, (rows, cols), np.float32 if esz == 4 else np.uint16)
    got = bf16_bits_to_f32(got) if esz == 2 else got
    want = rounded((big if a_is_big else small).astype(np.float64) @ (small if a_is_big else big).T.astype(np.float64), out)
    np.testing.assert_array_equal(got[-last:] if a_is_big else got[:, -last:], want)
    rest = got[:-last] if a_is_big else got[:, :-last]
    assert not rest.any()


@pytest.mark.parametrize("weights,H,K", [("dense", 4096, 2304), ("fp8", 8192, 2304), ("mx4", 8192, 4352)])
def test_expert_layer(memory, weights, H, K):  # noqa: F811
    """The last of 256 experts, whose matrices start past 2^32 bytes; whole numbers."""
    T, E = 3, 256
    x = ints(3, (T, K), 1)
    x[:, 0] = 1
    router = np.zeros((E, K), np.float32)
    router[-1, 0] = 64
    up, down = np.zeros((1, H, K), np.float32), np.zeros((1, K, H), np.float32)
    rng = np.random.default_rng(4)
    for a in (up, down):  # few enough for sums below 2^8, which bf16 holds
        a[0, np.arange(a.shape[1]), rng.integers(0, a.shape[2], a.shape[1])] = 2
    print(f"[far layer] {weights}", flush=True)
    bases = []
    for a in (up, down):
        if weights == "dense":
            codes, scales = f32_to_bf16_bits(a), None
        elif weights == "fp8":
            scales = fp8_scales(a, 128)
            codes = fp8_codes(a, scales, 128)
        else:
            scales = mx4_scales(a)
            codes = mx4_codes(a, scales)
        assert E * codes.nbytes > 2**32
        base = memory(E * codes.nbytes)
        put(base + (E - 1) * codes.nbytes, codes)
        bases.append(base)
        if scales is not None:
            at = memory(E * scales.nbytes)
            put(at + (E - 1) * scales.nbytes, scales)
            bases.append(at)
        else:
            bases.append(None)
    d = capi.ExpertLayerDesc(dtype=1, weights=("dense", "fp8", "mx4").index(weights), activation=0, T=T, E=E, K=K, H=H, top_k=1, normalize=1)
    L = capi.lib()
    L.xtc_hip_expert_layer_workspace.restype = ctypes.c_uint64
    need = L.xtc_hip_expert_layer_workspace(ctypes.byref(d))
    xb, rb, ws, yb = memory(x.size * 2), memory(router.size * 2), memory(need), memory(x.size * 2)
    put(xb, f32_to_bf16_bits(x))
    put(rb, f32_to_bf16_bits(router))
    call("xtc_hip_expert_layer", d, xb, rb, bases[0], bases[1], bases[2], bases[3], ws, ctypes.c_uint64(need), yb)
    h = np.maximum(x.astype(np.float64) @ up[0].T, 0)
    want = h @ down[0].T
    assert want.any() and want.max() < 256
    np.testing.assert_array_equal(bf16_bits_to_f32(get(yb, (T, K), np.uint16)), want)
