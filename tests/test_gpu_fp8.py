# SPDX-License-Identifier: BSD-3-Clause
"""8-bit operands on the GPU.

Codes and scales are compared for equality with their definition in numpy.
Products: bound 128 B 2^-23 sum|a||b|: products of two 8-bit values and powers of two
are exact, and each of the additions changes a partial sum, at most sum|a||b|, by at
most one unit of 24 bits; plus half a step, 2^-8 |c|, of a bf16 result.  Products to bf16
run on instructions that add up eight products at a time, keeping 16 bits below the
largest's (beside 2^16 a product of 1 is lost): each of the eight is off by less than
2^-15 of the largest one, which is at most the eight's sum of |a||b|, so that all of
them add 8 2^-15 sum|a||b|.  Whole numbers whose sums stay below 2^24 are compared for
equality (products of up to 64 are within 16 bits of one another).
"""

from __future__ import annotations

import numpy as np
import pytest

from expert_calls import ints, rounded
from layer_calls import fp8_dequantize, fp8_encode, fp8_matmul, fp8_quantize, fp8_quantize_both
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.bf16 import bf16_bits_to_f32
from xtc_amd.utils.fp8 import fp8_codes, fp8_scales, fp8_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def turned(x):
    return np.ascontiguousarray(x.swapaxes(1, 2))


def check_quantize(x, dtype, rows=1, transpose=False, **how):
    codes, scales, values = fp8_quantize(x, dtype, rows, transpose, **how)
    v = turned(x) if transpose else x
    want = fp8_scales(v, rows)
    np.testing.assert_array_equal(scales, want)
    np.testing.assert_array_equal(codes, fp8_codes(v, want, rows))
    if values is not None:
        np.testing.assert_array_equal(values, rounded(fp8_values(codes, scales, x.shape[2]), dtype))


MODES = [(1, False), (128, False), (1, True), (128, True)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,transpose", MODES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 128), (1, 128, 128), (2, 3, 127), (1, 129, 130), (3, 200, 300), (1, 300, 1000),
                                   (1, 5, 20000), (1, 9000, 40), (2, 256, 512)])
def test_quantize(dtype, rows, transpose, shape):
    rng = np.random.default_rng(sum(shape))
    check_quantize(rounded(rng.normal(size=shape) * np.exp2(rng.integers(-30, 30, shape)), dtype), dtype, rows, transpose)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 128, 256), (2, 200, 300), (1, 1000, 77)])
def test_quantize_both(dtype, rows, shape):
    x = rounded(np.random.default_rng(sum(shape)).normal(size=shape), dtype)
    codes, scales, codes_t, scales_t = fp8_quantize_both(x, dtype, rows)
    for v, c, s in ((x, codes, scales), (turned(x), codes_t, scales_t)):
        np.testing.assert_array_equal(s, fp8_scales(v, rows))
        np.testing.assert_array_equal(c, fp8_codes(v, s, rows))


def test_every_bf16_beside_every_scale():
    """All 65536 bf16 values as elements of blocks whose largest element is one of a
    few (the value itself, its neighbours, the largest), then as codes for given scales."""
    v = bf16_bits_to_f32(np.arange(65536, dtype=np.uint16))
    for top in (0.0, 1.0, 1.75, 1.7578125, 448.0, 2.0**-126, 2.0**-119, 2.0**-130, 3.0e38):
        x = np.zeros((1, 4096, 2048), np.float32)
        x[0, :, ::128] = v.reshape(4096, 16)
        x[0, :, 7::128] = top
        check_quantize(x, "bfloat16")
    x = v.reshape(1, 512, 128)
    for s in (0, 1, 2, 100, 127, 128, 200, 252, 253, 254, 255):
        scales = np.full((1, 512, 1), s, np.uint8)
        np.testing.assert_array_equal(fp8_encode(x, scales, "bfloat16"), fp8_codes(x, scales))
        for rows, transpose in MODES[1:]:
            t = turned(x) if transpose else x
            given = np.full((1, -(-t.shape[1] // rows), t.shape[2] // 128), s, np.uint8)
            np.testing.assert_array_equal(fp8_encode(x, given, "bfloat16", rows, transpose), fp8_codes(t, given, rows))


def test_ties_and_edges_fp32():
    """Every value, midpoint and their neighbours, at many exponents of fp32."""
    grid = fp8_values(np.arange(128, dtype=np.uint8).reshape(1, 128), np.full((1, 1), 127, np.uint8))[0, :127].astype(np.float32)
    mids = (grid[1:] + grid[:-1]) / 2
    near = [grid, mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(500))]
    rows = []
    for e in range(-149, 110, 7):
        for n in near:
            with np.errstate(under="ignore"):
                r = np.ldexp(n[:126].astype(np.float64), e)
                rows += [np.concatenate([r, np.ldexp([448.0, -448.0], e)]), np.concatenate([-r, np.ldexp([448.0, 1.0], e)])]
    x = np.array(rows).astype(np.float32)[None]
    check_quantize(x, "float32")
    check_quantize(x, "float32", 1, True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,transpose", MODES)
def test_non_finite_blocks(dtype, rows, transpose):
    x = np.ones((1, 300, 400), np.float32)
    x[0, 7, 40], x[0, 140, 140], x[0, 299, 399], x[0, 200, 0] = np.nan, np.inf, -np.inf, np.nan
    x[0, 20:30] = 0
    x[0, 31] = -0.0
    check_quantize(x, dtype, rows, transpose)
    codes, scales, values = fp8_quantize(x, dtype, rows)
    np.testing.assert_array_equal(fp8_dequantize(codes, scales, 400, dtype), values)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,transpose", MODES)
@pytest.mark.parametrize("K", [128, 100, 384])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (128, 0), (5, 3)])
def test_quantize_strides_and_alignment(dtype, rows, transpose, K, pad, shift):
    check_quantize(rounded(np.random.default_rng(K).normal(size=(1, 137, K)), dtype), dtype, rows, transpose, pad=pad, shift=shift)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size,pad", [(1, 0), (128, 0), (45, 3), (300, 0), (256, 8)])
@pytest.mark.parametrize("square", [False, True])
def test_dequantize_every_code_and_scale(dtype, size, pad, square):
    nb = -(-size // 128)
    rng = np.random.default_rng(size)
    codes = rng.integers(0, 256, (2, 300, 128 * nb)).astype(np.uint8)
    scales = rng.integers(0, 256, (2, 3 if square else 300, nb)).astype(np.uint8)
    scales[0, :3, 0] = 0, 254, 255
    want = rounded(fp8_values(codes, scales, size), dtype)
    np.testing.assert_array_equal(fp8_dequantize(codes, scales, size, dtype, pad), want)


# --------------------------------------------------------------- products


def operand(seed, rows, nb, block_rows, spread=4):
    """Random codes (no NaN) and scales within `spread` powers of two of 1."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 127, (rows, 128 * nb)).astype(np.uint8) | (rng.integers(0, 2, (rows, 128 * nb)) << 7).astype(np.uint8)
    return codes, (127 + rng.integers(-spread, spread + 1, (-(-rows // block_rows), nb))).astype(np.uint8)


def check_product(M, N, nb, b_rows, out, seed=0, **how):
    (ac, asc), (bc, bsc) = operand(seed, M, nb, 1), operand(seed + 1, N, nb, b_rows)
    a, b = fp8_values(ac, asc, dtype=np.float64), fp8_values(bc, bsc, dtype=np.float64)
    got, want = fp8_matmul(ac, asc, bc, bsc, out, **how), a @ b.T
    sums, bf16 = abs(a) @ abs(b).T, out == "bfloat16"
    bound = (128 * nb * 2.0**-23 + (2.0**-12 if bf16 else 0)) * sums + (2.0**-8 * np.abs(want) if bf16 else 0)
    over = np.abs(got - want) - bound
    assert np.all(over <= 0), (np.unravel_index(np.argmax(over), over.shape), np.max(over))


# few rows; 64, 128 and 256 tiles; blocks of no whole reads of scales; walks past 64 blocks
PRODUCTS = [(1, 1, 1), (1, 33, 3), (16, 64, 64), (17, 100, 5), (32, 4096, 9), (33, 5000, 2), (100, 200, 7), (300, 3000, 4), (513, 1000, 16),
            (700, 900, 65), (2000, 2100, 3), (2050, 2300, 21), (4100, 4200, 2), (65, 4100, 130), (256, 256, 200)]


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("b_rows", [1, 128])
@pytest.mark.parametrize("M,N,nb", PRODUCTS)
def test_products(M, N, nb, b_rows, out):
    print(f"[fp8 product] {M}x{N}x{nb} blocks, {b_rows} rows a scale, {out}", flush=True)
    check_product(M, N, nb, b_rows, out)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (4, 0), (7, 3)])
@pytest.mark.parametrize("M,N,nb", [(5, 70, 3), (300, 500, 2), (700, 900, 3), (4100, 4200, 1)])
def test_product_strides_and_alignment(M, N, nb, pad, shift, out):
    check_product(M, N, nb, 128, out, pad=pad, shift=shift)


@pytest.mark.parametrize("M,N,K", [(3, 40, 300), (200, 260, 1000), (1000, 1500, 512), (2500, 2600, 640)])
def test_whole_numbers_are_exact(M, N, K):
    """Elements that 8 bits hold and sums below 2^24, through quantisation; a NaN block
    makes its row of c NaN."""
    a, b = ints(1, (M, K), 8), ints(2, (N, K), 8)
    (ac, asc, _), (bc, bsc, _) = fp8_quantize(a[None], "bfloat16"), fp8_quantize(b[None], "bfloat16", 128)
    got = fp8_matmul(ac[0], asc[0], bc[0], bsc[0])
    np.testing.assert_array_equal(got, a.astype(np.float64) @ b.astype(np.float64).T)
    asc[0, M // 2, 1], bsc[0, 0, 0] = 255, 255
    bad = fp8_matmul(ac[0], asc[0], bc[0], bsc[0])
    assert np.isnan(bad[M // 2]).all() and np.isnan(bad[:, :128]).all()
    rest = np.arange(M) != M // 2
    np.testing.assert_array_equal(bad[rest][:, 128:], got[rest][:, 128:])


def test_gradients_of_a_projection():
    """y = x w^T, dx = dy w, dw = dy^T x from operands quantised along what is summed
    over, on numbers that 8 bits hold: equal to the formulas, and to differences (the
    loss sum(y dy) is linear in x and in w)."""
    T, N, K = 150, 200, 260
    x, w, dy = ints(3, (T, K), 4), ints(4, (N, K), 4), ints(5, (T, N), 4)
    xq, xs, xqt, xst = (a[0] for a in fp8_quantize_both(x[None], "bfloat16"))
    wq, wsc, wqt, wst = (a[0] for a in fp8_quantize_both(w[None], "bfloat16", 128))
    dq, ds, dqt, dst = (a[0] for a in fp8_quantize_both(dy[None], "bfloat16"))
    y, dx, dw = fp8_matmul(xq, xs, wq, wsc), fp8_matmul(dq, ds, wqt, wst), fp8_matmul(dqt, dst, xqt, xst)
    np.testing.assert_array_equal(y, x @ w.T)
    np.testing.assert_array_equal(dx, dy @ w)
    np.testing.assert_array_equal(dw, dy.T @ x)
    x2, w2 = x + ints(6, x.shape, 1), w + ints(7, w.shape, 1)
    assert ((x2 @ w.T - x @ w.T) * dy).sum() == (dx * (x2 - x)).sum()
    assert ((x @ w2.T - x @ w.T) * dy).sum() == (dw * (w2 - w)).sum()


def test_same_bits_on_a_stream_of_its_own():
    stream = capi.lib().xtc_hip_stream_create()
    for M, N, nb in ((16, 4096, 32), (200, 300, 40), (1500, 1600, 9)):
        (ac, asc), (bc, bsc) = operand(M, M, nb, 1), operand(N, N, nb, 128)
        np.testing.assert_array_equal(fp8_matmul(ac, asc, bc, bsc), fp8_matmul(ac, asc, bc, bsc, stream=stream))
    capi.check(capi.lib().xtc_hip_stream_destroy(stream))


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,N,nb", [(4000, 3900, 65), (2500, 2000, 130), (520, 1030, 129)])
def test_long_walks(M, N, nb, out):
    """k past the blocks whose scales LDS holds at a time, in tiles of each size: whole
    numbers whose sums stay below 2^15, exact in the 8-bit instructions too, and scales that
    change from block to block by powers of two which a's and b's take from each other."""
    a, b = ints(5, (M, 128 * nb), 1), ints(6, (N, 128 * nb), 1)
    shift = np.random.default_rng(7).integers(-3, 4, nb)
    codes = [fp8_codes(v, np.full((len(v), nb), 127, np.uint8)) for v in (a, b)]
    scales = [np.broadcast_to(127 + s, (n, nb)).astype(np.uint8) for s, n in ((shift, M), (-shift, N))]
    print(f"[fp8 long] {M}x{N}x{nb} {out}", flush=True)
    got = fp8_matmul(codes[0], scales[0], codes[1], scales[1], out)
    np.testing.assert_array_equal(got, rounded(a @ b.T, out))
