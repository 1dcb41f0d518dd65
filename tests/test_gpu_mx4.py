# SPDX-License-Identifier: BSD-3-Clause
"""Microscaled 4-bit operators on the GPU.

Codes and scales are compared for equality with their definition in numpy.
Products: bound K 2^-23 sum|a||b|: products of two 4-bit values and powers of
two are exact, and each of the K additions changes a partial sum, at most
sum|a||b|, by at most one unit of 24 bits; plus half a unit in the last place,
2^-8 |c|, of a bf16 result.  Where every scale is 1 and sums stay below 2^22
(in halves of halves, 24 bits) results are compared for equality.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from expert_calls import bounds, dequantize, encode, mx4_matmul, mx4_quantize_matmul, quantize, rounded
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.runtimes.hip.device import HipDevice
from xtc_amd.utils.bf16 import bf16_bits_to_f32
from xtc_amd.utils.mx4 import mx4_codes, mx4_scales, mx4_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def check_quantize(x, dtype, **how):
    codes, scales, values = quantize(x, dtype, **how)
    np.testing.assert_array_equal(scales, mx4_scales(x))
    np.testing.assert_array_equal(codes, mx4_codes(x, scales))
    np.testing.assert_array_equal(values, rounded(mx4_values(codes, scales, x.shape[1]), dtype))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 1000), (64, 64), (130, 4096), (1000, 96), (2, 70000),
                                    (70000, 32), (33, 8192), (9, 256)])
def test_quantize(dtype, rows, K):
    print(f"[mx4 quantize] {dtype} {rows}x{K}", flush=True)
    rng = np.random.default_rng(rows + K)
    x = rounded(rng.normal(size=(rows, K)) * np.exp2(rng.integers(-30, 30, (rows, K))), dtype)
    check_quantize(x, dtype)


def test_every_bf16_beside_every_scale():
    """All 65536 bf16 values as elements of blocks whose largest element is one of
    a few (the value itself, its neighbours in exponent, the largest), then as
    codes for given scales."""
    v = bf16_bits_to_f32(np.arange(65536, dtype=np.uint16))
    for top in (0.0, 1.0, 6.0, 2.0**-126, 2.0**-130, 3.0e38):
        x = np.zeros((4096, 512), np.float32)
        x[:, ::32] = v.reshape(4096, 16)
        x[:, 7::32] = top
        print(f"[mx4 bf16] top {top}", flush=True)
        check_quantize(x, "bfloat16")
    x = v.reshape(2048, 32)
    for s in (0, 1, 2, 100, 127, 128, 200, 252, 253, 254, 255):
        scales = np.full((2048, 1), s, np.uint8)
        np.testing.assert_array_equal(encode(x, scales, "bfloat16"), mx4_codes(x, scales))


def test_ties_and_edges_fp32():
    """Every midpoint, its neighbours, and zeros, at every exponent of fp32."""
    mids = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.999], np.float32)
    near = np.concatenate([mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(9))])[:31]
    rows = []
    for e in range(-149, 126, 3):
        with np.errstate(under="ignore"):
            r = np.ldexp(np.concatenate([near, [np.float32(4.0)]]).astype(np.float64), e)
        rows += [r, -r, np.where(np.arange(32) == 31, np.ldexp(7.5, e), r)]
    x = np.array(rows).astype(np.float32)
    check_quantize(x, "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_non_finite_blocks(dtype):
    x = np.ones((6, 96), np.float32)
    x[0, 40], x[1, 0], x[2, 95], x[3, 33:60] = np.nan, np.inf, -np.inf, np.nan
    x[4] = 0
    x[5] = -0.0
    codes, scales, values = quantize(x, dtype)
    assert scales[0].tolist() == [125, 255, 125] and scales[1, 0] == 255 and scales[2, 2] == 255 and scales[4].tolist() == [0] * 3
    np.testing.assert_array_equal(codes, mx4_codes(x, scales))
    np.testing.assert_array_equal(values, mx4_values(codes, scales))
    np.testing.assert_array_equal(dequantize(codes, scales, 96, dtype), values)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("K", [96, 100, 64, 256])
@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (8, 0), (32, 0), (5, 3)])
def test_quantize_strides_and_alignment(dtype, K, pad, shift):
    print(f"[mx4 strides] {dtype} {K} pad {pad} shift {shift}", flush=True)
    check_quantize(rounded(np.random.default_rng(K).normal(size=(37, K)), dtype), dtype, pad=pad, shift=shift)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("K", [1, 32, 45, 96, 4096])
def test_dequantize_every_code_and_scale(dtype, K):
    nb = -(-K // 32)
    rng = np.random.default_rng(K)
    codes = rng.integers(0, 256, (256, 16 * nb)).astype(np.uint8)
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], nb, 1)
    print(f"[mx4 dequantize] {dtype} {K}", flush=True)
    want = rounded(mx4_values(codes, scales, K), dtype)
    np.testing.assert_array_equal(dequantize(codes, scales, K, dtype), want)


# --------------------------------------------------------------- products


def operand(seed, shape, nb, spread=4):
    """Random codes and scales within `spread` powers of two of 1."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (*shape, 16 * nb)).astype(np.uint8)
    scales = (127 + rng.integers(-spread, spread + 1, (*shape, nb))).astype(np.uint8)
    return codes, scales


def plain(ac, asc, bc, bsc, sizes):
    a, b = mx4_values(ac, asc, dtype=np.float64), mx4_values(bc, bsc, dtype=np.float64)
    if sizes is None:
        return a @ b.T, abs(a) @ abs(b).T
    y, s = np.zeros((len(a), b.shape[1])), np.zeros((len(a), b.shape[1]))
    for e, (lo, hi) in enumerate(bounds(sizes, len(a))):
        y[lo:hi], s[lo:hi] = a[lo:hi] @ b[e].T, abs(a[lo:hi]) @ abs(b[e]).T
    return y, s


def check_product(got, want, spread, K, out):
    bound = K * 2.0**-23 * spread + (2.0**-8 * np.abs(want) if out == "bfloat16" else 0)
    over = np.abs(got - want) - bound
    assert np.all(over <= 0), (np.unravel_index(np.argmax(over), over.shape), np.max(over))


PRODUCTS = [(1, 1, 1), (1, 16, 4), (1, 200, 5), (2, 4096, 64), (5, 64, 13), (16, 256, 128), (17, 65, 3), (32, 512, 256),
            (33, 300, 32), (64, 64, 4), (100, 130, 7), (129, 257, 31), (256, 256, 8), (300, 520, 32), (513, 1000, 36),
            (768, 512, 12), (1030, 264, 20)]


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,N,nb", PRODUCTS)
def test_product(out, M, N, nb):
    print(f"[mx4 product] {out} {M}x{N} blocks {nb}", flush=True)
    a, b = operand(1, (M,), nb), operand(2, (N,), nb)
    want, spread = plain(*a, *b, None)
    check_product(mx4_matmul(*a, *b, out_dtype=out, pad=M % 3, shift=M % 2), want, spread, 32 * nb, out)
    ones = np.full_like(a[1], 127), np.full_like(b[1], 127)
    want, _ = plain(a[0], ones[0], b[0], ones[1], None)
    np.testing.assert_array_equal(mx4_matmul(a[0], ones[0], b[0], ones[1], out_dtype=out), rounded(want, out))


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,E,N,nb", [(1, 1, 16, 4), (2, 8, 128, 32), (40, 65, 72, 5), (32, 16, 256, 128), (200, 3, 300, 8),
                                      (300, 64, 64, 12), (700, 4, 512, 16), (1100, 2, 264, 33), (130, 5, 96, 4)])
def test_grouped_product(out, T, E, N, nb):
    rng = np.random.default_rng(T)
    p = rng.dirichlet(np.full(E, 1.0))
    sizes = rng.multinomial(T - min(T - 1, 3), p).astype(np.int32)
    print(f"[mx4 grouped] {out} {T}x{N} blocks {nb} E {E}", flush=True)
    a, b = operand(3, (T,), nb), operand(4, (E, N), nb)
    want, spread = plain(*a, *b, sizes)
    check_product(mx4_matmul(*a, *b, sizes=sizes, out_dtype=out), want, spread, 32 * nb, out)


@pytest.mark.parametrize("sizes", [[0, 0, 0], [-5, 40, -1], [100, 100, 100], [2**31 - 1] * 3, [0, 90, 0], [1, 1, 1]])
@pytest.mark.parametrize("N,nb", [(64, 4), (256, 8), (45, 5)])
def test_any_sizes(sizes, N, nb):
    print(f"[mx4 sizes] {sizes} {N} {nb}", flush=True)
    a, b = operand(5, (130,), nb), operand(6, (3, N), nb)
    want, spread = plain(*a, *b, sizes)
    check_product(mx4_matmul(*a, *b, sizes=sizes), want, spread, 32 * nb, "float32")


# a block of scale 255 is NaN: its row of a, or its column through b, and no other
@pytest.mark.parametrize("M,N,nb", [(3, 64, 4), (40, 70, 5), (300, 256, 8)])
def test_nan_blocks(M, N, nb):
    a, b = operand(7, (M,), nb), operand(8, (N,), nb)
    want, spread = plain(*a, *b, None)
    a[1][1, nb - 1] = 255
    b[1][9, 0] = 255
    got = mx4_matmul(*a, *b)
    assert np.isnan(got[1]).all() and np.isnan(got[:, 9]).all()
    rest = np.ix_([i for i in range(M) if i != 1], [j for j in range(N) if j != 9])
    check_product(got[rest], want[rest], spread[rest], 32 * nb, "float32")


@pytest.mark.parametrize("sa,sb", [(1, 200), (254, 1), (60, 60), (200, 150), (0, 220)])
def test_extreme_scales(sa, sb):
    nb = 8
    a, b = operand(9, (40,), nb, 0), operand(10, (64,), nb, 0)
    a[1][:], b[1][:] = sa, sb
    want, spread = plain(*a, *b, None)
    # a sum of halves of halves times 2^(sa + sb - 254): exact
    np.testing.assert_array_equal(mx4_matmul(*a, *b), want.astype(np.float32))


def test_groups_do_not_mix():
    nb, sizes = 8, [50, 30, 0, 40]
    a, b = operand(11, (150,), nb), operand(12, (4, 96), nb)
    want, spread = plain(*a, *b, sizes)
    a[1][50:80], a[1][120:], b[1][1:3] = 255, 255, 255
    got = mx4_matmul(*a, *b, sizes=sizes)
    rows = np.r_[0:50, 80:150]
    check_product(got[rows], want[rows], spread[rows], 32 * nb, "float32")
    assert np.isnan(got[50:80]).all()


def test_same_results_every_time_on_any_stream():
    L = capi.lib()
    stream = ctypes.c_void_p(L.xtc_hip_stream_create())
    for M, N, nb in ((16, 512, 64), (300, 256, 16)):
        a, b = operand(13, (M,), nb), operand(14, (N,), nb)
        first = mx4_matmul(*a, *b)
        for s in (None, stream, stream):
            np.testing.assert_array_equal(mx4_matmul(*a, *b, stream=s), first)
    capi.check(L.xtc_hip_stream_destroy(stream))


# grids large enough for the 128 x 128 and the 256 x 256 tiles, cut in rows and
# columns, with fewer slabs than stages and more
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,N", [(1500, 2056), (4100, 3336)])
@pytest.mark.parametrize("nb", [4, 8, 20, 36])
def test_large_tiles(out, M, N, nb):
    print(f"[mx4 tiles] {out} {M}x{N} blocks {nb}", flush=True)
    a, b = operand(15, (M,), nb), operand(16, (N,), nb)
    want, spread = plain(*a, *b, None)
    check_product(mx4_matmul(*a, *b, out_dtype=out), want, spread, 32 * nb, out)
    sizes = [M // 3, 1, 0, M // 5, 257, M // 4]
    b = operand(17, (6, N), nb)
    want, spread = plain(*a, *b, sizes)
    check_product(mx4_matmul(*a, *b, sizes=sizes, out_dtype=out), want, spread, 32 * nb, out)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,E,N,K", [(1, 0, 1, 8), (1, 0, 40, 4096), (3, 0, 200, 1000), (16, 0, 256, 96), (17, 0, 65, 31), (40, 0, 33, 5000),
                                     (250, 0, 80, 640), (16, 0, 8192, 264), (700, 0, 500, 128), (1, 5, 64, 512), (20, 3, 100, 1032),
                                     (300, 4, 256, 64)])
def test_quantised_on_the_way(out, dtype, M, E, N, K):
    """As by two calls, to the bit: blocks of NaN, infinities, zeros, the smallest and
    the largest numbers among them."""
    nb = -(-K // 32)
    rng = np.random.default_rng(M + N)
    x = rng.normal(size=(M, K)) * 2.0 ** rng.integers(-20, 21, (M, K))
    for i, v in enumerate((np.nan, np.inf, 0.0, 2.0**-133, 3.3e38)):
        x[i % M, 32 * i % K :: 97 * (i + 1)] = v
    x = rounded(x, dtype)
    bc, bsc = operand(K, ((E, N) if E else (N,)), nb)
    sizes = rng.multinomial(M - M // 8, np.full(E, 1 / E)) if E else None
    print(f"[mx4 quantise matmul] {M} {E} {N} {K} {dtype} {out}", flush=True)
    codes, scales, _ = quantize(x, dtype)
    want = mx4_matmul(codes, scales, bc, bsc, sizes, out)
    for pad, ldx, shift in ((0, 0, 0), (3, 5, 1)):
        got = mx4_quantize_matmul(x, dtype, bc, bsc, sizes, out, pad, ldx, shift)
        np.testing.assert_array_equal(got, want)


# calls of the 64 x 64, 128 x 128 and 256 x 256 tiles, whose last slab is cut
TILES = [(700, 1000, 12), (2100, 2056, 68), (4100, 3336, 36)]


@pytest.mark.parametrize("M,N,nb", TILES)
def test_nan_beside_the_last_slab(M, N, nb):
    """The scales after a row's last ones are the next row's: NaN there stays there."""
    print(f"[mx4 nan tiles] {M}x{N} blocks {nb}", flush=True)
    a, b = operand(41, (M,), nb), operand(42, (N,), nb)
    want, spread = plain(*a, *b, None)
    a[1][2::3, 0] = 255
    b[1][4::5, :4] = 255
    got = mx4_matmul(*a, *b)
    assert np.isnan(got[2::3]).all() and np.isnan(got[:, 4::5]).all()
    rest = np.ix_([i for i in range(M) if i % 3 != 2], [j for j in range(N) if j % 5 != 4])
    check_product(got[rest], want[rest], spread[rest], 32 * nb, "float32")


@pytest.mark.parametrize("M,N,nb", TILES)
@pytest.mark.parametrize("sa,sb", [(254, 1), (0, 220)])
def test_extreme_scales_of_tiles(M, N, nb, sa, sb):
    print(f"[mx4 extreme tiles] {M}x{N} blocks {nb} {sa} {sb}", flush=True)
    a, b = operand(43, (M,), nb, 0), operand(44, (N,), nb, 0)
    a[1][:], b[1][:] = sa, sb
    want, _ = plain(*a, *b, None)
    np.testing.assert_array_equal(mx4_matmul(*a, *b), want.astype(np.float32))


@pytest.mark.parametrize("M,N,nb", TILES)
def test_groups_of_tiles_do_not_mix(M, N, nb):
    print(f"[mx4 groups tiles] {M}x{N} blocks {nb}", flush=True)
    sizes = [M // 3, M // 5, 0, M // 4]
    b0, b1, end = sizes[0], sizes[0] + sizes[1], sum(sizes)
    a, b = operand(45, (M,), nb), operand(46, (4, N), nb)
    want, spread = plain(*a, *b, sizes)
    a[1][b0:b1], a[1][end:], b[1][1:3] = 255, 255, 255
    first = mx4_matmul(*a, *b, sizes=sizes)
    rows = np.r_[0:b0, b1:M]
    check_product(first[rows], want[rows], spread[rows], 32 * nb, "float32")
    assert np.isnan(first[b0:b1]).all()
    np.testing.assert_array_equal(mx4_matmul(*a, *b, sizes=sizes), first)
