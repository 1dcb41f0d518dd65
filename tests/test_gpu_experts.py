# SPDX-License-Identifier: BSD-3-Clause
"""Products by group and their weight gradients on the GPU, against plain
float64 sums.

On whole numbers whose sums stay below 2^24 every order of fp32 sums is exact:
results are compared for equality (after the one rounding of a bf16 result).
Otherwise the bound is (d + 2) 2^-24 sum|a||b| for sums of d terms (products of
bf16 are exact in fp32, an fp32 product and each addition round once), plus half
a unit in the last place, 2^-8 |y|, of a bf16 result.
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from expert_calls import bounds, grad_w, grouped, ints, plain_grad_w, plain_grouped, rounded
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.runtimes.hip.device import HipDevice

pytestmark = pytest.mark.gpu

TYPES = [("float32", "float32"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")]


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def sizes_of(seed, T, E, spare=0):
    rng = np.random.default_rng(seed)
    p = rng.dirichlet(np.full(E, 1.0))
    p[rng.random(E) < 0.2] = 0
    p = p / p.sum() if p.sum() else np.full(E, 1 / E)
    return rng.multinomial(T - spare, p).astype(np.int32)


def within(got, want, spread, depth, out_dtype):
    bound = (depth + 2) * 2.0**-24 * spread + (2.0**-8 * np.abs(want) if out_dtype == "bfloat16" else 0)
    over = np.abs(got - want) - bound
    assert np.all(over <= 0), (np.unravel_index(np.argmax(over), over.shape), np.max(over))


# one row, one expert, more experts than rows, one of a wave's 64 lanes more or
# less; widths at and beside the vectors, slabs and tiles; long sums
SHAPES = [(1, 1, 8, 8), (1, 5, 33, 17), (3, 64, 64, 64), (200, 63, 64, 72), (130, 65, 96, 40), (300, 200, 128, 256),
          (257, 3, 256, 256), (700, 4, 320, 384), (1000, 2, 1024, 512), (515, 7, 1000, 250), (64, 2, 8192, 64),
          (513, 1, 512, 264), (2100, 3, 192, 512)]


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("T,E,K,N", SHAPES)
def test_grouped_whole_numbers(dtype, out, trans_w, T, E, K, N):
    sizes = sizes_of(T + E, T, E, spare=min(T - 1, 5))
    x, w = ints(1, (T, K)), ints(2, (E, K, N))
    print(f"[grouped] {dtype}->{out} trans {trans_w} {T}x{K}x{N} E {E}", flush=True)
    np.testing.assert_array_equal(grouped(x, w, sizes, dtype, out, trans_w), rounded(plain_grouped(x, w, sizes), out))


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("T,E,K,N", SHAPES)
def test_grad_w_whole_numbers(dtype, out, T, E, K, N):
    sizes = sizes_of(T + E, T, E, spare=min(T - 1, 5))
    x, dy = ints(3, (T, K)), ints(4, (T, N))
    print(f"[grad_w] {dtype}->{out} {T}x{K}x{N} E {E}", flush=True)
    np.testing.assert_array_equal(grad_w(x, dy, sizes, dtype, out), rounded(plain_grad_w(x, dy, sizes), out))


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("T,E,K,N", [(300, 4, 515, 129), (600, 3, 512, 256)])
def test_uniform(dtype, out, T, E, K, N):
    rng = np.random.default_rng(9)
    x, w, dy = (rounded(rng.uniform(-1, 1, s), dtype) for s in ((T, K), (E, K, N), (T, N)))
    sizes = sizes_of(6, T, E, 3)
    print(f"[experts uniform] {dtype}->{out} {T}x{K}x{N}", flush=True)
    within(grouped(x, w, sizes, dtype, out), plain_grouped(x, w, sizes), plain_grouped(abs(x), abs(w), sizes), K, out)
    within(grad_w(x, dy, sizes, dtype, out), plain_grad_w(x, dy, sizes), plain_grad_w(abs(x), abs(dy), sizes), T, out)


# sizes that no router makes: none at all, below zero, past the rows, past 32 bits
# in their sum, a single group in the middle
@pytest.mark.parametrize("sizes", [[0, 0, 0], [-5, 40, -1], [100, 100, 100], [2**31 - 1] * 3, [0, 90, 0], [64, 0, 64],
                                   [1, 1, 1], [127, 1, 2**31 - 1]])
@pytest.mark.parametrize("K,N", [(64, 64), (256, 256), (37, 29)])
def test_any_sizes(sizes, K, N):
    T = 130
    x, w, dy = ints(5, (T, K)), ints(6, (3, K, N)), ints(7, (T, N))
    print(f"[experts sizes] {sizes} {K}x{N}", flush=True)
    for trans in (False, True):
        np.testing.assert_array_equal(grouped(x, w, sizes, "bfloat16", "float32", trans), plain_grouped(x, w, sizes))
    np.testing.assert_array_equal(grad_w(x, dy, sizes, "bfloat16", "float32"), plain_grad_w(x, dy, sizes))


# strides with NaN between the rows, and operands off every alignment
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N", [(64, 72), (256, 512), (45, 51)])
@pytest.mark.parametrize("pad,shift", [((8, 16, 8), (0, 0, 0)), ((1, 3, 5), (0, 0, 0)), ((0, 0, 0), (1, 0, 0)),
                                       ((0, 0, 0), (0, 1, 0)), ((0, 0, 0), (0, 0, 1)), ((8, 8, 8), (1, 3, 1))])
def test_strides_and_alignment(dtype, K, N, pad, shift):
    T, sizes = 150, [40, 0, 100]
    x, w, dy = ints(8, (T, K)), ints(9, (3, K, N)), ints(10, (T, N))
    print(f"[experts strides] {dtype} {K}x{N} pad {pad} shift {shift}", flush=True)
    for trans in (False, True):
        got = grouped(x, w, sizes, dtype, "float32", trans, pad, shift)
        np.testing.assert_array_equal(got, plain_grouped(x, w, sizes))
    np.testing.assert_array_equal(grad_w(x, dy, sizes, dtype, "float32", pad, shift), plain_grad_w(x, dy, sizes))


# what a group must not see: the rows and matrices of the others and the rows of
# nobody hold NaN and infinities
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,K,N", [(150, 64, 64), (600, 256, 256), (150, 37, 43), (20, 512, 128)])
def test_groups_do_not_mix(dtype, T, K, N):
    sizes = [T // 3, T // 5, 0, T // 4]
    x, w, dy = ints(11, (T, K)), ints(12, (4, K, N)), ints(13, (T, N))
    b = bounds(sizes, T)
    want, grads = plain_grouped(x, w, sizes), plain_grad_w(x, dy, sizes)
    bad_x, bad_w, bad_dy = x.copy(), w.copy(), dy.copy()
    for rows, bad in ((slice(*b[1]), np.nan), (slice(b[3][1], T), np.inf)):
        bad_x[rows], bad_dy[rows] = bad, bad
    bad_w[1:3] = np.nan
    clean = np.r_[0 : b[0][1], b[3][0] : T]
    print(f"[experts mix] {dtype} {T}x{K}x{N}", flush=True)
    for trans in (False, True):
        got = grouped(bad_x, bad_w, sizes, dtype, "float32", trans)
        np.testing.assert_array_equal(got[clean], want[clean])
        assert np.isnan(got[slice(*b[1])]).all()
    got = grad_w(bad_x, bad_dy, sizes, dtype, "float32")
    np.testing.assert_array_equal(got[[0, 2, 3]], grads[[0, 2, 3]])
    assert np.isnan(got[1]).all()


def test_infinities_stay_where_they_belong():
    x, w = np.ones((70, 64), np.float32), np.ones((1, 64, 64), np.float32)
    x[3, 5], w[0, 7, 9] = np.inf, -np.inf
    with np.errstate(invalid="ignore"):
        want = plain_grouped(x, w, [70])
    for dtype in ("float32", "bfloat16"):
        np.testing.assert_array_equal(grouped(x, w, [70], dtype, "float32"), want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N", [(64, 128), (19, 23)])
def test_gradients_are_differences(dtype, K, N):
    """L = sum(y * c): dL/dw and dL/dx against differences of L itself, exact on
    whole numbers since L is linear in each."""
    T, E, sizes = 50, 3, [20, 0, 27]
    x, w, c = ints(14, (T, K), 2), ints(15, (E, K, N), 2), ints(16, (T, N), 2)
    print(f"[experts differences] {dtype} {K}x{N}", flush=True)

    def loss(x, w):
        return float((grouped(x, w, sizes, dtype, "float32").astype(np.float64) * c).sum())

    dw = grad_w(x, c, sizes, dtype, "float32")
    dx = grouped(c, w.swapaxes(1, 2), sizes, dtype, "float32", trans_w=True)
    base = loss(x, w)
    for e, k, n in ((0, 0, 0), (2, K - 1, N - 1), (1, 3, 4), (0, 7, N // 2)):
        moved = w.copy()
        moved[e, k, n] += 1
        assert loss(x, moved) - base == dw[e, k, n]
    for r, k in ((0, 0), (46, K - 1), (49, 1), (19, 5), (20, 5)):
        moved = x.copy()
        moved[r, k] += 1
        assert loss(moved, w) - base == dx[r, k]


@pytest.mark.parametrize("K,N", [(256, 256), (33, 65)])
def test_same_results_every_time_on_any_stream(K, N):
    T, sizes = 300, [100, 30, 150]
    rng = np.random.default_rng(17)
    x, w, dy = (rounded(rng.uniform(-1, 1, s), "bfloat16") for s in ((T, K), (3, K, N), (T, N)))
    L = capi.lib()
    stream = ctypes.c_void_p(L.xtc_hip_stream_create())
    first = grouped(x, w, sizes, "bfloat16"), grad_w(x, dy, sizes, "bfloat16")
    for s in (None, stream, stream):
        np.testing.assert_array_equal(grouped(x, w, sizes, "bfloat16", stream=s), first[0])
        np.testing.assert_array_equal(grad_w(x, dy, sizes, "bfloat16", stream=s), first[1])
    capi.check(L.xtc_hip_stream_destroy(stream))


def _put(dev, base, offset, array):
    a = np.ascontiguousarray(array)
    dev.memory_copy_to(base + offset, a.ctypes.data_as(ctypes.c_void_p), a.nbytes)


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("K,N", [(64, 128), (35, 41)])
def test_offsets_past_32_bits(trans_w, K, N):
    """Rows of x and y, and matrices of w, more than 2^32 bytes apart."""
    from xtc_amd.utils.bf16 import f32_to_bf16_bits

    dev, L = HipDevice(), capi.lib()
    T, E, sizes = 6, 3, np.array([1, 2, 2], np.int32)
    ldx, stride_w, ldy = 2**29 + 8, 2**30 + 16, 2**28 + 4
    x, w = ints(18, (T, K)), ints(19, (E, K, N))
    print(f"[experts 32 bits] trans {trans_w} {K}x{N}", flush=True)
    xb = dev.memory_allocate(((T - 1) * ldx + K) * 2)
    wb = dev.memory_allocate(((E - 1) * stride_w + K * N) * 2)
    yb = dev.memory_allocate(((T - 1) * ldy + N) * 4)
    sb = dev.memory_allocate(64)
    for r in range(T):
        _put(dev, xb, r * ldx * 2, f32_to_bf16_bits(x[r]))
    for e in range(E):
        _put(dev, wb, e * stride_w * 2, f32_to_bf16_bits(w[e].T if trans_w else w[e]))
    _put(dev, sb, 0, sizes)
    d = capi.GroupedMatmulDesc(dtype=1, out_dtype=0, E=E, T=T, N=N, K=K, ldx=ldx, ldy=ldy, trans_w=int(trans_w),
                               stride_w=stride_w)
    capi.check(L.xtc_hip_grouped_matmul(ctypes.byref(d), xb, wb, sb, yb))
    capi.check(L.xtc_hip_synchronize())
    got = np.empty((T, N), np.float32)
    for r in range(T):
        dev.memory_copy_from(yb + r * ldy * 4, got[r].ctypes.data_as(ctypes.c_void_p), N * 4)
    np.testing.assert_array_equal(got, plain_grouped(x, w, sizes))
    # the gradient of w over the same x, its matrices far apart
    gb = dev.memory_allocate(((E - 1) * stride_w + K * N) * 4)
    dy = ints(20, (T, N))
    db = dev.memory_allocate(T * N * 2)
    _put(dev, db, 0, f32_to_bf16_bits(dy))
    d = capi.GroupedMatmulDesc(dtype=1, out_dtype=0, E=E, T=T, N=N, K=K, ldx=ldx, stride_w=stride_w)
    capi.check(L.xtc_hip_grouped_matmul_grad_w(ctypes.byref(d), xb, db, sb, gb))
    capi.check(L.xtc_hip_synchronize())
    dw = np.empty((E, K, N), np.float32)
    for e in range(E):
        dev.memory_copy_from(gb + e * stride_w * 4, dw[e].ctypes.data_as(ctypes.c_void_p), K * N * 4)
    np.testing.assert_array_equal(dw, plain_grad_w(x, dy, sizes))
    for p in (xb, wb, yb, sb, gb, db):
        dev.memory_free(p)


def test_no_rows():
    L = capi.lib()
    dev = HipDevice()
    sizes, dw = dev.memory_allocate(64), dev.memory_allocate(2 * 8 * 16 * 4)
    _put(dev, sizes, 0, np.array([3, 4], np.int32))
    d = capi.GroupedMatmulDesc(dtype=1, out_dtype=0, E=2, T=0, N=16, K=8)
    capi.check(L.xtc_hip_grouped_matmul(ctypes.byref(d), None, None, sizes, None))
    capi.check(L.xtc_hip_grouped_matmul_grad_w(ctypes.byref(d), None, None, sizes, dw))
    capi.check(L.xtc_hip_synchronize())
    got = np.ones((2, 8, 16), np.float32)
    dev.memory_copy_from(dw, got.ctypes.data_as(ctypes.c_void_p), got.nbytes)
    assert not got.any()
    for p in (sizes, dw):
        dev.memory_free(p)


# grids large enough for the 128 x 128 and the 256 x 256 tiles, cut in every
# direction: rows and columns inside a tile, K inside a slab, one slab and fewer
# slabs than stages, groups of one row and of none
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,N", [(1500, 2056), (4100, 3336)])
@pytest.mark.parametrize("K", [8, 32, 72, 136, 200])
def test_large_tiles(out, T, N, K):
    sizes = [T // 3, 1, 0, T // 5, 257, T // 4]
    x, w = ints(21, (T, K), 3), ints(22, (6, K, N), 3)
    print(f"[experts tiles] {out} {T}x{K}x{N}", flush=True)
    want = rounded(plain_grouped(x, w, sizes), out)
    for trans in (False, True):
        np.testing.assert_array_equal(grouped(x, w, sizes, "bfloat16", out, trans), want)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N,sizes", [(904, 776, [70, 0, 33, 1, 8, 129]), (1544, 1800, [32, 300, 0, 5, 97])])
def test_large_gradient_tiles(out, K, N, sizes):
    T = sum(sizes) + 6
    x, dy = ints(23, (T, K), 3), ints(24, (T, N), 3)
    print(f"[experts gradient tiles] {out} {T}x{K}x{N}", flush=True)
    np.testing.assert_array_equal(grad_w(x, dy, sizes, "bfloat16", out), rounded(plain_grad_w(x, dy, sizes), out))


# gradients of few tiles over many rows, summed in parts: groups of many slabs, of
# one, of none, of fewer slabs than parts; tiles of every size, cut by K and N
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("K,N,sizes", [(64, 72, [4000]), (264, 520, [3000, 0, 40, 2900]), (128, 136, [1500, 31, 33, 1, 0, 2500]),
                                       (520, 264, [6000]), (1032, 776, [5000, 20])])
def test_gradients_in_parts(out, K, N, sizes):
    T = sum(sizes) + 3
    x, dy = ints(25, (T, K), 3), ints(26, (T, N), 3)
    print(f"[experts parts] {out} {T}x{K}x{N}", flush=True)
    want = rounded(plain_grad_w(x, dy, sizes), out)
    for _ in range(2):  # the counters are left as they were
        np.testing.assert_array_equal(grad_w(x, dy, sizes, "bfloat16", out, pad=(8, 8, 8)), want)
