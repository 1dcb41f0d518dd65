# SPDX-License-Identifier: BSD-3-Clause
"""Layer norm and its gradients on the GPU against float64, within what fp32 sums may
be off by (layer_calls.plain_norm, plain_norm_grad), and half a step of a bf16 result."""

from __future__ import annotations

import numpy as np
import pytest

from expert_calls import rounded
from layer_calls import check_close, layer_norm, layer_norm_grad, plain_norm, plain_norm_grad
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device

pytestmark = pytest.mark.gpu

KINDS = [("float32", "float32"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")]


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def inputs(seed, rows, K, dtype, params, offset=1.0):
    rng = np.random.default_rng(seed)
    x = rounded(rng.normal(size=(rows, K)) * rng.choice([1, 16], K) + offset * rng.normal(size=(rows, 1)), dtype)
    w, b = rounded(rng.normal(1, 0.3, K), params), rounded(rng.normal(0, 0.3, K), params)
    return x, w, b, rounded(rng.normal(0, 0.1, (rows, K)), dtype)


SIZES = [(1, 1), (3, 2), (1, 4096), (5, 7), (4, 512), (9, 513), (6, 1000), (700, 1024), (11, 1025), (3, 2048), (13, 4095),
         (600, 2049), (2, 8192), (3, 8193), (2, 16384), (2, 16385), (3, 50001), (1500, 333)]


@pytest.mark.parametrize("dtype,params", KINDS)
@pytest.mark.parametrize("rows,K", SIZES)
def test_forward(dtype, params, rows, K):
    x, w, b, _ = inputs(rows + K, rows, K, dtype, params)
    check_close(layer_norm(x, w, b, dtype, params), *plain_norm(x, w, b, 1e-5), dtype)


@pytest.mark.parametrize("dtype,params", KINDS)
@pytest.mark.parametrize("rows,K", SIZES)
def test_gradients(dtype, params, rows, K):
    x, w, _, dy = inputs(rows + K, rows, K, dtype, params)
    got = layer_norm_grad(x, w, dy, dtype, params)
    want, off = plain_norm_grad(x, w, dy, 1e-5)
    for g, v, o, t in zip(got, want, off, (dtype, "float32", "float32")):
        check_close(g, v, o, t)


@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)])
@pytest.mark.parametrize("K", [96, 3000, 20000])
def test_any_of_the_gradients(want, K):
    x, w, _, dy = inputs(K, 37, K, "float32", "float32")
    for w_given in (w, None):
        all_three = layer_norm_grad(x, w_given, dy, "float32", "float32")
        some = layer_norm_grad(x, w_given, dy, "float32", "float32", want=want)
        for a, s, asked in zip(all_three, some, want):
            assert (s is not None) == bool(asked)
            if asked:
                np.testing.assert_array_equal(a, s)
    check_close(all_three[0], plain_norm_grad(x, None, dy, 1e-5)[0][0], plain_norm_grad(x, None, dy, 1e-5)[1][0], "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("K", [100, 1030, 5000, 17000])
@pytest.mark.parametrize("pad,shift", [((3, 5), (0, 0)), ((8, 16), (1, 3)), ((0, 0), (1, 1))])
def test_strides_alignment_and_no_parameters(dtype, K, pad, shift):
    x, w, b, dy = inputs(K, 19, K, dtype, "float32")
    check_close(layer_norm(x, None, None, dtype, "float32", pad=pad, shift=shift), *plain_norm(x, None, None, 1e-5), dtype)
    check_close(layer_norm(x, w, None, dtype, "float32", pad=pad, shift=shift), *plain_norm(x, w, None, 1e-5), dtype)
    got = layer_norm_grad(x, w, dy, dtype, "float32", pad=pad)
    for g, v, o, t in zip(got, *plain_norm_grad(x, w, dy, 1e-5), (dtype, "float32", "float32")):
        check_close(g, v, o, t)


def test_a_mean_far_from_zero():
    """The deviation is a 4000th of the mean: a difference of two sums would lose it."""
    x, w, b, dy = inputs(5, 40, 2000, "float32", "float32", offset=0)
    x = (x + 65536).astype(np.float32)
    check_close(layer_norm(x, w, b, "float32", "float32"), *plain_norm(x, w, b, 1e-5), "float32")


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1.0])
@pytest.mark.parametrize("K", [64, 3000])
def test_eps_and_equal_elements(eps, K):
    x, w, b, dy = inputs(6, 10, K, "float32", "float32")
    check_close(layer_norm(x, w, b, "float32", "float32", eps=eps), *plain_norm(x, w, b, eps), "float32")
    x[3] = 2.5  # its sums are exact
    if eps > 0:
        y = layer_norm(x, w, b, "float32", "float32", eps=eps)
        np.testing.assert_array_equal(y[3], b)


@pytest.mark.parametrize("K", [64, 3000, 20000])
def test_a_bad_row_stays_alone(K):
    x, w, b, dy = inputs(7, 12, K, "bfloat16", "float32")
    good = layer_norm(x, w, b, "bfloat16", "float32")
    dgood = layer_norm_grad(x, w, dy, "bfloat16", "float32")[0]
    for value in (np.nan, np.inf, -np.inf):
        bad = x.copy()
        bad[5, K // 2] = value
        y = layer_norm(bad, w, b, "bfloat16", "float32")
        dx = layer_norm_grad(bad, w, dy, "bfloat16", "float32")[0]
        rest = np.arange(12) != 5
        assert np.isnan(y[5]).all() and np.isnan(dx[5]).all()
        np.testing.assert_array_equal(y[rest], good[rest])
        np.testing.assert_array_equal(dx[rest], dgood[rest])


def test_no_rows():
    w = np.ones(9, np.float32)
    assert layer_norm(np.zeros((0, 9), np.float32), w, w, "float32", "float32").shape == (0, 9)
    dx, dw, db = layer_norm_grad(np.zeros((0, 9), np.float32), w, np.zeros((0, 9), np.float32), "float32", "float32")
    assert dx.shape == (0, 9) and not dw.any() and not db.any()


def test_gradients_against_differences():
    """d sum(y dy) along a direction, by the float64 form of y at x, w, b moved both ways:
    the gradients are linear in dy, the differences off by the third derivative."""
    rng = np.random.default_rng(8)
    rows, K, h = 6, 40, 1e-4
    x, w, b, dy = inputs(8, rows, K, "float32", "float32")
    dx, dw, db = (g.astype(np.float64) for g in layer_norm_grad(x, w, dy, "float32", "float32"))
    for _ in range(5):
        vx, vw, vb = rng.normal(size=x.shape), rng.normal(size=K), rng.normal(size=K)

        def loss(s):
            m = x + s * vx
            c = m - m.mean(1, keepdims=True)
            z = c / np.sqrt((c * c).mean(1, keepdims=True) + np.float64(np.float32(1e-5)))
            return ((z * (w + s * vw) + b + s * vb) * dy).sum()

        got = (dx * vx).sum() + (dw * vw).sum() + (db * vb).sum()
        scale = np.abs(dx * vx).sum() + np.abs(dw * vw).sum() + np.abs(db * vb).sum()
        # h^2 times a third derivative of order 1, and 2^-53 / h of the difference
        assert abs(got - (loss(h) - loss(-h)) / (2 * h)) < 1e-5 * scale


def test_same_bits_on_a_stream_of_its_own():
    x, w, b, dy = inputs(9, 3000, 777, "bfloat16", "float32")
    stream = capi.lib().xtc_hip_stream_create()
    for a, c in zip(layer_norm_grad(x, w, dy, "bfloat16", "float32"), layer_norm_grad(x, w, dy, "bfloat16", "float32", stream=stream)):
        np.testing.assert_array_equal(a, c)
    np.testing.assert_array_equal(layer_norm(x, w, b, "bfloat16", "float32"), layer_norm(x, w, b, "bfloat16", "float32", stream=stream))
    capi.check(capi.lib().xtc_hip_stream_destroy(stream))


@pytest.mark.parametrize("dtype,rows,K", [("bfloat16", 16448, 4104), ("bfloat16", 131200, 515), ("float32", 2112, 16384)])
def test_results_past_the_caches(dtype, rows, K):
    """A result of more than 128 MB is stored past the caches: the bits of a small call, whose
    rows it repeats."""
    rng = np.random.default_rng(K)
    x, dy = (rounded(rng.normal(size=(64, K)), dtype) for _ in range(2))
    w, b = (rng.normal(size=K).astype(np.float32) for _ in range(2))
    assert rows * K * (2 if dtype == "bfloat16" else 4) > 128 << 20
    big = np.tile(x, (-(-rows // 64), 1))[:rows]
    y = layer_norm(big, w, b, dtype, "float32")
    small = layer_norm(x, w, b, dtype, "float32")
    assert np.array_equal(y, np.tile(small, (-(-rows // 64), 1))[:rows])
    del y
    dx = layer_norm_grad(big, w, np.tile(dy, (-(-rows // 64), 1))[:rows], dtype, "float32", want=(True, False, False))[0]
    small = layer_norm_grad(x, w, dy, dtype, "float32", want=(True, False, False))[0]
    assert np.array_equal(dx, np.tile(small, (-(-rows // 64), 1))[:rows])
