# SPDX-License-Identifier: BSD-3-Clause
"""The layer of experts for a few tokens on the GPU against float64, within what
layer_calls.plain_layer derives, and half a step of a bf16 result.  Whole numbers with
relu, and weights that are powers of two, are compared for equality."""

from __future__ import annotations

import numpy as np
import pytest

from expert_calls import ints, rounded
from layer_calls import HALF, check_close, expert_layer, plain_layer, unclear
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.fp8 import fp8_codes, fp8_scales, fp8_values
from xtc_amd.utils.mx4 import mx4_codes, mx4_scales, mx4_values

pytestmark = pytest.mark.gpu

KINDS = [("float32", "dense"), ("bfloat16", "dense"), ("bfloat16", "fp8"), ("bfloat16", "mx4")]


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def pack(w, weights):
    """The matrices as the call takes them, and their values in float64."""
    if weights == "fp8":
        s = fp8_scales(w, 128)
        c = fp8_codes(w, s, 128)
        return (c, s), fp8_values(c, s, w.shape[2], np.float64)
    if weights == "mx4":
        s = mx4_scales(w)
        c = mx4_codes(w, s)
        return (c, s), mx4_values(c, s, w.shape[2], np.float64)
    return w, w.astype(np.float64)


def inputs(seed, T, E, K, H, dtype, weights, activation, top_k):
    """Tokens whose choice of top_k experts rounding could change are drawn again."""
    rng = np.random.default_rng(seed)
    x, router = rounded(rng.normal(size=(T, K)), dtype), rounded(rng.normal(0, 1.5 * K**-0.5, (E, K)), dtype)
    while (again := unclear(x, router, top_k)).any():
        x[again] = rounded(rng.normal(size=(again.sum(), K)), dtype)
    up = rounded(rng.normal(0, K**-0.5, (E, 2 * H if activation == "swiglu" else H, K)), dtype)
    down = rounded(rng.normal(0, H**-0.5, (E, K, H)), dtype)
    return x, router, pack(up, weights), pack(down, weights)


def check(seed, T, E, top_k, K, H, dtype, weights, activation="swiglu", normalize=True, **how):
    print(f"[layer] T {T} E {E} top {top_k} K {K} H {H} {dtype} {weights} {activation} {normalize}", flush=True)
    x, router, (up, upv), (down, downv) = inputs(seed, T, E, K, H, dtype, weights, activation, top_k)
    got = expert_layer(x, router, up, down, top_k, dtype, weights, activation, normalize, **how)
    # a bf16 layer's activations are bf16 numbers: half a step, as its result
    mid = HALF["bfloat16"] if dtype == "bfloat16" else 0.0
    check_close(got, *plain_layer(x, router, upv, downv, top_k, activation, normalize, mid), dtype)


# one token to all, one expert to many, sizes of no whole run or slice, both forms of the
# logits, tokens beyond one and two tiles at one expert
SIZES = [(1, 1, 1, 1, 1), (1, 8, 2, 64, 32), (1, 8, 2, 1024, 512), (3, 5, 5, 33, 17), (2, 64, 4, 256, 96), (16, 16, 2, 130, 100), (17, 4, 1, 300, 60),
         (64, 2, 1, 200, 129), (64, 8, 3, 512, 256), (40, 256, 16, 100, 40), (64, 1, 1, 77, 50), (5, 33, 2, 2050, 70), (64, 64, 8, 640, 128),
         (8, 3, 2, 128, 2100)]


@pytest.mark.parametrize("dtype,weights", KINDS)
@pytest.mark.parametrize("activation", ["swiglu", "relu"])
@pytest.mark.parametrize("T,E,top_k,K,H", SIZES)
def test_layer(T, E, top_k, K, H, activation, dtype, weights):
    check(T + E, T, E, top_k, K, H, dtype, weights, activation, normalize=(T + K) % 2 == 0)


@pytest.mark.parametrize("dtype,weights", KINDS)
@pytest.mark.parametrize("T,K,H", [(4, 256, 4096), (33, 1500, 1100), (64, 2048, 1536)])
def test_wide_slices(T, K, H, dtype, weights):
    check(T, T, 32, 2, K, H, dtype, weights)


@pytest.mark.parametrize("dtype,weights", KINDS)
@pytest.mark.parametrize("pad,shift", [((1, 3), 1), ((8, 8), 0)])
def test_strides_and_alignment(pad, shift, dtype, weights):
    check(1, 9, 6, 2, 140, 75, dtype, weights, pad=pad, shift=shift)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_ties_go_to_the_lowest_expert(dtype):
    """Equal logits, the two zeros among them: the first experts; weights 1 / top_k."""
    T, E, K, H = 5, 12, 32, 32
    x, router = ints(1, (T, K), 2), np.zeros((E, K), np.float32)
    router[3:7] = -0.0
    up, down = ints(2, (E, H, K), 2), ints(3, (E, K, H), 2)
    for top_k in (1, 2, 4):
        got = expert_layer(x, router, up, down, top_k, dtype, activation="relu")
        want = sum(np.maximum(x @ up[e].T, 0) @ down[e].T for e in range(top_k)) / top_k
        np.testing.assert_array_equal(got, rounded(want, dtype))
    # one expert ahead: all of a softmax that holds exp(-200) beside it
    router[9, 0] = 1
    x[:, 0] = 200
    got = expert_layer(x, router, up, down, 1, dtype, activation="relu", normalize=False)
    mid = rounded(np.maximum(x @ up[9].T, 0), dtype)  # past 256: a bf16 layer's activations are rounded
    np.testing.assert_array_equal(got, rounded(mid @ down[9].T, dtype))


def test_the_same_expert_for_all():
    """64 tokens at one of 8 experts: four tiles, every other workgroup empty."""
    T, E, K, H = 64, 8, 64, 48
    x = ints(4, (T, K), 2)
    x[:, 0] = 8
    router = np.zeros((E, K), np.float32)
    router[5, 0] = 16
    up, down = ints(5, (E, H, K), 2), ints(6, (E, K, H), 2)
    got = expert_layer(x, router, up, down, 1, "float32", activation="relu")
    np.testing.assert_array_equal(got, np.maximum(x @ up[5].T, 0) @ down[5].T)


@pytest.mark.parametrize("dtype,weights", KINDS)
def test_a_bad_token_stays_alone(dtype, weights):
    x, router, (up, _), (down, _) = inputs(7, 20, 6, 96, 64, dtype, weights, "swiglu", 2)
    good = expert_layer(x, router, up, down, 2, dtype, weights)
    for value in (np.nan, np.inf, -np.inf):
        bad = x.copy()
        bad[11, 5] = value
        y = expert_layer(bad, router, up, down, 2, dtype, weights)
        assert np.isnan(y[11]).all()
        rest = np.arange(20) != 11
        np.testing.assert_array_equal(y[rest], good[rest])


@pytest.mark.parametrize("dtype,weights", KINDS)
def test_a_bad_expert_reaches_its_tokens_alone(dtype, weights):
    x, router, (up, _), (down, _) = inputs(8, 24, 6, 96, 64, dtype, weights, "swiglu", 1)
    good = expert_layer(x, router, up, down, 1, dtype, weights)
    chosen = np.argmax(x.astype(np.float64) @ router.astype(np.float64).T, axis=1)
    if weights == "dense":
        up = up.copy()
        up[2, 3, 4] = np.nan
    else:
        up = (up[0], up[1].copy())
        up[1][2, 0, 0] = 255
    y = expert_layer(x, router, up, down, 1, dtype, weights)
    assert (chosen == 2).any() and np.isnan(y[chosen == 2]).all()
    np.testing.assert_array_equal(y[chosen != 2], good[chosen != 2])


@pytest.mark.parametrize("dtype,weights", KINDS)
def test_same_bits_again_and_on_a_stream_of_its_own(dtype, weights):
    x, router, (up, _), (down, _) = inputs(9, 30, 16, 512, 256, dtype, weights, "swiglu", 4)
    stream = capi.lib().xtc_hip_stream_create()
    first = expert_layer(x, router, up, down, 4, dtype, weights)
    for s in (None, stream, stream):
        np.testing.assert_array_equal(first, expert_layer(x, router, up, down, 4, dtype, weights, stream=s))
    capi.check(capi.lib().xtc_hip_stream_destroy(stream))


def test_no_tokens():
    up, down = np.zeros((2, 8, 4), np.float32), np.zeros((2, 4, 4), np.float32)
    assert expert_layer(np.zeros((0, 4), np.float32), np.zeros((2, 4), np.float32), up, down, 1, "float32").shape == (0, 4)
