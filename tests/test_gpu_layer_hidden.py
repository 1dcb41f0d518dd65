# SPDX-License-Identifier: BSD-3-Clause
"""The expert layer on the GPU with activations in fp32 between its products.

Bounds: layer_calls.plain_layer's for a layer that rounds nothing between its products,
and for the three numbers that an activation is split into 3 H additions instead of H: 2 H
units of 24 bits more, 2 H 2^-23."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import xtc_amd.graphs.xtc.op as O
from expert_calls import Mem, ints, padded, rounded
from layer_calls import U, check_close, finish, layer_desc, plain_layer
from test_gpu_expert_layer import SIZES, inputs, pack
from test_gpu_layer_graphs import payload
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device

pytestmark = pytest.mark.gpu

WEIGHTS = ["dense", "fp8", "mx4"]


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def layer(x, router, up, down, top_k, weights="dense", activation="swiglu", normalize=True, pad=(0, 0), shift=0, stream=None, hidden=1):
    """up, down: arrays, or (codes, scales) of 8-bit or 4-bit matrices; bf16."""
    T, K = x.shape
    ups, downs = ((up, None), (down, None)) if weights == "dense" else (up, down)
    d = layer_desc(x, router, ups[0].shape[1] // (2 if activation == "swiglu" else 1), top_k, "bfloat16", weights, activation, normalize, pad, stream)
    d.hidden_f32 = hidden
    print(f"[layer] T {T} E {len(router)} top {top_k} K {K} H {d.H} {weights} {activation} hidden {hidden}", flush=True)
    L = capi.lib()
    L.xtc_hip_expert_layer_workspace.restype = ctypes.c_uint64
    need = L.xtc_hip_expert_layer_workspace(ctypes.byref(d))
    kind = "bfloat16" if weights == "dense" else "uint8"
    mems = [Mem(padded(x, K + pad[0]), "bfloat16", shift), Mem(router, "bfloat16"),
            *(m for c, s in (ups, downs) for m in (Mem(c, kind, shift if weights == "dense" else 0), Mem(s, "uint8", 1) if s is not None else None))]
    ws = Mem(np.full(need, 0xFF), "uint8")
    out = Mem(padded(np.full((T, K), 7.0), K + pad[1]), "bfloat16")
    capi.check(L.xtc_hip_expert_layer(ctypes.byref(d), *[m and m.ptr for m in mems], ws.ptr, ctypes.c_uint64(need), out.ptr))
    ws.numpy()  # nothing around it was written
    (y,) = finish([*mems, ws], [out], stream)
    assert np.isnan(y[:, K:]).all(), "written past the columns"
    return y[:, :K]


def large(T, H):
    """Whole numbers whose activations need up to 19 bits, for one expert of two."""
    K = 64
    x, router = ints(1, (T, K), 3), np.zeros((2, K), np.float32)
    x[:, 0] = 200  # all of a softmax that holds exp(-200) beside it
    router[1, 0] = 1
    up, down = ints(2, (2, H, K), 4), np.zeros((2, K, H), np.float32)
    up[:, :, 0] = ints(3, (2, H), 4) * 512
    # few enough for sums below 2^24
    down[:, np.arange(K), np.random.default_rng(4).integers(0, H, K)] = 1
    down[:, np.arange(K), np.random.default_rng(5).integers(0, H, K)] = -4
    hidden = np.maximum(x.astype(np.float64) @ up[1].T, 0)
    assert hidden.max() > 2**17 and (hidden % 2 == 1).any()
    return x, router, up, down, hidden @ down[1].T


@pytest.mark.parametrize("T,H", [(1, 40), (7, 40), (64, 200)])
def test_activations_past_bf16_are_kept(T, H):
    x, router, up, down, want = large(T, H)
    np.testing.assert_array_equal(layer(x, router, up, down, 1, activation="relu", normalize=False), rounded(want, "bfloat16"))


@pytest.mark.parametrize("hidden", ["float32", "bfloat16", None])
def test_the_operator_keeps_fp32_unless_asked(hidden):
    """By default too; rounded to bf16 where it says so, other numbers."""
    x, router, up, down, want = large(20, 72)
    given = [O.tensor(a.shape, "bfloat16") for a in (x, router, up, down)]
    attrs = {} if hidden is None else {"hidden_dtype": hidden}
    with O.graph(name="hidden") as gb:
        O.expert_layer(*given, top_k=1, activation="relu", normalize=False, **attrs)
    (got,) = payload(gb.graph, [x, router, up, down], [np.empty(x.shape, np.float32)], 2.0**-8)
    assert np.array_equal(got, rounded(want, "bfloat16")) == (hidden != "bfloat16")


def check(seed, T, E, top_k, K, H, weights, activation="swiglu", normalize=True, **how):
    x, router, (up, upv), (down, downv) = inputs(seed, T, E, K, H, "bfloat16", weights, activation, top_k)
    got = layer(x, router, up, down, top_k, weights, activation, normalize, **how)
    check_close(got, *plain_layer(x, router, upv, downv, top_k, activation, normalize, 2 * H * 2 * U), "bfloat16")


@pytest.mark.parametrize("weights", WEIGHTS)
@pytest.mark.parametrize("activation", ["swiglu", "relu"])
@pytest.mark.parametrize("T,E,top_k,K,H", SIZES)
def test_layer(T, E, top_k, K, H, activation, weights):
    check(T + E, T, E, top_k, K, H, weights, activation, normalize=(T + K) % 2 == 0)


@pytest.mark.parametrize("weights", WEIGHTS)
@pytest.mark.parametrize("T,K,H", [(4, 256, 4096), (33, 1500, 1100), (64, 2048, 1536)])
def test_wide_slices(T, K, H, weights):
    check(T, T, 32, 2, K, H, weights)


@pytest.mark.parametrize("weights", WEIGHTS)
@pytest.mark.parametrize("pad,shift", [((1, 3), 1), ((8, 8), 0)])
def test_strides_and_alignment(pad, shift, weights):
    check(1, 9, 6, 2, 140, 75, weights, pad=pad, shift=shift)


@pytest.mark.parametrize("weights", WEIGHTS)
def test_a_bad_token_stays_alone(weights):
    x, router, (up, _), (down, _) = inputs(7, 20, 6, 96, 64, "bfloat16", weights, "swiglu", 2)
    good = layer(x, router, up, down, 2, weights)
    for value in (np.nan, np.inf, -np.inf):
        bad = x.copy()
        bad[11, 5] = value
        y = layer(bad, router, up, down, 2, weights)
        assert np.isnan(y[11]).all()
        rest = np.arange(20) != 11
        np.testing.assert_array_equal(y[rest], good[rest])


def test_activations_at_the_end_of_the_range():
    """Past bf16's largest number and below fp32's; infinite; and a NaN of infinities."""
    most = np.float32(255 * 2.0**120)  # bf16's
    x, router = np.ones((1, 2), np.float32), np.zeros((1, 2), np.float32)
    up = np.array([[[most, 1.5 * 2.0**119], [most, most], [1, 1], [0, 0]]], np.float32)
    assert 2.0**128 - 2.0**119 < float(up[0, 0].astype(np.float64).sum()) < 2.0**128 - 2.0**103
    for column, want in ((0, float(up[0, 0].astype(np.float64).sum()) * 2.0**-100), (1, np.inf), (2, 2 * 2.0**-100), (3, 0.0)):
        down = np.zeros((1, 2, 4), np.float32)
        down[0, :, column] = 2.0**-100
        # the others' zeros times the infinite activation are NaN, as in any product
        one = up[:, column : column + 1], down[:, :, column : column + 1]
        got = layer(x, router, *one, 1, activation="relu")
        np.testing.assert_array_equal(got, rounded(np.full((1, 2), want), "bfloat16"))
    assert np.isnan(layer(x, router, up, np.full((1, 2, 4), 2.0**-100, np.float32) * np.array([1, 0, 1, 1]), 1, activation="relu")).all()


@pytest.mark.parametrize("weights", WEIGHTS)
def test_same_bits_again_and_on_a_stream_of_its_own(weights):
    x, router, (up, _), (down, _) = inputs(9, 30, 16, 512, 256, "bfloat16", weights, "swiglu", 4)
    stream = capi.lib().xtc_hip_stream_create()
    first = layer(x, router, up, down, 4, weights)
    for s in (None, stream, stream):
        np.testing.assert_array_equal(first, layer(x, router, up, down, 4, weights, stream=s))
    capi.check(capi.lib().xtc_hip_stream_destroy(stream))


@pytest.mark.parametrize("weights", WEIGHTS)
def test_a_token_keeps_its_bits_beside_others(weights):
    """One expert for all: the first tokens of calls of more and more."""
    x, router, (up, _), (down, _) = inputs(10, 64, 1, 200, 120, "bfloat16", weights, "swiglu", 1)
    most = layer(x, router, up, down, 1, weights)
    for T in (1, 5, 16, 17):
        np.testing.assert_array_equal(layer(x[:T], router, up, down, 1, weights), most[:T])
