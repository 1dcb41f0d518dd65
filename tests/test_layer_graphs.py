# SPDX-License-Identifier: BSD-3-Clause
"""Graphs with layer norm, 8-bit operands and the expert layer, on the CPU: types,
refusals, the numpy semantics against brute force, what the HIP backend makes of
them, and the example's graphs."""

from __future__ import annotations

import ctypes
import re
from fractions import Fraction
from math import log2
from pathlib import Path

import numpy as np
import pytest

import xtc_amd.graphs.xtc.op as O
from test_expert_graphs import build, forward
from xtc_amd.backends.hip import Backend
from xtc_amd.backends.hip.lowering import NORM_PARTS, expert_layer_attrs, expert_layer_workspace
from xtc_amd.graphs.xtc.layer_operators import MOST_CHOSEN, MOST_EXPERTS, MOST_TOKENS
from xtc_amd.utils.fp8 import fp8_codes, fp8_scales, fp8_values
from xtc_amd.utils.mx4 import mx4_codes, mx4_scales

F, B, U8 = "float32", "bfloat16", "uint8"
ROOT = Path(__file__).resolve().parents[1]


def kinds(graph):
    return [ln.kind for ln in Backend(graph).plan.launches]


def compiled(graph):
    backend = Backend(graph)
    return backend.get_compiler(schedule_policy="strict").compile(backend.get_scheduler().schedule()).source


# ---------------------------------------------------------------- the formats


def exact_values():
    """The magnitudes of the codes 0 to 126, from their bits."""
    return [Fraction(c & 7, 512) if c < 8 else Fraction(8 + (c & 7), 8) * Fraction(2) ** ((c >> 3) - 7) for c in range(127)]


def brute_block(block):
    """(scale byte, codes) of numbers in exact arithmetic."""
    if not np.isfinite(block).all():
        return 255, [0] * block.size
    top = max(abs(Fraction(float(v))) for v in block)
    s = next(s for s in range(255) if top <= 448 * Fraction(2) ** (s - 127))
    values, codes = exact_values(), []
    for v in block:
        y = abs(Fraction(float(v))) / Fraction(2) ** (s - 127)
        codes.append(min(range(127), key=lambda i: (abs(values[i] - y), i % 2)) | (128 if np.signbit(v) else 0))
    return s, codes


def test_fp8_against_exact_arithmetic():
    rng = np.random.default_rng(0)
    x = (rng.normal(size=(12, 128)) * np.exp2(rng.integers(-9, 9, (12, 128)))).astype(np.float32)
    x[0] = 0
    x[1, 5:] = 0
    x[2], x[3] = np.ldexp(np.float32(1), -140), np.ldexp(np.float32(3), -126)
    x[4, 7], x[5, 100], x[6, 1] = np.inf, np.nan, 3.4e38
    x[7, :4], x[8, :4] = 448, 449  # the largest code, and one past it
    x[9] = -x[9]
    values = exact_values()
    x[10, :126] = [float((a + b) / 2) for a, b in zip(values, values[1:])]
    scales = fp8_scales(x)
    codes = fp8_codes(x, scales)
    for r in range(12):
        s, want = brute_block(x[r])
        assert scales[r, 0] == s, r
        assert codes[r].tolist() == want, r
    values = fp8_values(codes, scales, dtype=np.float64)
    assert np.isnan(values[4]).all() and not values[0].any() and values[7, 0] == 448 and values[8, 0] == 448
    assert values[6, 1] == 2.0**128  # past fp32's range: 3.4e38 to 4 bits
    again = fp8_scales(values[7:].astype(np.float32))
    np.testing.assert_array_equal(fp8_values(fp8_codes(values[7:], again), again, dtype=np.float64), values[7:])


def test_fp8_blocks_of_rows():
    x = np.random.default_rng(1).normal(size=(2, 200, 300)).astype(np.float32)
    x[1, 130, 260] = 1e6
    s = fp8_scales(x, 128)
    assert s.shape == (2, 2, 3)
    for e in range(2):
        for i in range(2):
            for j in range(3):
                top = np.abs(x[e, 128 * i : 128 * i + 128, 128 * j : 128 * j + 128]).max()
                assert top <= 448 * 2.0 ** (int(s[e, i, j]) - 127) < 2 * top
    c = fp8_codes(x, s, 128)
    assert c.shape == (2, 200, 384) and not c[..., 300:].any()
    v = fp8_values(c, s, 300, np.float64)
    step = np.maximum(2.0**-4 * np.abs(x), (2.0 ** (s.astype(int) - 127 - 10)).repeat(128, -1).repeat(128, -2)[:, :200, :300])
    assert (np.abs(v - x) <= step).all()


def test_codes_for_other_scales():
    x = np.array([[1e9, -1e9, np.inf, -np.inf, np.nan, -np.nan, 1.0, 0.0]], np.float32)
    codes = fp8_codes(x, np.array([[127]], np.uint8))[0, :8]
    assert codes.tolist() == [0x7E, 0xFE, 0x7E, 0xFE, 0x7F | (np.signbit(x[0, 4]) << 7), 0x7F | (np.signbit(x[0, 5]) << 7), 0x38, 0]
    assert not fp8_codes(x, np.array([[255]], np.uint8)).any()


# ------------------------------------------------------------------ semantics


def test_layer_norm_and_gradients_against_differences():
    rng = np.random.default_rng(2)
    x, w, b, dy = rng.normal(size=(6, 10)), rng.normal(size=10), rng.normal(size=10), rng.normal(size=(6, 10))
    x, w, b, dy = (a.astype(np.float32) for a in (x, w, b, dy))
    types = [((6, 10), F), ((10,), F), ((10,), F)]
    graph = build(lambda *a: O.layer_norm(*a, eps=1e-3), *types)

    def y64(x, w, b):
        x = x.astype(np.float64)
        c = x - x.mean(-1, keepdims=True)
        return c / np.sqrt((c * c).mean(-1, keepdims=True) + np.float64(np.float32(1e-3))) * w + b

    np.testing.assert_allclose(forward(graph, x, w, b)[0], y64(x, w, b), rtol=2**-22, atol=2**-22)
    grads = build(lambda x, w, dy: O.outputs(*O.layer_norm_grad(x, w, dy, eps=1e-3)), types[0], types[1], types[0])
    dx, dw, db = forward(grads, x, w, dy)
    h = 2.0**-12  # central differences: errors of h^2 and of 2^-53 / h
    for got, at in ((dx, 0), (dw, 1), (db, 2)):
        args = [x.astype(np.float64), w.astype(np.float64), b.astype(np.float64)]
        for i in np.ndindex(got.shape):
            up, down = ([a.copy() for a in args] for _ in range(2))
            up[at][i] += h
            down[at][i] -= h
            want = ((y64(*up) - y64(*down)) * dy).sum() / (2 * h)
            assert abs(got[i] - want) < 1e-5 * (1 + abs(want)), (at, i)


def test_expert_layer_against_a_loop():
    rng = np.random.default_rng(3)
    T, E, K, H = 7, 5, 12, 6
    x, router = (rng.normal(size=s).astype(np.float32) for s in ((T, K), (E, K)))
    x[3] = 0  # all logits equal
    for act, rows in (("swiglu", 2 * H), ("relu", H)):
        up, down = (rng.normal(size=s).astype(np.float32) for s in ((E, rows, K), (E, K, H)))
        for normalize in (True, False):
            graph = build(lambda *a: O.expert_layer(*a, top_k=3, activation=act, normalize=normalize), ((T, K), F), ((E, K), F),
                          (up.shape, F), (down.shape, F))
            (y,) = forward(graph, x, router, up, down)
            for t in range(T):
                logits = x[t].astype(np.float64) @ router.T.astype(np.float64)
                p = np.exp(logits - logits.max())
                p /= p.sum()
                order = sorted(range(E), key=lambda e: (-np.float32(logits[e]), e))[:3]
                if t == 3:
                    assert order == [0, 1, 2]
                total = sum(p[e] for e in order) if normalize else 1.0
                want = np.zeros(K)
                for e in order:
                    u = up[e].astype(np.float64) @ x[t]
                    a = u[:H] / (1 + np.exp(-u[:H])) * u[H:] if act == "swiglu" else np.maximum(u, 0)
                    want += p[e] / total * (down[e].astype(np.float64) @ a)
                np.testing.assert_allclose(y[t], want, rtol=1e-6, atol=1e-6)


def test_types_and_refusals():
    x, w, dy = ((4, 8), F), ((8,), F), ((4, 8), F)
    wrong = [
        ("float32 or bfloat16 rows", O.layer_norm, [((4, 8), U8), w, w]),
        ("parameters must be", O.layer_norm, [x, ((7,), F), ((7,), F)]),
        ("parameters must be", O.layer_norm, [x, w, ((8,), B)]),
        ("parameters must be", O.layer_norm, [x, ((8,), B), ((8,), B)]),
        ("eps", lambda *a: O.layer_norm(*a, eps=-1), [x, w, w]),
        ("of one type and shape", O.layer_norm_grad_x, [x, w, ((4, 8), B)]),
        ("of one type and shape", O.layer_norm_grad_weight, [x, ((5, 8), F)]),
        ("rank >= 2", O.fp8_scales, [((8,), F)]),
        ("blocks of 64 rows", lambda a: O.fp8_scales(a, rows=64), [x]),
        ("do not match", O.fp8_codes, [x, ((4, 2), U8)]),
        ("do not match", lambda a, s: O.fp8_codes(a, s, rows=128), [((200, 8), F), ((200, 1), U8)]),
        ("must be uint8", O.fp8_dequantize, [((4, 100), U8), ((4, 1), U8)]),
        ("do not hold", lambda c, s: O.fp8_dequantize(c, s, size=129), [((4, 128), U8), ((4, 1), U8)]),
        ("one depth", O.fp8_matmul, [((4, 128), U8), ((4, 1), U8), ((4, 256), U8), ((4, 2), U8)]),
        ("a has a scale", O.fp8_matmul, [((4, 128), U8), ((1, 1), U8), ((4, 128), U8), ((4, 1), U8)]),
    ]
    for why, fn, types in wrong:
        with pytest.raises(ValueError, match=why):
            build(fn, *types).outputs_types

    def layer(T=4, E=8, K=64, H=32, up=None, down=None, router=B, **attrs):
        rows = H if attrs.get("activation") == "relu" else 2 * H
        up, down = up or ((E, rows, K), B), down or ((E, K, H), B)
        return build(lambda *a: O.expert_layer(*a, **attrs), ((T, K), B), ((E, K), router), up, down).outputs_types

    assert layer()[0].constant_shape == (4, 64)
    for why, kw in (("of one type", dict(router=F)), ("at most", dict(T=65)), ("at most", dict(E=257)), ("from 1 to", dict(top_k=0)),
                    ("from 1 to", dict(top_k=9)), ("from 1 to", dict(E=64, top_k=17)), ("neither", dict(activation="gelu")),
                    ("of x's type", dict(up=((8, 64, 64), F))), ("do not match", dict(down=((8, 64, 33), B))),
                    ("odd number", dict(up=((8, 63, 64), B)))):
        with pytest.raises(ValueError, match=why):
            layer(**kw)
    with pytest.raises(ValueError, match="codes and scales"):
        build(lambda x, r, a, b, c, d: O.expert_layer(x, r, (a, b), (c, d)), ((4, 64), B), ((8, 64), B), ((8, 64, 128), U8),
              ((8, 64, 1), U8), ((8, 64, 128), U8), ((8, 1, 1), U8)).outputs_types
    with pytest.raises(TypeError, match="4 or 6"):
        build(lambda x, r, a, b, c: O.expert_layer(x, r, (a, b), c), ((4, 64), B), ((8, 64), B), ((8, 64, 64), U8), ((8, 1, 1), U8),
              ((8, 64, 32), U8))


# ------------------------------------------------------------------- lowering


@pytest.mark.parametrize("want,fn", [
    (["layer_norm", "layer_norm_grad"], lambda x, w, dy: O.outputs(O.layer_norm(x, w, w), *O.layer_norm_grad(x, w, dy))),
    (["layer_norm_grad"], lambda x, w, dy: O.layer_norm_grad_x(x, w, dy)),
    (["layer_norm_grad"], lambda x, w, dy: O.outputs(O.layer_norm_grad_weight(x, dy), O.layer_norm_grad_bias(dy))),
    (["layer_norm_grad"], lambda x, w, dy: O.layer_norm_grad_bias(dy)),
    # sums first: the rows' gradient is a call of its own, and nothing is summed twice
    (["layer_norm_grad", "layer_norm_grad"], lambda x, w, dy: O.outputs(
        *reversed(O.layer_norm_grad(x, w, dy)[1:2]), O.layer_norm_grad_bias(dy), O.layer_norm_grad_x(x, w, dy))),
    # another eps is another norm
    (["layer_norm_grad", "layer_norm_grad"], lambda x, w, dy: O.outputs(O.layer_norm_grad_x(x, w, dy), O.layer_norm_grad_weight(x, dy, eps=1e-3))),
])
def test_norm_plans(want, fn):
    graph = build(fn, ((64, 256), F), ((256,), F), ((64, 256), F))
    assert kinds(graph)[: len(want)] == want and len(kinds(graph)) <= len(want) + 1
    compiled(graph)


@pytest.mark.parametrize("want,fn", [
    (["fp8_quantize"], lambda x: O.fp8_scales(x)),
    (["fp8_quantize"], lambda x: O.outputs(*O.fp8_quantize(x))),
    (["fp8_quantize"], lambda x: O.outputs(*O.fp8_quantize(x), *O.fp8_quantize(x, transpose=True))),
    (["fp8_quantize"], lambda x: O.outputs(*O.fp8_quantize(x, rows=128, transpose=True), *O.fp8_quantize(x, rows=128))),
    (["fp8_quantize"], lambda x: (lambda q: O.outputs(*q, O.fp8_dequantize(*q, size=256)))(O.fp8_quantize(x))),
    # one block size and the other share nothing
    (["fp8_quantize"] * 2, lambda x: O.outputs(*O.fp8_quantize(x), *O.fp8_quantize(x, rows=128, transpose=True))),
    (["relu", "fp8_quantize", "fp8_encode"], lambda x: O.fp8_codes(O.relu(x), O.fp8_scales(x))),
    (["fp8_quantize", "fp8_dequantize"], lambda x: O.fp8_dequantize(*O.fp8_quantize(x), out_dtype="bfloat16")),
    (["fp8_quantize", "fp8_matmul"], lambda x: (lambda q: O.fp8_matmul(*q, *q))(O.fp8_quantize(x))),
])
def test_fp8_plans(want, fn):
    graph = build(fn, ((200, 256), F))
    assert sorted(kinds(graph)) == sorted(want)
    compiled(graph)


def test_constants_are_the_librarys():
    header = (ROOT / "include" / "xtc_hip.h").read_text()
    assert int(re.search(r"XTC_HIP_LAYER_NORM_PARTS (\d+)", header)[1]) == NORM_PARTS
    assert f"(<= {MOST_TOKENS};" in header and f"(<= {MOST_EXPERTS})" in header and f"<= {MOST_CHOSEN} and E" in header


def test_workspace_is_the_librarys():
    from xtc_amd.runtimes.hip import capi

    if not capi.library_available():
        pytest.skip("libxtc_hip.so is not built")
    lib = capi.lib()
    lib.xtc_hip_expert_layer_workspace.restype = ctypes.c_uint64
    for T, E, top_k, K, H in ((1, 1, 1, 1, 1), (64, 256, 16, 4096, 2048), (17, 33, 3, 1000, 333), (4, 8, 2, 64, 31)):
        for activation in ("relu", "swiglu"):
            up = 2 * H if activation == "swiglu" else H
            graph = build(lambda *a: O.expert_layer(*a, top_k=top_k, activation=activation), ((T, K), B), ((E, K), B), ((E, up, K), B), ((E, K, H), B))
            node = next(n for n in graph.nodes.values() if n.operation.name == "expert_layer")
            attrs = expert_layer_attrs(node.operation, [(T, K), (E, K), (E, up, K), (E, K, H)], B)
            d = capi.ExpertLayerDesc(dtype=1, weights=0, activation=int(activation == "swiglu"), T=T, E=E, K=K, H=H, top_k=top_k)
            assert expert_layer_workspace(attrs) == lib.xtc_hip_expert_layer_workspace(ctypes.byref(d)) > 0, capi.last_error()


def test_example_graphs():
    """Their launches, and the 8-bit step against products of whole numbers."""
    from xtc_amd.cli import experts

    T, E, K, N = 20, 3, 64, 96
    graphs = {g.name: g for g in (experts.norm_graph(T, K), experts.project_graph(T, K, N),
                                  *(experts.few_graph(T, E, K, N, w) for w in ("dense", "fp8", "mx4")))}
    for g in graphs.values():
        compiled(g)
    assert {name: kinds(g) for name, g in graphs.items()} == {
        "experts_norm": ["layer_norm", "layer_norm_grad"],
        "experts_project": ["fp8_quantize", "fp8_quantize", "fp8_matmul", "fp8_quantize", "fp8_matmul", "fp8_matmul"],
        **{f"experts_few_{w}": ["layer_norm", "expert_layer"] for w in ("dense", "fp8", "mx4")}}
    rng = np.random.default_rng(6)
    x, w, dy = (rng.integers(-8, 9, s).astype(np.float32) for s in ((T, K), (N, K), (T, N)))
    y, dx, dw = forward(graphs["experts_project"], x, w, dy)
    assert log2(8 * 8 * 96) < 24  # whole numbers that fp32 holds
    np.testing.assert_array_equal(dw, dy.T @ x)
    for got, want in ((y, x @ w.T), (dx, dy @ w)):
        assert (np.abs(got - want) <= 2.0**-8 * np.abs(want)).all()
    up, down = rng.normal(0, 0.1, (E, 2 * N, K)).astype(np.float32), rng.normal(0, 0.1, (E, K, N)).astype(np.float32)
    rest = (rng.normal(size=(T, K)).astype(np.float32), np.ones(K, np.float32), np.zeros(K, np.float32), rng.normal(size=(E, K)).astype(np.float32))
    dense, = forward(graphs["experts_few_dense"], *rest, up, down)
    pairs = [m for a in (up, down) for s in [fp8_scales(a, 128)] for m in (fp8_codes(a, s, 128), s)]
    eight, = forward(graphs["experts_few_fp8"], *rest, *pairs)
    pairs = [m for a in (up, down) for s in [mx4_scales(a)] for m in (mx4_codes(a, s), s)]
    four, = forward(graphs["experts_few_mx4"], *rest, *pairs)
    # a matrix's elements are off by 2^-4 of themselves at most in 8 bits, by a tenth on average in 4
    off8, off4 = (np.linalg.norm(v - dense) / np.linalg.norm(dense) for v in (eight, four))
    assert 0 < off8 < 3 * 2.0**-4 and off8 < off4 < 0.6
