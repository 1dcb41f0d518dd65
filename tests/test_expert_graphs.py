# SPDX-License-Identifier: BSD-3-Clause
"""Graphs with the expert and 4-bit operators, on the CPU: types, refusals, the
numpy semantics against brute force, and what the HIP backend makes of them."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest

import xtc_amd.graphs.xtc.op as O
from xtc_amd.backends.hip import Backend
from xtc_amd.backends.hip.lowering import UnsupportedGraph
from xtc_amd.backends.hip.scheduler import ScheduleError
from xtc_amd.graphs.xtc.data import XTCTensor
from xtc_amd.utils.mx4 import mx4_codes, mx4_scales, mx4_values

VALUES = [Fraction(0), Fraction(1, 2), Fraction(1), Fraction(3, 2), Fraction(2), Fraction(3), Fraction(4), Fraction(6)]


def build(fn, *types, name="graph"):
    ins = [O.tensor(shape, dtype, **more) for shape, dtype, *rest in types for more in [rest[0] if rest else {}]]
    with O.graph(name=name) as gb:
        fn(*ins)
    return gb.graph


def forward(graph, *arrays):
    outs = graph.forward([XTCTensor(a, dtype=t.constant_dtype) for a, t in zip(arrays, graph.inputs_types)])
    return [o.numpy() for o in outs]


def brute_block(block):
    """(scale byte, codes) of 32 numbers in exact arithmetic."""
    if not np.isfinite(block).all():
        return 255, [0] * 32
    top = max(abs(Fraction(float(v))) for v in block)
    s = 0
    while s < 254 and Fraction(2) ** (s + 1 - 125) <= top:  # floor(log2 top) - 2 + 127
        s += 1
    if top < Fraction(2) ** (1 - 125):
        s = 0
    codes = []
    for v in block:
        y = abs(Fraction(float(v))) / Fraction(2) ** (s - 127)
        best = min(range(8), key=lambda i: (abs(VALUES[i] - y), i % 2))
        codes.append(best | (8 if np.signbit(v) else 0))
    return s, codes


def test_mx4_against_exact_arithmetic():
    rng = np.random.default_rng(0)
    x = (rng.normal(size=(40, 64)) * np.exp2(rng.integers(-8, 8, (40, 64)))).astype(np.float32)
    x[0] = 0
    x[1, :32] = np.ldexp(np.float32(1), -140)
    x[2, :32] = np.ldexp(np.float32(3), -126)
    x[3, 0], x[4, 40], x[5, 1] = np.inf, np.nan, 3e38
    x[6, :32] = np.repeat([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7], 4)
    x[7, :32] = -x[6, :32]
    scales = mx4_scales(x)
    codes = mx4_codes(x, scales)
    for r in range(40):
        for b in range(2):
            s, want = brute_block(x[r, 32 * b : 32 * b + 32])
            assert scales[r, b] == s, (r, b)
            got = codes[r, 16 * b : 16 * b + 16]
            assert np.stack((got & 15, got >> 4), -1).reshape(-1).tolist() == want, (r, b)
    values = mx4_values(codes, scales)
    assert values[5, 1] == np.ldexp(6.0, 125) and np.isnan(values[3, :32]).all() and not values[0].any()
    again = mx4_scales(values[6:])  # what is on the grid stays
    np.testing.assert_array_equal(mx4_values(mx4_codes(values[6:], again), again), values[6:])


def test_mx4_graph_is_one_launch():
    x = O.tensor((6, 100), "float32")
    with O.graph(name="round_trip") as gb:
        codes, scales = O.mx4_quantize(x)
        y = O.mx4_dequantize(codes, scales, size=100)
        O.outputs(codes, scales, y)
    a = np.random.default_rng(1).normal(size=(6, 100)).astype(np.float32)
    c, s, v = forward(gb.graph, a)
    np.testing.assert_array_equal(s, mx4_scales(a))
    np.testing.assert_array_equal(v, mx4_values(c, s, 100))
    assert (c[:, -14:] == 0).all()  # 4 elements of the last block exist
    launches = Backend(gb.graph).plan.launches
    assert [ln.kind for ln in launches] == ["mx4_quantize"] and len(launches[0].absorbed) == 2


@pytest.mark.parametrize("kinds,fn", [
    (["mx4_quantize"], lambda x: O.mx4_scales(x)),
    # codes for the scales of another tensor, and the values of another type
    (["mx4_quantize", "mx4_encode"], lambda x: O.mx4_codes(O.relu(x), O.mx4_scales(x))),
    (["mx4_quantize", "mx4_dequantize"], lambda x: O.mx4_dequantize(*O.mx4_quantize(x), out_dtype="bfloat16")),
    (["mx4_quantize", "mx4_quantize_matmul"], lambda x: O.mx4_matmul(*O.mx4_quantize(x), *O.mx4_quantize(x))),
    (["mx4_quantize", "mx4_matmul"], lambda x: (lambda q: O.mx4_matmul(*q, *q))(O.mx4_quantize(x))),
    (["mx4_quantize", "mx4_matmul"], lambda x: (lambda q, w: O.outputs(*q, O.mx4_matmul(*q, *w)))(
        O.mx4_quantize(x), O.mx4_quantize(x))),
    (["mx4_quantize", "mx4_matmul"], lambda x: (lambda q, w: O.outputs(O.mx4_matmul(*q, *w), O.mx4_dequantize(*q, size=64)))(
        O.mx4_quantize(x), O.mx4_quantize(x))),
])
def test_mx4_plans(kinds, fn):
    graph = build(fn, ((64, 64), "float32"))
    got = [ln.kind for ln in Backend(graph).plan.launches if ln.kind != "relu"]
    assert [k for i, k in enumerate(got) if k not in got[:i]] == kinds


def test_expert_layer():
    """Two products by group with a relu between, and their gradients."""
    T, E, K, H = 20, 3, 8, 12
    types = [((T, K), "float32"), ((E, K, H), "float32"), ((E, H, K), "float32"), ((E,), "int32")]

    def layer(x, up, down, sizes):
        O.grouped_matmul(O.relu(O.grouped_matmul(x, up, sizes)), down, sizes)

    rng = np.random.default_rng(2)
    x, up, down = (rng.integers(-3, 4, t[0]).astype(np.float32) for t in types[:3])
    sizes = np.array([7, 0, 9], np.int32)
    graph = build(layer, *types)
    (y,) = forward(graph, x, up, down, sizes)
    expert = [0] * 7 + [2] * 9
    want = np.zeros((T, K), np.float32)
    for r, e in enumerate(expert):
        want[r] = np.maximum(x[r] @ up[e], 0) @ down[e]
    np.testing.assert_array_equal(y, want)
    assert [ln.kind for ln in Backend(graph).plan.launches] == ["grouped_matmul", "relu", "grouped_matmul"]

    graph = build(O.grouped_matmul_grad_w, ((T, K), "float32"), ((T, H), "float32"), ((E,), "int32"))
    dy = rng.integers(-3, 4, (T, H)).astype(np.float32)
    (dw,) = forward(graph, x, dy, sizes)
    want = np.zeros((E, K, H), np.float32)
    for r, e in enumerate(expert):
        want[e] += np.outer(x[r], dy[r])
    np.testing.assert_array_equal(dw, want)


def test_sizes_are_clipped():
    graph = build(O.grouped_matmul, ((5, 2), "float32"), ((3, 2, 2), "float32"), ((3,), "int32"))
    x, w = np.ones((5, 2), np.float32), np.arange(1, 4, dtype=np.float32)[:, None, None] * np.ones((3, 2, 2), np.float32)
    for sizes, rows in (([2**31 - 1, 2, 2], [2] * 5), ([-1, 2, 9], [4, 4, 6, 6, 6]), ([0, 0, 1], [6, 0, 0, 0, 0])):
        (y,) = forward(graph, x, w, np.array(sizes, np.int32))
        np.testing.assert_array_equal(y[:, 0], rows)


def test_grouped_mx4():
    nb, T, E, N = 2, 9, 2, 4
    types = [((T, 16 * nb), "uint8"), ((T, nb), "uint8"), ((E, N, 16 * nb), "uint8"), ((E, N, nb), "uint8"), ((E,), "int32")]
    rng = np.random.default_rng(3)
    a, b = rng.integers(0, 256, (T, 16 * nb)), rng.integers(0, 256, (E, N, 16 * nb))
    sa, sb = rng.integers(120, 130, (T, nb)), rng.integers(120, 130, (E, N, nb))
    (y,) = forward(build(O.grouped_mx4_matmul, *types), *(v.astype(np.uint8) for v in (a, sa, b, sb)), np.array([4, 3], np.int32))
    av, bv = mx4_values(a.astype(np.uint8), sa), mx4_values(b.astype(np.uint8), sb)
    np.testing.assert_allclose(y[:4], av[:4] @ bv[0].T, rtol=1e-5, atol=1e-6)
    np.testing.assert_allclose(y[4:7], av[4:7] @ bv[1].T, rtol=1e-5, atol=1e-6)
    assert not y[7:].any()
    (c,) = forward(build(O.mx4_matmul, *types[:2], ((N, 16 * nb), "uint8"), ((N, nb), "uint8")),
                   *(v.astype(np.uint8) for v in (a, sa, b[1], sb[1])))
    np.testing.assert_allclose(c, av @ bv[1].T, rtol=1e-5, atol=1e-6)


F, B, U, I = "float32", "bfloat16", "uint8", "int32"


@pytest.mark.parametrize("fn,types", [
    (O.grouped_matmul, [((4, 8), F), ((2, 8, 4), B), ((2,), I)]),
    (O.grouped_matmul, [((4, 8), "float64"), ((2, 8, 4), "float64"), ((2,), I)]),
    (O.grouped_matmul, [((4, 8), F), ((2, 9, 4), F), ((2,), I)]),
    (O.grouped_matmul, [((4, 8), F), ((8, 4), F), ((2,), I)]),
    (O.grouped_matmul, [((4, 8), F), ((2, 8, 4), F), ((3,), I)]),
    (O.grouped_matmul, [((4, 8), F), ((2, 8, 4), F), ((2,), "int64")]),
    (lambda *a: O.grouped_matmul(*a, out_dtype=B), [((4, 8), F), ((2, 8, 4), F), ((2,), I)]),
    (O.grouped_matmul_grad_w, [((4, 8), F), ((5, 8), F), ((2,), I)]),
    (O.grouped_matmul_grad_w, [((4, 8), F), ((4, 8), F), ((2, 1), I)]),
    (O.mx4_scales, [((64,), F)]),
    (O.mx4_scales, [((4, 64), U)]),
    (O.mx4_codes, [((4, 64), F), ((4, 3), U)]),
    (O.mx4_dequantize, [((4, 32), U), ((4, 3), U)]),
    (lambda *a: O.mx4_dequantize(*a, size=65), [((4, 32), U), ((4, 2), U)]),
    (lambda *a: O.mx4_dequantize(*a, out_dtype="float64"), [((4, 32), U), ((4, 2), U)]),
    (O.mx4_matmul, [((4, 32), U), ((4, 2), U), ((4, 48), U), ((4, 3), U)]),
    (O.mx4_matmul, [((4, 32), F), ((4, 2), U), ((4, 32), U), ((4, 2), U)]),
    (O.grouped_mx4_matmul, [((4, 32), U), ((4, 2), U), ((4, 32), U), ((4, 2), U), ((4,), I)]),
    (O.grouped_mx4_matmul, [((4, 32), U), ((4, 2), U), ((2, 4, 32), U), ((2, 4, 2), U), ((3,), I)]),
])
def test_types_that_do_not_fit(fn, types):
    with pytest.raises(ValueError):
        build(fn, *types)


def test_layouts():
    w = ((2, 8, 4), F, {"layout": [0, 2, 1]})
    graph = build(O.grouped_matmul, ((4, 8), F), w, ((2,), I))
    assert Backend(graph).plan.launches[0].attrs["trans_w"] is True
    for bad in ([1, 0, 2], [2, 1, 0]):
        with pytest.raises(UnsupportedGraph):
            Backend(build(O.grouped_matmul, ((4, 8), F), ((2, 8, 4), F, {"layout": bad}), ((2,), I)))
    with pytest.raises(UnsupportedGraph):
        Backend(build(O.grouped_matmul_grad_w, ((4, 8), F, {"layout": [1, 0]}), ((4, 8), F), ((2,), I)))


def test_schedules_are_refused():
    graph = build(lambda x, w, s: O.grouped_matmul(x, w, s, name="Y"), ((64, 32), F), ((2, 32, 64), F), ((2,), I))
    backend = Backend(graph)
    compiler = backend.get_compiler(schedule_policy="strict")
    assert compiler.kernel_configs(backend.get_scheduler().schedule()) == {}
    sch = backend.get_scheduler()
    sch.tile("i", {"i1": 16})
    with pytest.raises(ScheduleError, match="choose"):
        compiler.compile(sch.schedule())


def test_graph_file_round_trip(tmp_path):
    x = O.tensor((4, 64), "float32")
    with O.graph(name="quantized") as gb:
        O.mx4_dequantize(*O.mx4_quantize(x), name="Y")
    gb.graph.dump(tmp_path / "g.yaml")
    with O.graph() as again:
        O.graph.load(tmp_path / "g.yaml")
    a = np.random.default_rng(4).normal(size=(4, 64)).astype(np.float32)
    np.testing.assert_array_equal(forward(again.graph, a)[0], forward(gb.graph, a)[0])


def test_equal_graphs_make_equal_payloads():
    """Unnamed nodes do not tell two builds of one graph apart."""
    def source():
        backend = Backend(build(lambda x: O.mx4_matmul(*O.mx4_quantize(x), *O.mx4_quantize(x)), ((4, 64), F)))
        return backend.get_compiler().compile(backend.get_scheduler().schedule()).source

    assert source() == source()


def test_example_graphs_lower():
    """The graphs of the example: their launches, and their numpy semantics chained."""
    from xtc_amd.cli import experts

    T, E, K, N = 20, 3, 64, 96
    rng = np.random.default_rng(5)
    kinds = {}
    for graph in (experts.step_graph(T, E, K, N), experts.quantize_graph(E, N, K), experts.serve_graph(T, E, K, N)):
        backend = Backend(graph)
        backend.get_compiler(schedule_policy="strict").compile(backend.get_scheduler().schedule())
        kinds[graph.name] = [launch.kind for launch in backend.plan.launches]
    assert kinds == {"experts_step": ["grouped_matmul"] * 2 + ["grouped_matmul_grad_w"], "experts_quantize": ["mx4_quantize"],
                     "experts_serve": ["mx4_quantize_matmul", "relu", "mx4_quantize_matmul"]}
    up, down = (rng.normal(size=s).astype(np.float32) for s in ((E, N, K), (E, K, N)))
    x, sizes = rng.normal(size=(T, K)).astype(np.float32), np.array([7, 0, 9], np.int32)
    packed = [a for w in (up, down) for a in forward(experts.quantize_graph(*w.shape), w)]
    y, = forward(experts.serve_graph(T, E, K, N), x, *packed, sizes)
    full = np.concatenate([np.maximum(x[b:e] @ up[i].T, 0) @ down[i].T for i, (b, e) in enumerate(((0, 7), (7, 7), (7, 16)))])
    assert y.shape == (T, K) and not y[16:].any()
    # each of the four 4-bit operands is off by about a tenth of its norm
    assert np.linalg.norm(y[:16] - full) < 0.5 * np.linalg.norm(full)
