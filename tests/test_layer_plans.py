# SPDX-License-Identifier: BSD-3-Clause
"""Plans of graphs that ask for the same 8-bit operands or gradients more than once: every
tensor is written by one launch, on the CPU."""

from __future__ import annotations

import itertools

import pytest

import xtc_amd.graphs.xtc.op as O
from test_expert_graphs import build
from test_layer_graphs import F, compiled
from xtc_amd.backends.hip import Backend


def written(ln):
    a = ln.attrs
    return [u for u in (ln.output, a.get("codes"), a.get("values"), *(a.get("other") or ()), *(a.get("results") or ())) if u]


def check(graph, most):
    """No tensor is written twice, and every scale, code and gradient is."""
    launches = Backend(graph).plan.launches
    outs = [u for ln in launches for u in dict.fromkeys(written(ln))]
    assert len(outs) == len(set(outs)), [(ln.kind, written(ln)) for ln in launches]
    assert {uid for uid, n in graph.nodes.items() if n.operation.name.startswith(("fp8_", "layer_norm"))} <= set(outs)
    assert len(launches) <= most, [ln.kind for ln in launches]
    compiled(graph)


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("order", sorted(set(itertools.permutations((False, False, True, True))) | {(False, True, True), (True, True, False)}))
def test_the_same_operand_quantised_again(order, rows):
    def fn(x):
        return O.outputs(*(t for turned in order for t in O.fp8_quantize(x, rows=rows, transpose=turned)))

    check(build(fn, ((200, 256), F)), len(order))


def test_values_and_both_layouts():
    def fn(x):
        a, b, c = O.fp8_quantize(x), O.fp8_quantize(x, transpose=True), O.fp8_quantize(x, transpose=True)
        return O.outputs(*a, O.fp8_dequantize(*a, size=256), *b, *c, O.fp8_codes(x, a[1]))

    check(build(fn, ((200, 256), F)), 4)


def test_gradients_asked_for_twice():
    def fn(x, w, dy):
        return O.outputs(*O.layer_norm_grad(x, w, dy), *O.layer_norm_grad(x, w, dy))

    check(build(fn, ((64, 256), F), ((256,), F), ((64, 256), F)), 2)
