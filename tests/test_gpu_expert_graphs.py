# SPDX-License-Identifier: BSD-3-Clause
"""The expert and 4-bit operators through graphs and payloads, the example that
runs them together, and their calls in a captured graph."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import xtc_amd.graphs.xtc.op as O
from expert_calls import Mem, ints, plain_grad_w, plain_grouped, rounded
from xtc_amd.backends.hip import Backend
from xtc_amd.cli import experts
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.bf16 import f32_to_bf16_bits
from xtc_amd.utils.mx4 import mx4_codes, mx4_scales, mx4_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def evaluate(graph, ins, outs):
    """The payload's outputs, which the evaluator has also compared with the
    graph's numpy semantics."""
    backend = Backend(graph)
    module = backend.get_compiler(schedule_policy="strict").compile(backend.get_scheduler().schedule())
    res, code, msg = module.get_evaluator(parameters=(ins, outs), validate=True, repeat=1, number=1, min_repeat_ms=0).evaluate()
    assert code == 0, msg
    return outs


@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")])
def test_training_graph(dtype, out):
    T, E, K, N = 90, 3, 64, 48
    x, w, dy = ints(1, (T, K)), ints(2, (E, K, N)), ints(3, (T, N))
    sizes = np.array([30, 0, 50], np.int32)
    tx, tw, tdy = O.tensor((T, K), dtype), O.tensor((E, K, N), dtype), O.tensor((T, N), dtype)
    twt, ts = O.tensor((E, N, K), dtype, layout=[0, 2, 1]), O.tensor((E,), "int32")
    with O.graph(name="step") as gb:
        O.outputs(O.grouped_matmul(tx, tw, ts, out_dtype=out), O.grouped_matmul(tdy, twt, ts, out_dtype=out),
                  O.grouped_matmul_grad_w(tx, tdy, ts, out_dtype=out))
    outs = [np.empty(s, np.float32) for s in ((T, N), (T, K), (E, K, N))]
    y, dx, dw = evaluate(gb.graph, [x, w, dy, w.swapaxes(1, 2), sizes], outs)
    np.testing.assert_array_equal(y, rounded(plain_grouped(x, w, sizes), out))
    np.testing.assert_array_equal(dx, rounded(plain_grouped(dy, w.swapaxes(1, 2), sizes), out))
    np.testing.assert_array_equal(dw, rounded(plain_grad_w(x, dy, sizes), out))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(5, 100), (2, 3, 64), (64, 256)])
def test_quantisation_graph(dtype, shape):
    x = rounded(np.random.default_rng(4).normal(size=shape), dtype)
    tx = O.tensor(shape, dtype)
    with O.graph(name="round_trip") as gb:
        codes, scales = O.mx4_quantize(tx)
        same = O.mx4_dequantize(codes, scales, size=shape[-1], out_dtype=dtype)
        other = O.mx4_dequantize(codes, scales, out_dtype="float32" if dtype == "bfloat16" else "bfloat16")
        O.outputs(codes, scales, same, other, O.mx4_codes(tx, scales))
    nb = -(-shape[-1] // 32)
    outs = [np.empty((*shape[:-1], 16 * nb), np.uint8), np.empty((*shape[:-1], nb), np.uint8), np.empty(shape, np.float32),
            np.empty((*shape[:-1], 32 * nb), np.float32), np.empty((*shape[:-1], 16 * nb), np.uint8)]
    c, s, v, o, again = evaluate(gb.graph, [x], outs)
    np.testing.assert_array_equal(s, mx4_scales(x))
    np.testing.assert_array_equal(c, mx4_codes(x, s))
    np.testing.assert_array_equal(again, c)
    np.testing.assert_array_equal(v, mx4_values(c, s, shape[-1]))
    np.testing.assert_array_equal(o, mx4_values(c, s))


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_serving_graph(out):
    """Quantised on the way in; whole numbers, so that every sum is exact."""
    M, E, N, K = 40, 2, 64, 160
    x, w = ints(5, (M, K), 4), ints(6, (E, N, K), 4)
    ws = mx4_scales(w)
    wc = mx4_codes(w, ws)
    sizes = np.array([25, 10], np.int32)
    tx, tc, tsc = O.tensor((M, K), "bfloat16"), O.tensor(wc.shape, "uint8"), O.tensor(ws.shape, "uint8")
    t0, t0s = O.tensor(wc.shape[1:], "uint8"), O.tensor(ws.shape[1:], "uint8")
    ts = O.tensor((E,), "int32")
    with O.graph(name="serve") as gb:
        q = O.mx4_quantize(tx)
        O.outputs(O.grouped_mx4_matmul(*q, tc, tsc, ts, out_dtype=out), O.mx4_matmul(*q, t0, t0s, out_dtype=out))
    grp, one = evaluate(gb.graph, [x, wc, ws, wc[1], ws[1], sizes], [np.empty((M, N), np.float32) for _ in range(2)])
    xv, wv = mx4_values(mx4_codes(x, mx4_scales(x)), mx4_scales(x)), mx4_values(wc, ws)
    np.testing.assert_array_equal(grp, rounded(plain_grouped(xv, wv.swapaxes(1, 2), sizes), out))
    np.testing.assert_array_equal(one, rounded(xv.astype(np.float64) @ wv[1].T, out))


def test_example(capsys):
    assert experts.main(["--tokens", "200", "--experts", "3", "--width", "256", "--hidden", "544"]) == 0
    assert "ok" in capsys.readouterr().out


def test_captured_calls_replay():
    """A graph of the expert calls (a gradient that eager calls sum in parts among
    them) gives the same results at every replay, with eager calls and other
    contents of the operands between."""
    L = capi.lib()
    hip = ctypes.CDLL(next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln))
    stream = ctypes.c_void_p(L.xtc_hip_stream_create())

    def ok(code):
        assert code == 0, code

    T, E, K, N = 3000, 2, 128, 64
    sizes = np.array([2000, 900], np.int32)
    w = ints(8, (E, K, N), 3)
    mx, mw, mdy, ms = (Mem(a, d) for a, d in ((ints(7, (T, K), 3), "bfloat16"), (w, "bfloat16"), (ints(9, (T, N), 3), "bfloat16"),
                                              (sizes, "int32")))
    y, dw = Mem(np.zeros((T, N)), "float32"), Mem(np.zeros((E, K, N), np.float32), "float32")
    nb = K // 32
    codes, scales = Mem(np.zeros((T, 16 * nb)), "uint8"), Mem(np.zeros((T, nb)), "uint8")
    c = Mem(np.zeros((T, T), np.float32), "float32")

    def calls():
        d = capi.GroupedMatmulDesc(dtype=1, out_dtype=0, E=E, T=T, N=N, K=K, stream=stream)
        capi.check(L.xtc_hip_grouped_matmul(ctypes.byref(d), mx.ptr, mw.ptr, ms.ptr, y.ptr))
        capi.check(L.xtc_hip_grouped_matmul_grad_w(ctypes.byref(d), mx.ptr, mdy.ptr, ms.ptr, dw.ptr))
        q = capi.Mx4Desc(dtype=1, rows=T, K=K, stream=stream)
        capi.check(L.xtc_hip_mx4_quantize(ctypes.byref(q), mx.ptr, codes.ptr, scales.ptr, None))
        m = capi.Mx4MatmulDesc(out_dtype=0, E=0, M=T, N=T, blocks=nb, stream=stream)
        capi.check(L.xtc_hip_mx4_matmul(ctypes.byref(m), codes.ptr, scales.ptr, codes.ptr, scales.ptr, None, c.ptr))

    calls()
    capi.check(L.xtc_hip_stream_synchronize(stream))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    ok(hip.hipStreamBeginCapture(stream, 1))
    calls()
    ok(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
    ok(hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)))
    dev = mx.dev
    for seed in (10, 11, 12, 13):
        x, dy = ints(seed, (T, K), 3), ints(seed + 20, (T, N), 3)
        for mem, a in ((mx, x), (mdy, dy)):
            bits = f32_to_bf16_bits(a)
            dev.memory_copy_to(mem.base + mem.at, bits.ctypes.data_as(ctypes.c_void_p), bits.nbytes)
        for mem in (y, dw, c):
            dev.memory_fill_zero(mem.base + mem.at, mem.nbytes)
        capi.check(L.xtc_hip_synchronize())
        ok(hip.hipGraphLaunch(run, stream))
        capi.check(L.xtc_hip_stream_synchronize(stream))
        np.testing.assert_array_equal(y.numpy(), plain_grouped(x, w, sizes))
        np.testing.assert_array_equal(dw.numpy(), plain_grad_w(x, dy, sizes))
        s = mx4_scales(x)
        v = mx4_values(mx4_codes(x, s), s)
        np.testing.assert_array_equal(c.numpy(), v @ v.T)
        calls()  # eager, between the replays
        capi.check(L.xtc_hip_stream_synchronize(stream))
        np.testing.assert_array_equal(dw.numpy(), plain_grad_w(x, dy, sizes))
    ok(hip.hipGraphExecDestroy(run))
    ok(hip.hipGraphDestroy(graph))
    capi.check(L.xtc_hip_stream_destroy(stream))
    for m in (mx, mw, mdy, ms, y, dw, codes, scales, c):
        m.free()
