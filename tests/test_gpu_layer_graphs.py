# SPDX-License-Identifier: BSD-3-Clause
"""Layer norm, 8-bit operands and the expert layer through graphs and payloads, one
after another as a model's layers use them, captured and replayed, and on two streams at
once."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import xtc_amd.graphs.xtc.op as O
from expert_calls import Mem, ints, rounded
from layer_calls import HALF, check_close, plain_layer, plain_norm, plain_norm_grad
from test_gpu_expert_graphs import evaluate
from test_gpu_expert_layer import inputs, pack
from xtc_amd.backends.hip import Backend
from xtc_amd.cli import experts
from xtc_amd.graphs.xtc.data import XTCTensor
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.bf16 import f32_to_bf16_bits
from xtc_amd.utils.fp8 import fp8_codes, fp8_scales, fp8_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


def payload(graph, ins, outs, scaled=None):
    """The payload's outputs; with `scaled` the evaluator has also compared them with the
    graph's numpy semantics, within that part of an output's largest element."""
    backend = Backend(graph)
    module = backend.get_compiler(schedule_policy="strict").compile(backend.get_scheduler().schedule())
    evaluator = module.get_evaluator(parameters=(ins, outs), validate=scaled is not None, scaled_tolerance=scaled, repeat=1, number=1,
                                     min_repeat_ms=0)
    _, code, msg = evaluator.evaluate()
    assert code == 0, msg
    return outs


@pytest.mark.parametrize("dtype,params", [("float32", "float32"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("shape", [(5, 96), (2, 3, 200), (64, 2500)])
def test_norm_graph(shape, dtype, params):
    rng = np.random.default_rng(shape[-1])
    K = shape[-1]
    x, dy = (rounded(rng.normal(size=shape), dtype) for _ in range(2))
    w, b = (rounded(rng.normal(size=K), params) for _ in range(2))
    tx, tw, tb, tdy = O.tensor(shape, dtype), O.tensor((K,), params), O.tensor((K,), params), O.tensor(shape, dtype)
    with O.graph(name="norm") as gb:
        O.outputs(O.layer_norm(tx, tw, tb, eps=1e-3), *O.layer_norm_grad(tx, tw, tdy, eps=1e-3))
    outs = [np.empty(s, np.float32) for s in (shape, shape, (K,), (K,))]
    # an element of a sum that cancels is off by its terms' roundings, not by its own: the
    # numpy form is met within half a step of the largest, and K or rows additions
    y, dx, dw, db = payload(gb.graph, [x, w, b, dy], outs, HALF[dtype] + (K + 64) * 2.0**-24)
    flat = x.reshape(-1, K)
    check_close(y.reshape(-1, K), *plain_norm(flat, w, b, 1e-3), dtype)
    want, off = plain_norm_grad(flat, w, dy.reshape(-1, K), 1e-3)
    check_close(dx.reshape(-1, K), want[0], off[0], dtype)
    check_close(dw, want[1], off[1], "float32")
    check_close(db, want[2], off[2], "float32")
    # sums that a graph without the rows' gradient asks for are the same bits
    with O.graph(name="sums") as gb:
        O.outputs(O.layer_norm_grad_weight(tx, tdy, eps=1e-3), O.layer_norm_grad_bias(tdy))
    dw2, db2 = payload(gb.graph, [x, dy], [np.empty(K, np.float32) for _ in range(2)])
    np.testing.assert_array_equal(dw2, dw)
    np.testing.assert_array_equal(db2, db)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", [(5, 100), (2, 130, 200)])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantisation_graph(rows, shape, dtype):
    x = rounded(np.random.default_rng(4).normal(size=shape), dtype)
    tx = O.tensor(shape, dtype)
    with O.graph(name="round_trip") as gb:
        q = O.fp8_quantize(tx, rows=rows)
        qt = O.fp8_quantize(tx, rows=rows, transpose=True)
        O.outputs(*q, O.fp8_dequantize(*q, size=shape[-1]), *qt, O.fp8_codes(tx, q[1], rows=rows))
    src = [x, np.ascontiguousarray(x.swapaxes(-1, -2))]
    s = [fp8_scales(a, rows) for a in src]
    c = [fp8_codes(a, b, rows) for a, b in zip(src, s)]
    want = [c[0], s[0], fp8_values(c[0], s[0], shape[-1]), c[1], s[1], c[0]]
    for got, w in zip(evaluate(gb.graph, [x], [np.empty_like(w) for w in want]), want):
        np.testing.assert_array_equal(got, w)


@pytest.mark.parametrize("T,K,N", [(40, 256, 130), (300, 512, 384)])
def test_training_step(T, K, N):
    """Norm, an 8-bit projection and its gradients, and the norm's: one graph, against its
    numpy form.  8-bit codes of the same tensors are the same; a normed element that rounds
    to the neighbouring bf16 number moves a code by a step at most, 2^-4 of it, among K."""
    rng = np.random.default_rng(T)
    x, w, dy = (rounded(rng.normal(size=s), "bfloat16") for s in ((T, K), (N, K), (T, N)))
    g, b = rounded(rng.normal(1, 0.1, K), "float32"), rounded(rng.normal(0, 0.1, K), "float32")
    tx, tg, tb, tw, tdy = (O.tensor(s, d) for s, d in (((T, K), "bfloat16"), ((K,), "float32"), ((K,), "float32"), ((N, K), "bfloat16"),
                                                      ((T, N), "bfloat16")))
    with O.graph(name="step") as gb:
        h = O.layer_norm(tx, tg, tb)
        y = O.fp8_matmul(*O.fp8_quantize(h), *O.fp8_quantize(tw, rows=128))
        dh = O.fp8_matmul(*O.fp8_quantize(tdy), *O.fp8_quantize(tw, rows=128, transpose=True), out_dtype="bfloat16")
        dw = O.fp8_matmul(*O.fp8_quantize(tdy, transpose=True), *O.fp8_quantize(h, transpose=True))
        O.outputs(y, dw, *O.layer_norm_grad(tx, tg, dh))
    ins = [x, g, b, w, dy]
    want = [o.numpy() for o in gb.graph.forward([XTCTensor(a, dtype=t.constant_dtype) for a, t in zip(ins, gb.graph.inputs_types)])]
    got = payload(gb.graph, ins, [np.empty_like(v) for v in want])
    for i, (a, v) in enumerate(zip(got, want)):
        off = np.linalg.norm(a.astype(np.float64) - v) / np.linalg.norm(v)
        # every code off by a step would be 2^-4; bf16 results are off by half a step
        assert off < 2.0**-8, (i, off)


@pytest.mark.parametrize("weights", ["dense", "fp8", "mx4"])
def test_served_layer(weights):
    """Norm and expert layer in one payload: what the layer alone gives for the norm's rows."""
    T, E, K, H = 6, 8, 256, 160
    x, router, (up, upv), (down, downv) = inputs(3, T, E, K, H, "bfloat16", weights, "swiglu", 2)
    matrices = [up, down] if weights == "dense" else [*up, *down]
    tx, tr = O.tensor((T, K), "bfloat16"), O.tensor((E, K), "bfloat16")
    one, zero = np.ones(K, np.float32), np.zeros(K, np.float32)
    t1, t0 = O.tensor((K,), "float32"), O.tensor((K,), "float32")
    tm = [O.tensor(m.shape, "bfloat16" if weights == "dense" else "uint8") for m in matrices]
    pair = tm if weights == "dense" else [tuple(tm[:2]), tuple(tm[2:])]
    with O.graph(name="served") as gb:
        h = O.layer_norm(tx, t1, t0)
        O.outputs(h, O.expert_layer(h, tr, *pair))
    got = payload(gb.graph, [x, router, one, zero, *matrices], [np.empty((T, K), np.float32) for _ in range(2)])
    check_close(got[0], *plain_norm(x, one, zero, 1e-5), "bfloat16")
    check_close(got[1], *plain_layer(got[0], router, upv, downv, 2, "swiglu", True, 2.0**-8), "bfloat16")


def test_example(capsys):
    assert experts.main(["--tokens", "70", "--experts", "5", "--width", "320", "--hidden", "192", "--few", "7"]) == 0
    out = capsys.readouterr().out
    assert out.count("tokens, ") == 3 and "step in 8 bits" in out


def test_captured_calls_replay():
    """One captured graph of all the calls gives the same as eager ones at every replay, with
    eager calls and other contents of the operands between."""
    L = capi.lib()
    L.xtc_hip_expert_layer_workspace.restype = ctypes.c_uint64
    hip = ctypes.CDLL(next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln))
    stream = ctypes.c_void_p(L.xtc_hip_stream_create())

    def ok(code):
        assert code == 0, code

    T, K, N, E, H = 60, 256, 640, 8, 128
    w, router = ints(8, (N, K), 3), rounded(np.random.default_rng(1).normal(size=(E, K)), "bfloat16")
    up, down = (rounded(np.random.default_rng(i).normal(0, 0.1, s), "bfloat16") for i, s in ((2, (E, 2 * H, K)), (3, (E, K, H))))
    (uc, us), _ = pack(up, "fp8")
    (dc, ds), _ = pack(down, "fp8")
    mx, mdy, mw, mr = (Mem(a, "bfloat16") for a in (ints(7, (T, K), 3), ints(9, (T, K), 3), w, router))
    mg, muc, mus, mdc, mds = Mem(np.ones(K), "float32"), Mem(uc, "uint8"), Mem(us, "uint8"), Mem(dc, "uint8"), Mem(ds, "uint8")
    ln = capi.LayerNormDesc(dtype=1, param_dtype=0, rows=T, K=K, eps=1e-5, stream=stream)
    qd = capi.Fp8Desc(dtype=1, matrices=1, rows=T, K=K, block_rows=1, stream=stream)
    qw = capi.Fp8Desc(dtype=1, matrices=1, rows=N, K=K, block_rows=128, stream=stream)
    pd = capi.Fp8MatmulDesc(out_dtype=0, M=T, N=N, blocks=K // 128, b_block_rows=128, stream=stream)
    el = capi.ExpertLayerDesc(dtype=1, weights=1, activation=1, T=T, E=E, K=K, H=H, top_k=2, normalize=1, stream=stream)
    need = L.xtc_hip_expert_layer_workspace(ctypes.byref(el))
    zeros = lambda shape, dtype: Mem(np.zeros(shape), dtype)  # noqa: E731
    h, dx, y, z = zeros((T, K), "bfloat16"), zeros((T, K), "bfloat16"), zeros((T, N), "float32"), zeros((T, K), "bfloat16")
    dg, db, sums, ws = zeros(K, "float32"), zeros(K, "float32"), zeros(2 * T * K + 2 * T, "float32"), zeros(need, "uint8")
    hc, hs, hct, hst = (zeros(s, "uint8") for s in ((T, K), (T, K // 128), (K, 128), (K, 1)))
    wc, wsc = zeros((N, K), "uint8"), zeros((N // 128, K // 128), "uint8")
    results = (h, dx, dg, db, hct, hst, y, z)

    def calls():
        capi.check(L.xtc_hip_layer_norm(ctypes.byref(ln), mx.ptr, mg.ptr, None, h.ptr))
        capi.check(L.xtc_hip_layer_norm_grad(ctypes.byref(ln), mx.ptr, mg.ptr, mdy.ptr, dx.ptr, dg.ptr, db.ptr, sums.ptr))
        capi.check(L.xtc_hip_fp8_quantize_both(ctypes.byref(qd), h.ptr, hc.ptr, hs.ptr, hct.ptr, hst.ptr))
        capi.check(L.xtc_hip_fp8_quantize(ctypes.byref(qw), mw.ptr, wc.ptr, wsc.ptr, None))
        capi.check(L.xtc_hip_fp8_matmul(ctypes.byref(pd), hc.ptr, hs.ptr, wc.ptr, wsc.ptr, y.ptr))
        capi.check(L.xtc_hip_expert_layer(ctypes.byref(el), h.ptr, mr.ptr, muc.ptr, mus.ptr, mdc.ptr, mds.ptr, ws.ptr, ctypes.c_uint64(need), z.ptr))

    calls()
    capi.check(L.xtc_hip_stream_synchronize(stream))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    ok(hip.hipStreamBeginCapture(stream, 1))
    calls()
    ok(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
    ok(hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)))
    dev = mx.dev
    for seed in (10, 11, 12, 13):
        for mem, a in ((mx, ints(seed, (T, K), 3)), (mdy, ints(seed + 20, (T, K), 3))):
            bits = f32_to_bf16_bits(a)
            dev.memory_copy_to(mem.base + mem.at, bits.ctypes.data_as(ctypes.c_void_p), bits.nbytes)
        got = []
        for way in (lambda: ok(hip.hipGraphLaunch(run, stream)), calls):
            for mem in results:
                dev.memory_fill_zero(mem.base + mem.at, mem.nbytes)
            capi.check(L.xtc_hip_synchronize())
            way()
            capi.check(L.xtc_hip_stream_synchronize(stream))
            got.append([m.numpy() for m in results])
        for a, b in zip(*got):
            np.testing.assert_array_equal(a, b)
        assert got[0][0].any() and got[0][6].any() and got[0][7].any()
    ok(hip.hipGraphExecDestroy(run))
    ok(hip.hipGraphDestroy(graph))
    capi.check(L.xtc_hip_stream_destroy(stream))
    for m in (*results, mx, mdy, mw, mr, mg, muc, mus, mdc, mds, sums, ws, hc, hs, wc, wsc):
        m.free()


def test_two_layers_at_once():
    """Two streams, a workspace each, calls of one beside those of the other: the results of
    calls alone."""
    L = capi.lib()
    L.xtc_hip_expert_layer_workspace.restype = ctypes.c_uint64
    T, E, K, H = 48, 8, 512, 256
    streams = [ctypes.c_void_p(L.xtc_hip_stream_create()) for _ in range(2)]
    sides = []
    for i, stream in enumerate(streams):
        x, router, (up, _), (down, _) = inputs(i, T, E, K, H, "bfloat16", "dense", "swiglu", 2)
        d = capi.ExpertLayerDesc(dtype=1, weights=0, activation=1, T=T, E=E, K=K, H=H, top_k=2, normalize=1, stream=stream)
        need = L.xtc_hip_expert_layer_workspace(ctypes.byref(d))
        mems = [Mem(a, "bfloat16") for a in (x, router, up, down)]
        sides.append((d, need, mems, Mem(np.full(need, 0xFF), "uint8"), [Mem(np.zeros((T, K)), "bfloat16") for _ in range(9)]))

    def go(side, out):
        d, need, (x, r, u, w), ws, _ = side
        capi.check(L.xtc_hip_expert_layer(ctypes.byref(d), x.ptr, r.ptr, u.ptr, None, w.ptr, None, ws.ptr, ctypes.c_uint64(need), out.ptr))

    alone = []
    for side in sides:
        go(side, side[4][0])
        capi.check(L.xtc_hip_stream_synchronize(side[0].stream))
        alone.append(side[4][0].numpy())
    for i in range(1, 9):
        for side in sides:
            go(side, side[4][i])
    for stream in streams:
        capi.check(L.xtc_hip_stream_synchronize(stream))
    for side, want in zip(sides, alone):
        for out in side[4][1:]:
            np.testing.assert_array_equal(out.numpy(), want)
        for m in (*side[2], side[3], *side[4]):
            m.free()
    for stream in streams:
        capi.check(L.xtc_hip_stream_destroy(stream))
