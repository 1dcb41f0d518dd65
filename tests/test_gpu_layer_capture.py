# SPDX-License-Identifier: BSD-3-Clause
"""Captured and replayed: the expert layer with fp32 activations and 8-bit products with
either sums.  Every replay gives what eager calls give, with eager calls and other contents
of the operands between."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from expert_calls import Mem, ints
from fp8_cases import FP8, FP32
from test_gpu_expert_layer import inputs
from test_gpu_fp8_sums import random_rows
from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.buffer import ensure_device
from xtc_amd.utils.bf16 import f32_to_bf16_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


@pytest.mark.parametrize("weights", ["dense", "fp8", "mx4"])
def test_replays(weights):
    L = capi.lib()
    L.xtc_hip_expert_layer_workspace.restype = ctypes.c_uint64
    hip = ctypes.CDLL(next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln))
    stream = ctypes.c_void_p(L.xtc_hip_stream_create())

    def ok(code):
        assert code == 0, code

    T, E, K, H, M, N, nb = 40, 4, 256, 160, 500, 1100, 3
    x, router, (up, _), (down, _) = inputs(1, T, E, K, H, "bfloat16", weights, "swiglu", 2)
    mx, mr = Mem(x, "bfloat16"), Mem(router, "bfloat16")
    matrices = [Mem(up, "bfloat16"), None, Mem(down, "bfloat16"), None] if weights == "dense" else [Mem(m, "uint8") for m in (*up, *down)]
    el = capi.ExpertLayerDesc(dtype=1, weights=("dense", "fp8", "mx4").index(weights), activation=1, T=T, E=E, K=K, H=H, top_k=2,
                              normalize=1, hidden_f32=1, stream=stream)
    need = L.xtc_hip_expert_layer_workspace(ctypes.byref(el))
    ws, z = Mem(np.full(need, 0xFF), "uint8"), Mem(np.zeros((T, K)), "bfloat16")
    (ac, asc), (bc, bsc) = random_rows(1, M, nb), random_rows(2, N, nb, 128)
    operands = [Mem(v, "uint8") for v in (ac, asc, bc, bsc)]
    products = [(capi.Fp8MatmulDesc(out_dtype=1, M=M, N=N, blocks=nb, b_block_rows=128, sums=s, stream=stream), Mem(np.zeros((M, N)), "bfloat16"))
                for s in (FP32, FP8)]
    results = (z, *(c for _, c in products))

    def calls():
        capi.check(L.xtc_hip_expert_layer(ctypes.byref(el), mx.ptr, mr.ptr, *[m and m.ptr for m in matrices], ws.ptr, ctypes.c_uint64(need), z.ptr))
        for d, c in products:
            capi.check(L.xtc_hip_fp8_matmul(ctypes.byref(d), *[m.ptr for m in operands], c.ptr))

    calls()
    capi.check(L.xtc_hip_stream_synchronize(stream))
    graph, run = ctypes.c_void_p(), ctypes.c_void_p()
    ok(hip.hipStreamBeginCapture(stream, 1))
    calls()
    ok(hip.hipStreamEndCapture(stream, ctypes.byref(graph)))
    ok(hip.hipGraphInstantiate(ctypes.byref(run), graph, None, None, ctypes.c_size_t(0)))
    last = None
    for seed in (3, 4, 5, 6):
        for mem, raw in ((mx, f32_to_bf16_bits(ints(seed, (T, K), 3))), (operands[0], random_rows(seed, M, nb)[0])):
            mem.dev.memory_copy_to(mem.base + mem.at, raw.ctypes.data_as(ctypes.c_void_p), raw.nbytes)
        got = []
        for way in (lambda: ok(hip.hipGraphLaunch(run, stream)), calls):
            for mem in results:
                mem.dev.memory_fill_zero(mem.base + mem.at, mem.nbytes)
            capi.check(L.xtc_hip_synchronize())
            way()
            capi.check(L.xtc_hip_stream_synchronize(stream))
            got.append([m.numpy() for m in results])
        for a, b in zip(*got):
            np.testing.assert_array_equal(a, b)
            assert a.any()
        assert last is None or not any(np.array_equal(a, b) for a, b in zip(got[0], last))
        last = got[0]
    ok(hip.hipGraphExecDestroy(run))
    ok(hip.hipGraphDestroy(graph))
    capi.check(L.xtc_hip_stream_destroy(stream))
    for m in (*results, mx, mr, *matrices, ws, *operands):
        if m:
            m.free()
