# SPDX-License-Identifier: BSD-3-Clause
"""Layer norm and its gradients where the results are larger than what the caches keep, by
rows of each kind of registers, against float64 within layer_calls' bounds."""

from __future__ import annotations

import numpy as np
import pytest

from expert_calls import rounded
from layer_calls import check_close, layer_norm, layer_norm_grad, plain_norm, plain_norm_grad
from xtc_amd.runtimes.hip.buffer import ensure_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    ensure_device(0)
    yield


@pytest.mark.parametrize("dtype,rows,K", [("float32", 12000, 3001), ("float32", 4100, 8190), ("float32", 2500, 16001), ("bfloat16", 8300, 8190)])
def test_large_results(dtype, rows, K):
    rng = np.random.default_rng(K)
    x, dy = (rounded(rng.normal(size=(rows, K)).astype(np.float32), dtype) for _ in range(2))
    w, b = rng.normal(1, 0.2, K).astype(np.float32), rng.normal(size=K).astype(np.float32)
    print(f"[large norm] {rows} x {K} {dtype}", flush=True)
    check_close(layer_norm(x, w, b, dtype, "float32", pad=(1, 3)), *plain_norm(x, w, b, 1e-5), dtype)
    got = layer_norm_grad(x, w, dy, dtype, "float32", pad=(2, 1))
    want, off = plain_norm_grad(x, w, dy, 1e-5)
    for g, v, o, t in zip(got, want, off, (dtype, "float32", "float32")):
        check_close(g, v, o, t)
