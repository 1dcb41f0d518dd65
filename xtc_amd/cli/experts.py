# SPDX-License-Identifier: BSD-3-Clause
"""A layer of experts on the HIP backend: one training step of a projection in
bf16, and the whole layer served in 4 bits.

  python -m xtc_amd.cli.experts --tokens 512 --experts 8 --width 1024 --hidden 2048

Training: y = x w by expert, the gradients dx = dy w^T and dw = x^T dy, one graph
(the expert's matrices are passed twice, the second time as the transposed
operand that they are in memory).  Serving: the matrices are brought to 4 bits
once, by a graph of their own; then x -> 4 bits -> up -> relu -> 4 bits -> down.
Every graph is checked against its float64 form and timed.  (Extensions: the
reference's operators, src/xtc/graphs/xtc/operators.py:159-804, have neither
experts nor 4-bit types.)
"""

from __future__ import annotations

import argparse
from typing import Any

import numpy as np

from ..backends.hip import Backend
from ..graphs.xtc import op as O
from ..graphs.xtc.expert_operators import group_bounds
from ..utils.bf16 import round_to_bf16
from ..utils.mx4 import mx4_codes, mx4_scales, mx4_values

__all__ = ["main", "step_graph", "quantize_graph", "serve_graph"]


def step_graph(tokens: int, experts: int, width: int, hidden: int) -> Any:
    """(x, w, dy, w stored as in w, sizes) -> (y, dx, dw)."""
    x = O.tensor((tokens, width), "bfloat16", name="X")
    w = O.tensor((experts, width, hidden), "bfloat16", name="W")
    dy = O.tensor((tokens, hidden), "bfloat16", name="dY")
    wt = O.tensor((experts, hidden, width), "bfloat16", name="Wt", layout=[0, 2, 1])
    sizes = O.tensor((experts,), "int32", name="sizes")
    with O.graph(name="experts_step") as gb:
        y = O.grouped_matmul(x, w, sizes, name="Y")
        dx = O.grouped_matmul(dy, wt, sizes, name="dX")
        dw = O.grouped_matmul_grad_w(x, dy, sizes, out_dtype="float32", name="dW")
        O.outputs(y, dx, dw)
    return gb.graph


def quantize_graph(experts: int, rows: int, depth: int) -> Any:
    """(w [experts][rows][depth]) -> (codes, scales)."""
    w = O.tensor((experts, rows, depth), "bfloat16", name="W")
    with O.graph(name="experts_quantize") as gb:
        O.outputs(*O.mx4_quantize(w))
    return gb.graph


def serve_graph(tokens: int, experts: int, width: int, hidden: int) -> Any:
    """(x, codes and scales of up, of down, sizes) -> y."""
    def weights(rows: int, depth: int, name: str) -> tuple[Any, Any]:
        blocks = -(-depth // 32)
        return (O.tensor((experts, rows, 16 * blocks), "uint8", name=f"{name}_codes"),
                O.tensor((experts, rows, blocks), "uint8", name=f"{name}_scales"))

    x = O.tensor((tokens, width), "bfloat16", name="X")
    up, down = weights(hidden, width, "up"), weights(width, hidden, "down")
    sizes = O.tensor((experts,), "int32", name="sizes")
    with O.graph(name="experts_serve") as gb:
        h = O.relu(O.grouped_mx4_matmul(*O.mx4_quantize(x), *up, sizes, name="up"), name="act")
        O.grouped_mx4_matmul(*O.mx4_quantize(h), *down, sizes, name="down")
    return gb.graph


def _run(graph: Any, inputs: list[np.ndarray], outputs: list[np.ndarray]) -> float:
    """Fills `outputs`; microseconds a call."""
    backend = Backend(graph)
    module = backend.get_compiler(schedule_policy="strict").compile(backend.get_scheduler().schedule())
    evaluator = module.get_evaluator(parameters=(inputs, outputs), repeat=3, number=1, min_repeat_ms=20)
    times, code, message = evaluator.evaluate()
    if code:
        raise RuntimeError(f"{graph.name}: {message}")
    return 1e6 * min(times)


def _error(got: np.ndarray, want: np.ndarray) -> float:
    return float(np.linalg.norm(got.astype(np.float64) - want) / max(np.linalg.norm(want), 1e-300))


def _four_bits(a: np.ndarray) -> np.ndarray:
    scales = mx4_scales(a)
    return mx4_values(mx4_codes(a, scales), scales, a.shape[-1], np.float64)


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=512, help="rows, sorted by expert")
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args(argv)
    t, e, k, n = args.tokens, args.experts, args.width, args.hidden

    rng = np.random.default_rng(args.seed)

    def normal(scale: float, *shape: int) -> np.ndarray:
        return round_to_bf16(rng.normal(0, scale, shape).astype(np.float32))

    sizes = rng.multinomial(t, rng.dirichlet(np.full(e, 2.0))).astype(np.int32)
    x, dy, w = normal(1, t, k), normal(0.1, t, n), normal(k**-0.5, e, k, n)
    groups = group_bounds(sizes, t)
    print(f"{t} tokens at {e} experts of {k} x {n}: {sizes.tolist()}")

    y, dx, dw = np.empty((t, n), np.float32), np.empty((t, k), np.float32), np.empty((e, k, n), np.float32)
    us = _run(step_graph(t, e, k, n), [x, w, dy, w.swapaxes(1, 2), sizes], [y, dx, dw])
    x64, dy64, w64 = x.astype(np.float64), dy.astype(np.float64), w.astype(np.float64)
    want = (np.concatenate([x64[b:c] @ w64[i] for i, (b, c) in enumerate(groups)]),
            np.concatenate([dy64[b:c] @ w64[i].T for i, (b, c) in enumerate(groups)]),
            np.stack([x64[b:c].T @ dy64[b:c] for b, c in groups]))
    errors = [_error(got, ref) for got, ref in zip((y, dx, dw), want)]
    print(f"training step   {us:9.1f} us   relative errors y {errors[0]:.1e}, dx {errors[1]:.1e}, dw {errors[2]:.1e}")
    # bf16 results are rounded to 8 bits, fp32 sums of dw are not
    ok = max(errors[:2]) < 2.0**-8 and errors[2] < 1e-5

    up, down = normal(k**-0.5, e, n, k), normal(n**-0.5, e, k, n)
    packed: list[np.ndarray] = []
    for a in (up, down):
        codes = np.empty((*a.shape[:2], 16 * (-(-a.shape[2] // 32))), np.uint8)
        scales = np.empty((*a.shape[:2], codes.shape[2] // 16), np.uint8)
        us = _run(quantize_graph(*a.shape), [a], [codes, scales])
        same = np.array_equal(scales, mx4_scales(a)) and np.array_equal(codes, mx4_codes(a, scales))
        print(f"to 4 bits       {us:9.1f} us   {a.nbytes // 2 / 2**20:.0f} MiB to {(codes.nbytes + scales.nbytes) / 2**20:.0f}, "
              f"{'as defined' if same else 'WRONG'}")
        ok = ok and same
        packed += [codes, scales]
    z = np.empty((t, k), np.float32)
    us = _run(serve_graph(t, e, k, n), [x, *packed, sizes], [z])
    upv, downv = (mx4_values(packed[i], packed[i + 1], a.shape[2], np.float64) for i, a in ((0, up), (2, down)))
    x4 = _four_bits(x)
    h = np.concatenate([np.maximum(x4[b:c] @ upv[i].T, 0) for i, (b, c) in enumerate(groups)])
    h4 = _four_bits(h.astype(np.float32))
    error = _error(z, np.concatenate([h4[b:c] @ downv[i].T for i, (b, c) in enumerate(groups)]))
    print(f"served in 4 bits{us:9.1f} us   relative error {error:.1e}")
    # sums in another order: here and there a hidden value takes the neighbouring code
    ok = ok and error < 1e-2
    print("ok" if ok else "FAILED")
    return 0 if ok else 1


if __name__ == "__main__":
    raise SystemExit(main())
