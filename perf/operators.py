# SPDX-License-Identifier: BSD-3-Clause
"""The expert and 4-bit operators: calls of every kind that a model's layers
make, with inputs, required work, a plain form and float64 results.

Kinds of case:
  grouped   y[r] = x[r] @ w[e], e the expert whose group row r is in: rows come
            sorted by expert, `sizes` (int32, in HBM) says how many each has,
            rows past their sum belong to nobody and give zeros.  With trans_w
            an expert's matrix is stored transposed: a checkpoint's [out][in],
            or the gradient of x, dy @ w^T
  grad_w    the gradient of w: dw[e] = x_e^T @ dy_e over the rows of expert e
  mx4       x to microscaled 4-bit floats (blocks of 32, a power-of-two scale
            each) and back to values
  mx4_mm    bf16 activations quantised, times 4-bit weights [n][k]
  mx4_grp   the same, rows grouped by expert

Where `own` is true a case is a graph built with the operator DSL, compiled by
the HIP backend under its default schedule into a payload that queues its
kernels and returns.  Operands live in HBM.
"""

from __future__ import annotations

import ctypes
from typing import Any

import numpy as np
import torch

own = False

_TORCH = {"float32": torch.float32, "bfloat16": torch.bfloat16}
_BYTES = {"float32": 4, "bfloat16": 2}


def _grouped(name: str, dtype: str, out: str, t: int, e: int, k: int, n: int, trans_w: bool, spare: int = 0) -> dict[str, Any]:
    return {"name": name, "kind": "grouped", "dtype": dtype, "out": out, "t": t, "e": e, "k": k, "n": n,
            "trans_w": trans_w, "spare": spare}


def _grad_w(name: str, dtype: str, out: str, t: int, e: int, k: int, n: int, spare: int = 0) -> dict[str, Any]:
    return {"name": name, "kind": "grad_w", "dtype": dtype, "out": out, "t": t, "e": e, "k": k, "n": n, "spare": spare}


def _mx4(name: str, dtype: str, rows: int, k: int) -> dict[str, Any]:
    return {"name": name, "kind": "mx4", "dtype": dtype, "rows": rows, "k": k}


def _mx4_mm(name: str, out: str, m: int, n: int, k: int) -> dict[str, Any]:
    return {"name": name, "kind": "mx4_mm", "out": out, "m": m, "n": n, "k": k}


def _mx4_grp(name: str, out: str, t: int, e: int, k: int, n: int, spare: int = 0) -> dict[str, Any]:
    return {"name": name, "kind": "mx4_grp", "out": out, "t": t, "e": e, "k": k, "n": n, "spare": spare}


def listed() -> list[dict[str, Any]]:
    return [
        # one token at two of eight experts while decoding: latency and two weight matrices
        _grouped("experts_token", "bfloat16", "bfloat16", 2, 8, 1024, 1024, True),
        # a long prefill: the largest product by expert
        _grouped("experts_prefill", "bfloat16", "bfloat16", 32768, 16, 4096, 4096, False),
        # training: the gradient of the activations, weights read transposed
        _grouped("experts_grad_x", "bfloat16", "bfloat16", 8192, 8, 2048, 4096, True, 100),
        # fp32 at a user's own sizes: no row is 16-byte aligned
        _grouped("experts_f32_odd", "float32", "float32", 777, 5, 509, 301, False, 7),
        # training: the gradient of the weights, sums over ragged runs of rows, kept in fp32
        _grad_w("experts_grad_w", "bfloat16", "float32", 16384, 16, 2048, 2048),
        # the same in fp32 at odd sizes
        _grad_w("experts_grad_w_odd", "float32", "float32", 1001, 7, 333, 250, 9),
        # a large weight matrix brought to 4 bits, with the values that it then stands for
        _mx4("mx4_weights", "bfloat16", 8192, 8192),
        # a few fp32 rows whose last block is partial: latency
        _mx4("mx4_rows_odd", "float32", 5, 1000),
        # one decode step of 16 sequences through a square projection: streams the 4-bit weights
        _mx4_mm("mx4_decode", "bfloat16", 16, 8192, 8192),
        # the headline matmul size on 4-bit operands
        _mx4_mm("mx4_8192", "float32", 8192, 8192, 8192),
        # a decode batch over experts in 4 bits: each weight matrix serves a row or two
        _mx4_grp("mx4_experts_decode", "bfloat16", 32, 16, 4096, 2048),
        # a prefill over experts in 4 bits
        _mx4_grp("mx4_experts_prefill", "bfloat16", 8192, 16, 4096, 2048),
    ]


def _log(rng: Any, lo: int, hi: int) -> int:
    return int(round(lo * (hi / lo) ** rng.random()))


def _rows(rng: Any, hi: int) -> int:
    """1 to hi rows: odd counts mostly, powers of two otherwise."""
    n = _log(rng, 1, hi)
    return n | 1 if rng.random() < 0.7 else 1 << (n.bit_length() - 1)


def _wide(rng: Any, lo: int, hi: int) -> int:
    """A model's width: a power of two, or 5 or 7 quarters of one."""
    while True:
        v = (1 << rng.randint(lo.bit_length() - 1, hi.bit_length() - 1)) * rng.choice((4, 4, 5, 7)) // 4
        if lo <= v <= hi:
            return v


def draw(rng: Any) -> dict[str, Any]:
    # most operations of a listed case of the kind, and most bytes of any
    most = {"grouped": 1.1e12, "grad_w": 1.4e11, "mx4": 0.0, "mx4_mm": 1.1e12, "mx4_grp": 1.4e11}
    while True:
        case = _draw(rng)
        w = work(case)
        top = 3e9 if case.get("dtype") == "float32" and case["kind"] != "mx4" else most[case["kind"]]
        if w["flops"] <= top and w["bytes"] <= 1.07e9:
            del case["name"]
            return case


def _draw(rng: Any) -> dict[str, Any]:
    kind = rng.choice(("grouped", "grouped", "grouped", "grouped_f32", "grad_w", "grad_w", "grad_w_f32", "mx4", "mx4_mm",
                       "mx4_mm", "mx4_grp", "mx4_grp"))
    out = rng.choice(("float32", "bfloat16"))
    e = rng.choice((1, 2, 3, 5, 8, 12, 16, 24, 32, 64))
    spare = rng.choice((0, 0, 1, 17))
    if kind in ("grouped", "grad_w"):
        t, k, n = _rows(rng, 32768), _wide(rng, 64, 4096), _wide(rng, 64, 4096)
        if rng.random() < 0.25:  # sizes of no whole vectors
            k, n = _log(rng, 33, 2000) | 1, _log(rng, 33, 2000) | 1
        spare = min(spare, t - 1)
        if kind == "grad_w":
            return _grad_w("", "bfloat16", out, t, e, k, n, spare)
        return _grouped("", "bfloat16", out, t, e, k, n, rng.random() < 0.5, spare)
    if kind in ("grouped_f32", "grad_w_f32"):
        t, k, n = _log(rng, 1, 2000) | 1, _log(rng, 17, 1200), _log(rng, 17, 1200)
        spare = min(spare, t - 1)
        if kind == "grad_w_f32":
            return _grad_w("", "float32", "float32", t, min(e, 16), k, n, spare)
        return _grouped("", "float32", "float32", t, min(e, 16), k, n, rng.random() < 0.5, spare)
    if kind == "mx4":
        k = _wide(rng, 32, 8192) if rng.random() < 0.7 else _log(rng, 1, 3000) | 1
        return _mx4("", rng.choice(("float32", "bfloat16", "bfloat16")), _rows(rng, 8192), k)
    k = _wide(rng, 128, 8192) if rng.random() < 0.7 else 32 * (_log(rng, 1, 150) | 1)
    if kind == "mx4_mm":
        return _mx4_mm("", out, _rows(rng, 8192), _wide(rng, 64, 8192) if rng.random() < 0.7 else _log(rng, 17, 4000) | 1, k)
    t = _rows(rng, 8192)
    return _mx4_grp("", out, t, e, min(k, 4096), _wide(rng, 64, 4096), min(spare, t - 1))


# ------------------------------------------------------------------- inputs


def _sizes(case: dict[str, Any], seed: int) -> list[int]:
    """Rows of each expert: a router's skewed choice, some experts left out."""
    rng = np.random.default_rng([seed, 77])
    p = rng.dirichlet(np.full(case["e"], 2.0))
    if case["e"] >= 4:
        p[rng.random(case["e"]) < 0.12] = 0.0
    p = p / p.sum() if p.sum() > 0 else np.full(case["e"], 1.0 / case["e"])
    return [int(c) for c in rng.multinomial(case["t"] - case["spare"], p)]


def _normal(gen: torch.Generator, dtype: str, std: float, *shape: int) -> torch.Tensor:
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=gen).to(_TORCH[dtype])


def _activations(gen: torch.Generator, dtype: str, rows: int, k: int) -> torch.Tensor:
    """Normal with a few channels sixteen times as large, as hidden states are."""
    x = torch.empty((rows, k), device="cuda", dtype=torch.float32).normal_(0.0, 1.0, generator=gen)
    x[:, :: max(1, k // 5)] *= 16.0
    return x.to(_TORCH[dtype])


def _inputs(case: dict[str, Any], seed: int) -> dict[str, torch.Tensor]:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, k = case["kind"], case["k"]
    if kind == "mx4":
        if case["rows"] >= 64:  # weights
            return {"x": _normal(gen, case["dtype"], 0.02, case["rows"], k)}
        return {"x": _activations(gen, case["dtype"], case["rows"], k)}
    if kind in ("mx4_mm", "mx4_grp"):
        e, rows = case.get("e", 1), case["m"] if kind == "mx4_mm" else case["t"]
        codes, scales = _quantize(_normal(gen, "bfloat16", k**-0.5, e * case["n"], k))
        got = {"x": _activations(gen, "bfloat16", rows, k)}
        if kind == "mx4_grp":
            codes, scales = codes.view(e, case["n"], -1), scales.view(e, case["n"], -1)
            got["sizes"] = torch.tensor(_sizes(case, seed), dtype=torch.int32, device="cuda")
        return {**got, "codes": codes, "scales": scales}
    sizes = torch.tensor(_sizes(case, seed), dtype=torch.int32, device="cuda")
    x = _normal(gen, case["dtype"], 1.0, case["t"], k)
    if kind == "grad_w":
        return {"x": x, "dy": _normal(gen, case["dtype"], 0.1, case["t"], case["n"]), "sizes": sizes}
    shape = (case["e"], case["n"], k) if case["trans_w"] else (case["e"], k, case["n"])
    return {"x": x, "w": _normal(gen, case["dtype"], k**-0.5, *shape), "sizes": sizes}


# ---------------------------------------------------------------- plain form


def _quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [rows][16 * blocks] (two a byte, the even element low) and scales
    [rows][blocks] (the exponent plus 127) of blocks of 32; the last block of
    a row is filled up with zeros.  scale = 2^(floor(log2 max|x|) - 2),
    elements to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to even."""
    rows, k = x.shape
    nb = (k + 31) // 32
    v = torch.zeros((rows, nb * 32), device=x.device, dtype=torch.float32)
    v[:, :k] = x
    v = v.view(rows, nb, 32)
    top = v.abs().amax(2, keepdim=True)
    exp = ((top.view(torch.int32) >> 23) - 129).clamp(min=-127)
    y = v.abs() * ((127 - exp) << 23).view(torch.float32)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    q = (torch.round(y / step) * step).clamp(max=6.0)
    # 0, .5, 1, 1.5, 2, 3, 4, 6 -> 0 .. 7
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).view(rows, nb * 16, 2)
    return code[..., 0] | (code[..., 1] << 4), (exp + 127).to(torch.uint8).view(rows, nb)


def _dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    nib = torch.stack((codes & 15, codes >> 4), -1).view(*scales.shape, 32).int()
    mag = nib & 7
    val = torch.where(mag < 4, mag * 0.5, torch.where(mag < 6, mag - 2.0, mag * 2.0 - 8.0))
    val = torch.where(nib > 7, -val, val)
    exp = scales.int()
    scale = torch.where(exp > 0, exp << 23, 1 << 22).view(torch.float32)
    return (val * scale.unsqueeze(-1)).view(*codes.shape[:-1], -1)


def _plain(case: dict[str, Any], ins: dict[str, torch.Tensor]) -> torch.Tensor:
    kind = case["kind"]
    if kind == "mx4":
        return _dequantize(*_quantize(ins["x"]))[:, : case["k"]].to(_TORCH[case["dtype"]])
    out = _TORCH[case["out"]]
    if kind == "mx4_mm":
        return (_dequantize(*_quantize(ins["x"])) @ _dequantize(ins["codes"], ins["scales"]).t()).to(out)
    if kind == "grad_w":
        y = torch.zeros((case["e"], case["k"], case["n"]), device="cuda", dtype=torch.float32)
    else:
        y = torch.zeros((case["t"], case["n"]), device="cuda", dtype=torch.float32)
    x = _dequantize(*_quantize(ins["x"])) if kind == "mx4_grp" else ins["x"].float()
    row = 0
    for e, count in enumerate(ins["sizes"].tolist()):
        rows = slice(row, row + count)
        row += count
        if kind == "grad_w":
            y[e] = x[rows].t() @ ins["dy"][rows].float()
        elif count and kind == "mx4_grp":
            y[rows] = x[rows] @ _dequantize(ins["codes"][e], ins["scales"][e]).t()
        elif count:
            w = ins["w"][e].float()
            y[rows] = x[rows] @ (w.t() if case["trans_w"] else w)
    return y.to(out)


# ----------------------------------------------------- the framework's own


def _graph(case: dict[str, Any]) -> Any:
    import xtc_amd.graphs.xtc.op as O

    kind, k = case["kind"], case["k"]
    nb = (k + 31) // 32
    if kind == "mx4":
        x = O.tensor((case["rows"], k), case["dtype"], name="X")
        with O.graph(name="mx4_round_trip") as gb:
            codes, scales = O.mx4_quantize(x)
            y = O.mx4_dequantize(codes, scales, size=k, out_dtype=case["dtype"], name="Y")
            O.outputs(codes, scales, y)
        return gb.graph
    if kind == "mx4_mm":
        x = O.tensor((case["m"], k), "bfloat16", name="X")
        wc = O.tensor((case["n"], nb * 16), "uint8", name="W_codes")
        ws = O.tensor((case["n"], nb), "uint8", name="W_scales")
        with O.graph(name="mx4_projection") as gb:
            O.mx4_matmul(*O.mx4_quantize(x), wc, ws, out_dtype=case["out"], name="Y")
        return gb.graph
    # a graph's inputs are in the order in which the tensors were made
    if kind == "mx4_grp":
        x = O.tensor((case["t"], k), "bfloat16", name="X")
        wc = O.tensor((case["e"], case["n"], nb * 16), "uint8", name="W_codes")
        ws = O.tensor((case["e"], case["n"], nb), "uint8", name="W_scales")
        sizes = O.tensor((case["e"],), "int32", name="sizes")
        with O.graph(name="mx4_experts") as gb:
            O.grouped_mx4_matmul(*O.mx4_quantize(x), wc, ws, sizes, out_dtype=case["out"], name="Y")
        return gb.graph
    x = O.tensor((case["t"], k), case["dtype"], name="X")
    if kind == "grad_w":
        dy = O.tensor((case["t"], case["n"]), case["dtype"], name="dY")
        sizes = O.tensor((case["e"],), "int32", name="sizes")
        with O.graph(name="experts_grad_w") as gb:
            O.grouped_matmul_grad_w(x, dy, sizes, out_dtype=case["out"], name="dW")
        return gb.graph
    layout = {"layout": [0, 2, 1]} if case["trans_w"] else {}
    w = O.tensor((case["e"], k, case["n"]), case["dtype"], name="W", **layout)
    sizes = O.tensor((case["e"],), "int32", name="sizes")
    with O.graph(name="experts") as gb:
        O.grouped_matmul(x, w, sizes, out_dtype=case["out"], name="Y")
    return gb.graph


def _outputs(case: dict[str, Any]) -> list[torch.Tensor]:
    """The graph's output tensors; the last one is what the case is about."""
    kind = case["kind"]

    def empty(dtype: torch.dtype, *shape: int) -> torch.Tensor:
        return torch.empty(shape, device="cuda", dtype=dtype)

    if kind == "mx4":
        rows, k, nb = case["rows"], case["k"], (case["k"] + 31) // 32
        return [empty(torch.uint8, rows, nb * 16), empty(torch.uint8, rows, nb), empty(_TORCH[case["dtype"]], rows, k)]
    out = _TORCH[case["out"]]
    if kind == "grad_w":
        return [empty(out, case["e"], case["k"], case["n"])]
    return [empty(out, case["m"] if kind == "mx4_mm" else case["t"], case["n"])]


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    ins = _inputs(case, seed)
    state: dict[str, Any] = {"case": case, "ins": ins}
    if not own:
        return state
    from xtc_amd.backends.hip import Backend
    from xtc_amd.runtimes.hip.device import HipDevice

    backend = Backend(_graph(case))
    module = backend.get_compiler(synchronize=False, schedule_policy="strict").compile(backend.get_scheduler().schedule())
    device = HipDevice()
    device.init_device()
    device.load_module(module)
    call = device.get_module_function(module, module.payload_name)
    call.restype = None
    order = {"grouped": ("x", "w", "sizes"), "grad_w": ("x", "dy", "sizes"), "mx4": ("x",),
             "mx4_mm": ("x", "codes", "scales"), "mx4_grp": ("x", "codes", "scales", "sizes")}[case["kind"]]
    outs = _outputs(case)
    args = [ctypes.c_void_p(t.data_ptr()) for t in (*(ins[n] for n in order), *outs)]
    return {**state, "module": module, "call": call, "args": args, "outs": outs}


def run(state: dict[str, Any]) -> torch.Tensor:
    if not own:
        return _plain(state["case"], state["ins"])
    state["call"](*state["args"])
    return state["outs"][-1]


# ----------------------------------------------------------- float64 results


def _values64(x: torch.Tensor) -> torch.Tensor:
    """What x stands for in blocks of 32 4-bit floats: nearest grid points by
    comparison with the midpoints (an even neighbour takes the tie)."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(rows, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0**-125))) - 2)
    y = v.abs() / scale
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    at = torch.zeros_like(y, dtype=torch.int64)
    for mid, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        at += (y >= mid) if up else (y > mid)
    return (grid[at] * torch.sign(v) * scale).view(rows, -1)[:, :k]


def _weights64(ins: dict[str, torch.Tensor]) -> torch.Tensor:
    table = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=torch.float64, device="cuda") / 2
    codes = ins["codes"].long()
    v = torch.stack((table[codes % 16], table[codes // 16]), -1).flatten(-2)
    return v * torch.exp2(ins["scales"].double() - 127).repeat_interleave(32, -1)


def exact(case: dict[str, Any], seed: int) -> torch.Tensor:
    ins = _inputs(case, seed)
    kind = case["kind"]
    if kind == "mx4":
        return _values64(ins["x"])
    if kind in ("mx4_mm", "mx4_grp"):
        x, w = _values64(ins["x"]), _weights64(ins)[..., : case["k"]]
        if kind == "mx4_mm":
            return x @ w.t().contiguous()
    else:
        x = ins["x"].double()
        w = None if kind == "grad_w" else ins["w"]
    ends = np.cumsum(_sizes(case, seed))
    if kind == "grad_w":
        dy = ins["dy"].double()
        return torch.stack([x[a:b].t().contiguous() @ dy[a:b] for a, b in zip([0, *ends[:-1]], ends)])
    y = torch.zeros(case["t"], case["n"], dtype=torch.float64, device="cuda")
    for e, (a, b) in enumerate(zip([0, *ends[:-1]], ends)):
        we = w[e].double()
        y[a:b] = x[a:b] @ (we.t().contiguous() if kind == "mx4_grp" or case["trans_w"] else we)
    return y


# --------------------------------------------------------------------- work


def work(case: dict[str, Any]) -> dict[str, float]:
    kind, k = case["kind"], case["k"]
    nb = (k + 31) // 32
    if kind == "mx4":
        rows = case["rows"]
        return {"bytes": float(rows * (2 * k * _BYTES[case["dtype"]] + 17 * nb)), "flops": 0.0}
    n, out = case["n"], _BYTES[case["out"]]
    if kind == "mx4_mm":
        m = case["m"]
        return {"bytes": float(m * k * 2 + n * nb * 17 + m * n * out), "flops": 2.0 * m * n * k}
    t, e = case["t"], case["e"]
    rows = t - case["spare"]
    if kind == "grad_w":
        return {"bytes": float(rows * (k + n) * _BYTES[case["dtype"]] + e * k * n * out + 4 * e), "flops": 2.0 * rows * n * k}
    # the matrices of the experts that a fair router would reach
    hit = e * (1.0 - (1.0 - 1.0 / e) ** rows)
    weights = hit * (n * nb * 17 if kind == "mx4_grp" else k * n * _BYTES[case["dtype"]])
    row = k * (2 if kind == "mx4_grp" else _BYTES[case["dtype"]])
    return {"bytes": float(rows * row + t * n * out + weights + 4 * e), "flops": 2.0 * rows * n * k}
