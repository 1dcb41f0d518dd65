# SPDX-License-Identifier: BSD-3-Clause
"""Layer norm, 8-bit products and the expert layer of a few tokens: calls of
every kind that a model's layers make, with inputs, required work, a plain form
and float64 results.

Kinds of case:
  ln        y = (x - mean) / sqrt(var + eps) * w + b over rows
  ln_grad   dx, dw and db of the same for dy
  fp8       x to 8-bit floats (e4m3) and back to values: a power-of-two scale
            for each 128 elements of a row, for each 128 x 128 block, or for each
            128 elements of a row of x transposed
  fp8_mm    bf16 activations quantised by rows, times 8-bit weights [n][k] of
            128 x 128 blocks
  fp8_step  one training step of a projection from bf16 x, w and dy: y, dx and dw,
            each a product of 8-bit operands quantised on the way
  experts   a whole layer for a few tokens: router, top-k, up, activation, down,
            sum by the router's weights

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
_EPS = 1e-5


def _ln(name: str, kind: str, dtype: str, rows: int, k: int) -> dict[str, Any]:
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "k": k}


def _fp8(name: str, dtype: str, rows: int, k: int, blocks: str) -> dict[str, Any]:
    return {"name": name, "kind": "fp8", "dtype": dtype, "rows": rows, "k": k, "blocks": blocks}


def _mm(name: str, kind: str, out: str, m: int, n: int, k: int) -> dict[str, Any]:
    return {"name": name, "kind": kind, "out": out, "m": m, "n": n, "k": k}


def _experts(name: str, dtype: str, weights: str, t: int, e: int, top: int, k: int, hidden: int, act: str, normalize: bool) -> dict[str, Any]:
    return {"name": name, "kind": "experts", "dtype": dtype, "weights": weights, "t": t, "e": e, "top": top, "k": k,
            "hidden": hidden, "act": act, "normalize": normalize}


def listed() -> list[dict[str, Any]]:
    return [
        # the hidden states of four sequences at one decoding step: latency
        _ln("ln_decode", "ln", "bfloat16", 4, 4096),
        # a long prefill
        _ln("ln_prefill", "ln", "bfloat16", 32768, 4096),
        # training: all three gradients of a batch
        _ln("ln_grad", "ln_grad", "bfloat16", 16384, 4096),
        # the same in fp32 at a user's own sizes
        _ln("ln_grad_odd", "ln_grad", "float32", 1001, 333),
        # a large weight matrix brought to 8 bits, with the values that it then stands for
        _fp8("fp8_weights", "bfloat16", 8192, 8192, "square"),
        # a few fp32 rows whose last block is partial: latency
        _fp8("fp8_rows_odd", "float32", 5, 1000, "rows"),
        # one decode step of 16 sequences through a square projection: streams the 8-bit weights
        _mm("fp8_decode", "fp8_mm", "bfloat16", 16, 8192, 8192),
        # the headline matmul size on 8-bit operands
        _mm("fp8_8192", "fp8_mm", "bfloat16", 8192, 8192, 8192),
        # a training step of one projection, gradients among it
        _mm("fp8_step", "fp8_step", "bfloat16", 4096, 4096, 2048),
        # one token at two of eight bf16 experts: latency and six matrices
        _experts("layer_token", "bfloat16", "bfloat16", 1, 8, 2, 1024, 2048, "swiglu", True),
        # a decode batch over experts in 8 bits
        _experts("layer_fp8", "bfloat16", "fp8", 16, 64, 4, 2048, 1024, "swiglu", True),
        # a large decode batch over experts in 4 bits: every expert is read
        _experts("layer_mx4", "bfloat16", "mx4", 64, 16, 2, 4096, 2048, "relu", False),
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
    # most operations and bytes of a listed case of the kind
    flops = {"fp8_mm": 1.1e12, "fp8_step": 2.1e11}
    most = {"ln": 5.4e8, "ln_grad": 4.1e8, "fp8": 3.4e8, "fp8_mm": 4.0e8, "fp8_step": 1.3e8, "experts": 3.2e8}
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= most[case["kind"]] and w["flops"] <= flops.get(case["kind"], 1e18):
            del case["name"]
            return case


def _draw(rng: Any) -> dict[str, Any]:
    kind = rng.choice(("ln", "ln", "ln_grad", "ln_grad", "fp8", "fp8", "fp8_mm", "fp8_mm", "fp8_step", "experts", "experts",
                       "experts"))
    dtype = rng.choice(("float32", "bfloat16", "bfloat16"))
    out = rng.choice(("float32", "bfloat16"))
    if kind in ("ln", "ln_grad", "fp8"):
        rows = _rows(rng, 32768)
        k = _wide(rng, 64, 16384) if rng.random() < 0.7 else _log(rng, 1, 9000) | 1
        if kind == "fp8":
            return _fp8("", dtype, rows, k, rng.choice(("rows", "square", "columns")))
        return _ln("", kind, dtype, rows, k)
    if kind in ("fp8_mm", "fp8_step"):
        k = _wide(rng, 128, 8192) if rng.random() < 0.7 else _log(rng, 17, 4000) | 1
        n = _wide(rng, 64, 8192) if rng.random() < 0.7 else _log(rng, 17, 4000) | 1
        return _mm("", kind, out, _rows(rng, 8192), n, k)
    t, e = _log(rng, 1, 64), rng.choice((2, 4, 5, 8, 16, 24, 32, 64))
    weights = rng.choice((dtype, "fp8", "mx4")) if dtype == "bfloat16" else dtype
    k, hidden = _wide(rng, 128, 4096), _wide(rng, 128, 4096)
    if rng.random() < 0.25:
        k, hidden = _log(rng, 33, 2000) | 1, _log(rng, 33, 2000) | 1
    return _experts("", dtype, weights, t, e, rng.randint(1, min(8, e)), k, hidden, rng.choice(("swiglu", "swiglu", "relu")),
                    rng.random() < 0.6)


# ------------------------------------------------------------------- inputs


def _normal(gen: torch.Generator, dtype: str, std: float, *shape: int) -> torch.Tensor:
    return torch.empty(shape, device="cuda", dtype=torch.float32).normal_(0.0, std, generator=gen).to(_TORCH[dtype])


def _activations(gen: torch.Generator, dtype: str, rows: int, k: int) -> torch.Tensor:
    """Normal about an offset of each row, with a few channels sixteen times as
    large, as hidden states are."""
    x = torch.empty((rows, k), device="cuda", dtype=torch.float32).normal_(0.0, 1.0, generator=gen)
    x[:, :: max(1, k // 5)] *= 16.0
    x += torch.empty((rows, 1), device="cuda", dtype=torch.float32).normal_(0.0, 0.5, generator=gen)
    return x.to(_TORCH[dtype])


def _pack(case: dict[str, Any], w: torch.Tensor) -> tuple[torch.Tensor, ...]:
    """Matrices [e][rows][k] as the layer keeps them."""
    if case["weights"] == "fp8":
        return _fp8_quantize(w, 128)
    if case["weights"] == "mx4":
        return _mx4_quantize(w)
    return (w,)


def _inputs(case: dict[str, Any], seed: int) -> dict[str, Any]:
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, k = case["kind"], case["k"]
    if kind in ("ln", "ln_grad"):
        x = _activations(gen, case["dtype"], case["rows"], k)
        got = {"x": x, "w": 1 + _normal(gen, "float32", 0.2, k), "b": _normal(gen, "float32", 0.2, k)}
        return {**got, "dy": _normal(gen, case["dtype"], 0.1, case["rows"], k)} if kind == "ln_grad" else got
    if kind == "fp8":
        if case["blocks"] == "square":  # weights
            return {"x": _normal(gen, case["dtype"], 0.02, case["rows"], k)}
        return {"x": _activations(gen, case["dtype"], case["rows"], k)}
    if kind == "fp8_mm":
        codes, scales = _fp8_quantize(_normal(gen, "bfloat16", k**-0.5, case["n"], k), 128)
        return {"x": _activations(gen, "bfloat16", case["m"], k), "codes": codes, "scales": scales}
    if kind == "fp8_step":
        return {"x": _activations(gen, "bfloat16", case["m"], k), "w": _normal(gen, "bfloat16", k**-0.5, case["n"], k),
                "dy": _normal(gen, "bfloat16", 0.1, case["m"], case["n"])}
    e, h = case["e"], case["hidden"]
    x = _normal(gen, case["dtype"], 1.0, case["t"], k)  # normed
    router = _normal(gen, case["dtype"], 1.5 * k**-0.5, e, k)
    up = _normal(gen, case["dtype"], k**-0.5, e, 2 * h if case["act"] == "swiglu" else h, k)
    down = _normal(gen, case["dtype"], h**-0.5, e, k, h)
    return {"x": x, "router": router, "up": _pack(case, up), "down": _pack(case, down)}


# ---------------------------------------------------------------- plain form


def _to_blocks(x: torch.Tensor, rows: int) -> torch.Tensor:
    """x [..., r, k] filled up with zeros to [..., r / rows, rows, k / 128, 128]."""
    r, k = x.shape[-2:]
    v = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -r % rows))
    return v.view(*x.shape[:-2], v.shape[-2] // rows, rows, v.shape[-1] // 128, 128)


def _fp8_quantize(x: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [..., r][128 * blocks] (e4m3: sign, 4 exponent bits, 3 mantissa
    bits) and scales [..., r / rows][blocks] (the exponent plus 127): the smallest
    power of two that brings a block's largest magnitude to at most 448."""
    r = x.shape[-2]
    v = _to_blocks(x, rows)
    top = v.abs().amax((-3, -1), keepdim=True).view(torch.int32)
    # past 1.75 times a power of two the next one
    exp = ((top >> 23) - 127 - 8 + ((top & 0x7FFFFF) > 0x600000).int()).clamp(min=-127)
    y = v.abs() * ((127 - exp) << 23).view(torch.float32)
    low = ((y.view(torch.int32) >> 23) - 127).clamp(min=-6)  # the element's exponent, that of subnormals at least
    n = torch.round(y * ((127 + 3 - low) << 23).view(torch.float32)).int()  # in steps of 2^(low - 3)
    code = (n + 8 * (low + 6)).to(torch.uint8)
    code = code | (torch.signbit(v).to(torch.uint8) << 7)
    scales = (exp + 127).to(torch.uint8).squeeze(-1).squeeze(-2)
    return code.flatten(-2).flatten(-3, -2)[..., :r, :].contiguous(), scales.contiguous()


def _fp8_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What the codes stand for, [..., r][128 * blocks]."""
    c = codes.int()
    low = (c >> 3) & 15
    val = torch.where(low > 0, (c & 7) + 8, c & 7).float() * ((low.clamp(min=1) - 10 + 127) << 23).view(torch.float32)
    val = torch.where(c > 127, -val, val)
    s = scales.int()
    scale = torch.where(s > 0, s << 23, 1 << 22).view(torch.float32)
    scale = scale.repeat_interleave(128, -1)
    if scales.shape[-2] != codes.shape[-2]:
        scale = scale.repeat_interleave(128, -2)[..., : codes.shape[-2], :]
    return val * scale


def _fp8_rounded(x: torch.Tensor, rows: int) -> torch.Tensor:
    return _fp8_values(*_fp8_quantize(x, rows))[..., : x.shape[-1]]


def _mx4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Microscaled 4-bit floats: blocks of 32, codes two a byte, the even element
    low, scale = 2^(floor(log2 max|x|) - 2)."""
    k = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -k % 32))
    v = v.view(*x.shape[:-1], -1, 32)
    exp = ((v.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 129).clamp(min=-127)
    y = v.abs() * ((127 - exp) << 23).view(torch.float32)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    q = (torch.round(y / step) * step).clamp(max=6.0)
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).view(*x.shape[:-1], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), (exp + 127).to(torch.uint8).squeeze(-1)


def _mx4_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    nib = torch.stack((codes & 15, codes >> 4), -1).view(*scales.shape, 32).int()
    mag = nib & 7
    val = torch.where(mag < 4, mag * 0.5, torch.where(mag < 6, mag - 2.0, mag * 2.0 - 8.0))
    val = torch.where(nib > 7, -val, val)
    exp = scales.int()
    scale = torch.where(exp > 0, exp << 23, 1 << 22).view(torch.float32)
    return (val * scale.unsqueeze(-1)).view(*codes.shape[:-1], -1)


def _unpack(case: dict[str, Any], packed: tuple[torch.Tensor, ...], e: int, k: int) -> torch.Tensor:
    """Matrix e as float32 [rows][k]."""
    if case["weights"] == "fp8":
        return _fp8_values(packed[0][e], packed[1][e])[:, :k]
    if case["weights"] == "mx4":
        return _mx4_values(packed[0][e], packed[1][e])[:, :k]
    return packed[0][e].float()


def _normed(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(x - mean) / sqrt(var + eps) and 1 / sqrt(var + eps)."""
    c = x.float() - x.float().mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    return c * r, r


def _plain_layer(case: dict[str, Any], ins: dict[str, Any]) -> torch.Tensor:
    x, k, h = ins["x"].float(), case["k"], case["hidden"]
    logits = x @ ins["router"].float().t()
    p = torch.exp(logits - logits.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    chosen = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, : case["top"]]
    weight = torch.gather(p, 1, chosen)
    if case["normalize"]:
        weight = weight / weight.sum(1, keepdim=True)
    y = torch.zeros_like(x)
    for e in range(case["e"]):
        rows, slot = torch.nonzero(chosen == e, as_tuple=True)
        if not len(rows):
            continue
        up = x[rows] @ _unpack(case, ins["up"], e, k).t()
        act = up[:, :h] / (1 + torch.exp(-up[:, :h])) * up[:, h:] if case["act"] == "swiglu" else up.clamp(min=0.0)
        y[rows] += weight[rows, slot].unsqueeze(1) * (act @ _unpack(case, ins["down"], e, h).t())
    return y.to(_TORCH[case["dtype"]])


def _plain(case: dict[str, Any], ins: dict[str, Any]) -> Any:
    kind = case["kind"]
    if kind == "ln":
        return (_normed(ins["x"])[0] * ins["w"] + ins["b"]).to(ins["x"].dtype)
    if kind == "ln_grad":
        xh, r = _normed(ins["x"])
        dy = ins["dy"].float()
        g = dy * ins["w"]
        dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        return dx.to(ins["x"].dtype), (dy * xh).sum(0), dy.sum(0)
    if kind == "fp8":
        x = ins["x"].t().contiguous() if case["blocks"] == "columns" else ins["x"]
        return _fp8_rounded(x, 128 if case["blocks"] == "square" else 1).to(x.dtype)
    if kind == "fp8_mm":
        w = _fp8_values(ins["codes"], ins["scales"])[:, : case["k"]]
        return (_fp8_rounded(ins["x"], 1) @ w.t()).to(_TORCH[case["out"]])
    if kind == "fp8_step":
        x, w, dy = ins["x"], ins["w"], ins["dy"]
        q = _fp8_rounded(w, 128)
        y = _fp8_rounded(x, 1) @ q.t()
        dx = _fp8_rounded(dy, 1) @ q
        dw = _fp8_rounded(dy.t().contiguous(), 1) @ _fp8_rounded(x.t().contiguous(), 1).t()
        return y.to(_TORCH[case["out"]]), dx.to(_TORCH[case["out"]]), dw
    return _plain_layer(case, ins)


# ----------------------------------------------------- the framework's own


def _graph(case: dict[str, Any], ins: dict[str, Any]) -> tuple[Any, list[torch.Tensor], list[torch.Tensor]]:
    """The case's graph, its inputs and its output tensors."""
    import xtc_amd.graphs.xtc.op as O

    names = {torch.float32: "float32", torch.bfloat16: "bfloat16", torch.uint8: "uint8"}
    args: list[torch.Tensor] = []

    def given(t: torch.Tensor, name: str) -> Any:
        args.append(t)  # a graph's inputs are in the order in which the tensors were made
        return O.tensor(tuple(t.shape), names[t.dtype], name=name)

    def empty(dtype: str, *shape: int) -> torch.Tensor:
        return torch.empty(shape, device="cuda", dtype=_TORCH.get(dtype, torch.uint8))

    kind, k = case["kind"], case["k"]
    x = given(ins["x"], "X")
    if kind == "ln":
        w, b = given(ins["w"], "W"), given(ins["b"], "B")
        with O.graph(name="norm") as gb:
            O.layer_norm(x, w, b, eps=_EPS, name="Y")
        return gb.graph, args, [torch.empty_like(ins["x"])]
    if kind == "ln_grad":
        w, dy = given(ins["w"], "W"), given(ins["dy"], "dY")
        with O.graph(name="norm_grad") as gb:
            O.outputs(*O.layer_norm_grad(x, w, dy, eps=_EPS))
        return gb.graph, args, [torch.empty_like(ins["x"]), empty("float32", k), empty("float32", k)]
    if kind == "fp8":
        t, square = case["blocks"] == "columns", case["blocks"] == "square"
        rows, size = (k, case["rows"]) if t else (case["rows"], k)
        nb = (size + 127) // 128
        with O.graph(name="fp8_round_trip") as gb:
            codes, scales = O.fp8_quantize(x, rows=128 if square else 1, transpose=t)
            O.outputs(codes, scales, O.fp8_dequantize(codes, scales, size=size, out_dtype=case["dtype"], name="Y"))
        return gb.graph, args, [empty("uint8", rows, nb * 128), empty("uint8", (rows + 127) // 128 if square else rows, nb),
                                empty(case["dtype"], rows, size)]
    if kind == "fp8_mm":
        wc, ws = given(ins["codes"], "W_codes"), given(ins["scales"], "W_scales")
        with O.graph(name="fp8_projection") as gb:
            O.fp8_matmul(*O.fp8_quantize(x), wc, ws, out_dtype=case["out"], name="Y")
        return gb.graph, args, [empty(case["out"], case["m"], case["n"])]
    if kind == "fp8_step":
        w, dy = given(ins["w"], "W"), given(ins["dy"], "dY")
        with O.graph(name="fp8_training_step") as gb:
            y = O.fp8_matmul(*O.fp8_quantize(x), *O.fp8_quantize(w, rows=128), out_dtype=case["out"], name="Y")
            dx = O.fp8_matmul(*O.fp8_quantize(dy), *O.fp8_quantize(w, rows=128, transpose=True), out_dtype=case["out"], name="dX")
            dw = O.fp8_matmul(*O.fp8_quantize(dy, transpose=True), *O.fp8_quantize(x, transpose=True), out_dtype="float32", name="dW")
            O.outputs(y, dx, dw)
        return gb.graph, args, [empty(case["out"], case["m"], case["n"]), empty(case["out"], case["m"], k),
                                empty("float32", case["n"], k)]
    router = given(ins["router"], "router")
    up = tuple(given(t, f"up{i}") for i, t in enumerate(ins["up"]))
    down = tuple(given(t, f"down{i}") for i, t in enumerate(ins["down"]))
    with O.graph(name="layer") as gb:
        O.expert_layer(x, router, up if len(up) > 1 else up[0], down if len(down) > 1 else down[0], top_k=case["top"],
                       activation=case["act"], normalize=case["normalize"], name="Y")
    return gb.graph, args, [torch.empty_like(ins["x"])]


def prepare(case: dict[str, Any], seed: int) -> dict[str, Any]:
    ins = _inputs(case, seed)
    state: dict[str, Any] = {"case": case, "ins": ins}
    if not own:
        return state
    from xtc_amd.backends.hip import Backend
    from xtc_amd.runtimes.hip.device import HipDevice

    graph, given, outs = _graph(case, ins)
    backend = Backend(graph)
    module = backend.get_compiler(synchronize=False, schedule_policy="strict").compile(backend.get_scheduler().schedule())
    device = HipDevice()
    device.init_device()
    device.load_module(module)
    call = device.get_module_function(module, module.payload_name)
    call.restype = None
    args = [ctypes.c_void_p(t.data_ptr()) for t in (*given, *outs)]
    return {**state, "module": module, "call": call, "args": args, "outs": outs, "given": given}


def run(state: dict[str, Any]) -> Any:
    if not own:
        return _plain(state["case"], state["ins"])
    state["call"](*state["args"])
    # codes and scales are returned as the values that they stand for
    outs = state["outs"]
    return tuple(outs) if state["case"]["kind"] in ("ln_grad", "fp8_step") else outs[-1]


# ----------------------------------------------------------- float64 results


def _grid64(x: torch.Tensor, rows: int) -> torch.Tensor:
    """What x stands for in 8-bit floats: the nearest of the 127 magnitudes by
    comparison with their midpoints (an even neighbour takes the tie)."""
    r, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 128, 0, -r % rows))
    v = v.view(v.shape[0] // rows, rows, -1, 128)
    m, e = torch.frexp(v.abs().amax((1, 3), keepdim=True))
    scale = torch.exp2((e - 9 + (m > 0.875).int()).clamp(min=-127).double())
    grid = torch.tensor([i * 2.0**-9 for i in range(8)] + [(8 + i) * 2.0 ** (e - 10) for e in range(1, 16) for i in range(8)][:-1],
                        dtype=torch.float64, device=x.device)
    mids = (grid[1:] + grid[:-1]) / 2
    y = v.abs() / scale
    at = torch.bucketize(y, mids)  # midpoints below y
    tie = (at < 126) & (y == mids[at.clamp(max=125)])
    at = torch.where(tie & (at % 2 == 1), at + 1, at)
    return (grid[at] * torch.sign(v) * scale).reshape(-1, v.shape[2] * 128)[:r, :k]


def _fp8_weights64(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    table = [i * 2.0**-9 for i in range(8)] + [(8 + i) * 2.0 ** (e - 10) for e in range(1, 16) for i in range(8)]
    table = torch.tensor(table + [-v for v in table], dtype=torch.float64, device=codes.device)
    r, k = codes.shape
    s = torch.exp2(scales.double() - 127)[torch.arange(r, device=codes.device) // (1 if scales.shape[0] == r else 128)]
    return table[codes.long()] * s[:, torch.arange(k, device=codes.device) // 128]


def _mx4_weights64(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    table = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=torch.float64, device=codes.device) / 2
    c = codes.long()
    return torch.stack((table[c % 16], table[c // 16]), -1).flatten(-2) * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _layer64(case: dict[str, Any], ins: dict[str, Any]) -> torch.Tensor:
    x, k, h = ins["x"].double(), case["k"], case["hidden"]
    logits = x @ ins["router"].double().t().contiguous()
    y = torch.zeros_like(x)
    matrix = {"fp8": _fp8_weights64, "mx4": _mx4_weights64}.get(case["weights"], lambda w: w.double())
    known: dict[int, tuple[torch.Tensor, torch.Tensor]] = {}
    for t, row in enumerate(logits.tolist()):
        order = sorted(range(case["e"]), key=lambda e: (-row[e], e))[: case["top"]]
        shares = np.exp(np.array(row) - max(row))
        total = shares[order].sum() if case["normalize"] else shares.sum()
        for e in order:
            if e not in known:
                known[e] = (matrix(*(p[e] for p in ins["up"]))[:, :k], matrix(*(p[e] for p in ins["down"]))[:, :h])
            a = known[e][0] @ x[t]
            a = a[:h] * torch.sigmoid(a[:h]) * a[h:] if case["act"] == "swiglu" else torch.relu(a)
            y[t] += float(shares[e] / total) * (known[e][1] @ a)
    return y


def exact(case: dict[str, Any], seed: int) -> Any:
    ins = _inputs(case, seed)
    kind = case["kind"]
    if kind == "experts":
        return _layer64(case, ins)
    x = ins["x"].double()
    if kind in ("ln", "ln_grad"):
        n = case["k"]
        mean = x.sum(1) / n
        dev = torch.sqrt(((x - mean[:, None]) ** 2).sum(1) / n + _EPS)
        z = (x - mean[:, None]) / dev[:, None]
        if kind == "ln":
            return z * ins["w"].double() + ins["b"].double()
        dy = ins["dy"].double()
        dz = dy * ins["w"].double()
        dx = (n * dz - dz.sum(1)[:, None] - z * (dz * z).sum(1)[:, None]) / (n * dev[:, None])
        return dx, (z * dy).sum(0), dy.sum(0)
    if kind == "fp8":
        if case["blocks"] == "columns":
            x = x.t().contiguous()
        return _grid64(x, 128 if case["blocks"] == "square" else 1)
    if kind == "fp8_mm":
        return _grid64(x, 1) @ _fp8_weights64(ins["codes"], ins["scales"])[:, : case["k"]].t().contiguous()
    w, dy = _grid64(ins["w"], 128), ins["dy"]
    return (_grid64(x, 1) @ w.t().contiguous(), _grid64(dy, 1) @ w,
            _grid64(dy.t().contiguous(), 1) @ _grid64(x.t().contiguous(), 1).t().contiguous())


# --------------------------------------------------------------------- work


def work(case: dict[str, Any]) -> dict[str, float]:
    kind, k = case["kind"], case["k"]
    nb = (k + 127) // 128
    if kind in ("ln", "ln_grad"):
        size = case["rows"] * k * _BYTES[case["dtype"]]
        return {"bytes": float(2 * size + 8 * k if kind == "ln" else 3 * size + 12 * k), "flops": 0.0}
    if kind == "fp8":
        rows, size = (k, case["rows"]) if case["blocks"] == "columns" else (case["rows"], k)
        nb = (size + 127) // 128
        scales = nb * ((rows + 127) // 128 if case["blocks"] == "square" else rows)
        return {"bytes": float(2 * rows * size * _BYTES[case["dtype"]] + rows * nb * 128 + scales), "flops": 0.0}
    if kind == "fp8_mm":
        m, n = case["m"], case["n"]
        return {"bytes": float(2 * m * k + n * nb * 128 + (n + 127) // 128 * nb + m * n * _BYTES[case["out"]]), "flops": 2.0 * m * n * k}
    if kind == "fp8_step":
        m, n, out = case["m"], case["n"], _BYTES[case["out"]]
        return {"bytes": float(2 * (m * k + n * k + m * n) + out * (m * n + m * k) + 4 * n * k), "flops": 6.0 * m * n * k}
    t, e, h, top, elem = case["t"], case["e"], case["hidden"], case["top"], _BYTES[case["dtype"]]
    ups = 2 * h if case["act"] == "swiglu" else h

    def matrix(rows: int, depth: int) -> int:
        if case["weights"] == "fp8":
            return rows * ((depth + 127) // 128) * 128
        if case["weights"] == "mx4":
            return rows * ((depth + 31) // 32) * 17
        return rows * depth * elem

    # the matrices of the experts that a fair router would reach
    hit = e * (1.0 - (1.0 - top / e) ** t)
    return {"bytes": float(hit * (matrix(ups, k) + matrix(k, h)) + elem * (e * k + 2 * t * k)),
            "flops": 2.0 * t * top * (ups * k + k * h) + 2.0 * t * e * k}
