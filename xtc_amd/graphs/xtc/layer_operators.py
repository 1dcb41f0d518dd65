# SPDX-License-Identifier: BSD-3-Clause
"""Operators of a model's layers beside the products: layer norm with its
gradients, 8-bit operands with their product, and the whole layer of experts for
a few tokens, with their numpy semantics (extensions: the reference's operators,
src/xtc/graphs/xtc/operators.py:159-804, have none of them).

layer_norm, layer_norm_grad_x, layer_norm_grad_weight, layer_norm_grad_bias: the
norm of the rows along the last axis; sums in double precision here.

fp8_scales, fp8_codes, fp8_dequantize, fp8_matmul: 8-bit floats
(xtc_amd.utils.fp8) as two uint8 tensors, codes and scales.

expert_layer: router, choice, up, activation, down and weighted sum.
"""

from __future__ import annotations

from typing import Any

import numpy as np

from ...utils.bf16 import is_bf16, round_to_bf16
from ...utils.fp8 import BLOCK, blocks_of, fp8_codes, fp8_scales, fp8_values
from ...utils.mx4 import blocks_of as mx4_blocks_of
from ...utils.mx4 import mx4_values
from .data import XTCTensor, XTCTensorType
from .expert_operators import _Blocks, _float_result
from .operation import XTCOperation
from .operators import XTCOperator, _out_dtype

__all__ = [
    "XTCOperLayerNorm",
    "XTCOperLayerNormGradX",
    "XTCOperLayerNormGradWeight",
    "XTCOperLayerNormGradBias",
    "XTCOperFp8Scales",
    "XTCOperFp8Codes",
    "XTCOperFp8Dequantize",
    "XTCOperFp8Matmul",
    "XTCOperExpertLayer",
    "MOST_TOKENS",
    "MOST_EXPERTS",
    "MOST_CHOSEN",
    "FP8_SUMS",
]

# of expert_layer: tokens, experts, experts of a token
MOST_TOKENS, MOST_EXPERTS, MOST_CHOSEN = 64, 256, 16
# how fp8_matmul adds up: XTC_HIP_SUMS_..
FP8_SUMS = ("fp32", "fp8", "any")


def _eps(op: XTCOperator) -> float:
    eps = float(getattr(op.attrs, "eps", 1e-5))
    if not 0 <= eps <= 3.4e38:
        raise ValueError(f"{op.name}: eps {eps} is not a finite number from 0 on")
    return eps


def _rows_type(name: str, t: Any) -> tuple[int, ...]:
    if str(t.dtype) not in ("float32", "bfloat16") or len(t.constant_shape) < 1:
        raise ValueError(f"{name} expects float32 or bfloat16 rows, got {t}")
    return t.constant_shape  # type: ignore[no-any-return]


def _same_rows(name: str, x: Any, dy: Any) -> None:
    if str(x.dtype) != str(dy.dtype) or x.constant_shape != dy.constant_shape:
        raise ValueError(f"{name}: x {x} and dy {dy} must be of one type and shape")


def _params(name: str, x: Any, *params: Any) -> None:
    dtypes = {str(p.dtype) for p in params}
    if len(dtypes) != 1 or not dtypes <= {"float32", str(x.dtype)} or any(p.constant_shape != x.constant_shape[-1:] for p in params):
        raise ValueError(f"{name}: parameters must be ({x.constant_shape[-1]},) of float32 or {x.dtype}: {[str(p) for p in params]}")


class _Rows:
    """Iteration space of the row-wise operators: rows, and the elements that are
    summed over."""

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[no-untyped-def]
        shape = outs_types[0].constant_shape
        names = tuple(f"d{i}" for i in range(len(shape)))
        return self._operation(  # type: ignore[attr-defined]
            inps_types, outs_types, dict(zip(names, shape)), ("P",) * len(shape),
            tuple(names[-len(t.constant_shape):] for t in inps_types), (names,))


class _Columns:
    """Iteration space of the sums over rows."""

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[no-untyped-def]
        shape = inps_types[0].constant_shape
        names = tuple(f"d{i}" for i in range(len(shape)))
        return self._operation(  # type: ignore[attr-defined]
            inps_types, outs_types, dict(zip(names, shape)), (*("R",) * (len(shape) - 1), "P"),
            tuple(names for _ in inps_types), (names[-1:],))


def _normed(x: np.ndarray, eps: float) -> tuple[np.ndarray, np.ndarray]:
    """(x - mean) r and r, in double precision."""
    with np.errstate(invalid="ignore", divide="ignore"):
        c = x.astype(np.float64) - x.astype(np.float64).mean(-1, keepdims=True)
        r = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        return c * r, r


class XTCOperLayerNorm(_Rows, XTCOperator):
    """y = (x - mean) / sqrt(variance + eps) * weight + bias over the last axis.

    x (..., K), weight (K,), bias (K,) -> (..., K).  Attribute eps (1e-5).
    """

    def __init__(self, **attrs: Any) -> None:
        super().__init__("layer_norm", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        x, w, b = inputs_types
        _eps(self)
        shape = _rows_type(self.name, x)
        _params(self.name, x, w, b)
        return [XTCTensorType(shape=shape, dtype=x.dtype, device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        x, w, b = (i.numpy() for i in inputs)
        y = _normed(x, _eps(self))[0] * w + b
        return [self._check(XTCTensor(y, dtype=inputs[0].type.dtype), inputs)]


class XTCOperLayerNormGradX(_Rows, XTCOperator):
    """The gradient of layer_norm's x: x (..., K), weight (K,), dy (..., K) -> (..., K)."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("layer_norm_grad_x", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        x, w, dy = inputs_types
        _eps(self)
        shape = _rows_type(self.name, x)
        _same_rows(self.name, x, dy)
        _params(self.name, x, w)
        return [XTCTensorType(shape=shape, dtype=x.dtype, device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        x, w, dy = (i.numpy() for i in inputs)
        xh, r = _normed(x, _eps(self))
        g = dy.astype(np.float64) * w
        dx = r * (g - g.mean(-1, keepdims=True) - xh * (g * xh).mean(-1, keepdims=True))
        return [self._check(XTCTensor(dx, dtype=inputs[0].type.dtype), inputs)]


class XTCOperLayerNormGradWeight(_Columns, XTCOperator):
    """The gradient of layer_norm's weight: x (..., K), dy (..., K) -> (K,) float32."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("layer_norm_grad_weight", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        x, dy = inputs_types
        _eps(self)
        shape = _rows_type(self.name, x)
        _same_rows(self.name, x, dy)
        return [XTCTensorType(shape=shape[-1:], dtype="float32", device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        x, dy = (i.numpy() for i in inputs)
        dw = (_normed(x, _eps(self))[0] * dy).reshape(-1, x.shape[-1]).sum(0)
        return [self._check(XTCTensor(dw, dtype="float32"), inputs)]


class XTCOperLayerNormGradBias(_Columns, XTCOperator):
    """The gradient of layer_norm's bias: dy (..., K) -> (K,) float32."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("layer_norm_grad_bias", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        shape = _rows_type(self.name, inputs_types[0])
        return [XTCTensorType(shape=shape[-1:], dtype="float32", device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        dy = inputs[0].numpy().astype(np.float64)
        return [self._check(XTCTensor(dy.reshape(-1, dy.shape[-1]).sum(0), dtype="float32"), inputs)]


# ------------------------------------------------------------- 8-bit operands


def _fp8_source(op: XTCOperator, t: Any) -> tuple[tuple[int, ...], int]:
    """Shape of the quantised matrices (transposed where the attribute says so) and
    the rows of a block."""
    if str(t.dtype) not in ("float32", "bfloat16") or len(t.constant_shape) < 2:
        raise ValueError(f"{op.name} expects a float32 or bfloat16 tensor of rank >= 2, got {t}")
    rows = getattr(op.attrs, "rows", 1)
    if rows not in (1, BLOCK):
        raise ValueError(f"{op.name}: blocks of {rows} rows (they have 1 or {BLOCK})")
    shape = t.constant_shape
    if getattr(op.attrs, "transpose", False):
        shape = (*shape[:-2], shape[-1], shape[-2])
    return shape, rows


def _fp8_scales_shape(shape: tuple[int, ...], rows: int) -> tuple[int, ...]:
    return (*shape[:-2], -(-shape[-2] // rows), blocks_of(shape[-1]))


def _fp8_pair(name: str, codes: Any, scales: Any) -> tuple[tuple[int, ...], int]:
    """Shape of the codes of a pair of tensors and the rows of a block."""
    c, s = codes.constant_shape, scales.constant_shape
    if str(codes.dtype) == "uint8" and str(scales.dtype) == "uint8" and len(c) >= 2 and c[-1] % BLOCK == 0:
        for rows in (1, BLOCK):
            if s == _fp8_scales_shape(c, rows):
                return c, rows
    raise ValueError(f"{name}: codes (..., R, 128 B) and scales (..., R or ceil(R / 128), B) must be uint8: {codes} {scales}")


def _turned(op: XTCOperator, x: np.ndarray) -> np.ndarray:
    return np.ascontiguousarray(x.swapaxes(-1, -2)) if getattr(op.attrs, "transpose", False) else x


class XTCOperFp8Scales(_Blocks, XTCOperator):
    """Scales of the blocks of x: (..., R, K) -> (..., ceil(R / rows), ceil(K / 128)) uint8.
    Attributes rows (1, or 128: blocks of 128 x 128) and transpose (those of the
    transposed matrices)."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("fp8_scales", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        shape = _fp8_scales_shape(*_fp8_source(self, inputs_types[0]))
        return [XTCTensorType(shape=shape, dtype="uint8", device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        _, rows = _fp8_source(self, inputs[0].type)
        return [self._check(XTCTensor(fp8_scales(_turned(self, inputs[0].numpy()), rows), dtype="uint8"), inputs)]


class XTCOperFp8Codes(_Blocks, XTCOperator):
    """Codes of x for given scales: (..., R, K) and fp8_scales' shape -> (..., R, 128 ceil(K
    / 128)) uint8.  0 where the scale is 255; elsewhere 448 of its sign for what
    passes 448 scale, infinities among it, and the NaN code of its sign for a NaN."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("fp8_codes", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        shape, rows = _fp8_source(self, inputs_types[0])
        scales = inputs_types[1]
        if str(scales.dtype) != "uint8" or scales.constant_shape != _fp8_scales_shape(shape, rows):
            raise ValueError(f"{self.name}: scales {scales} do not match {inputs_types[0]}")
        return [XTCTensorType(shape=(*shape[:-1], BLOCK * blocks_of(shape[-1])), dtype="uint8", device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        _, rows = _fp8_source(self, inputs[0].type)
        codes = fp8_codes(_turned(self, inputs[0].numpy()), inputs[1].numpy(), rows)
        return [self._check(XTCTensor(codes, dtype="uint8"), inputs)]


class XTCOperFp8Dequantize(_Blocks, XTCOperator):
    """Values of codes and scales: (..., R, 128 B), (..., R or ceil(R / 128), B) -> (..., R,
    size), size defaulting to 128 B, of type out_dtype (float32)."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("fp8_dequantize", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        shape, _ = _fp8_pair(self.name, *inputs_types)
        size = getattr(self.attrs, "size", None) or shape[-1]
        if BLOCK * blocks_of(size) != shape[-1]:
            raise ValueError(f"{self.name}: {shape[-1] // BLOCK} blocks do not hold rows of {size} elements")
        out = _float_result(self.name, "uint8", getattr(self.attrs, "out_dtype", None) or "float32")
        return [XTCTensorType(shape=(*shape[:-1], size), dtype=out, device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        t = self.forward_types([i.type for i in inputs])[0]
        values = fp8_values(inputs[0].numpy(), inputs[1].numpy(), t.constant_shape[-1])
        return [self._check(XTCTensor(values, dtype=t.dtype), inputs)]


class XTCOperFp8Matmul(XTCOperator):
    """c[i, j] = sum_k a[i, k] b[j, k] of 8-bit operands.

    a codes (M, 128 B) and scales (M, B), b codes (N, 128 B) and scales (N, B) or
    (ceil(N / 128), B) -> (M, N) of type out_dtype (float32).  Attribute sums, on the
    GPU: "fp32" (fp32 sums of exact products, for scale bytes from 3 to 246), "fp8" (those
    of the 8-bit matrix instructions, at twice the rate: off by up to 2^-12 sum |a b|, by
    1.5e-5 of themselves for normal numbers) or "any" (the faster of the two for a bfloat16
    result, whichever its sizes make it).
    """

    def __init__(self, **attrs: Any) -> None:
        super().__init__("fp8_matmul", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        a, a_rows = _fp8_pair(self.name, *inputs_types[:2])
        b, _ = _fp8_pair(self.name, *inputs_types[2:4])
        if len(a) != 2 or len(b) != 2 or a[1] != b[1]:
            raise ValueError(f"{self.name} expects operands of one depth: codes {a} {b}")
        if a_rows != 1:
            raise ValueError(f"{self.name}: a has a scale for every {BLOCK} elements of a row, got {inputs_types[1]}")
        if (sums := getattr(self.attrs, "sums", "fp32")) not in FP8_SUMS:
            raise ValueError(f"{self.name}: sums {sums!r} are none of {FP8_SUMS}")
        out = _float_result(self.name, "uint8", getattr(self.attrs, "out_dtype", None) or "float32")
        return [XTCTensorType(shape=(a[0], b[0]), dtype=out, device=self.device)]

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[override]
        m, n = outs_types[0].constant_shape
        return self._operation(inps_types, outs_types, {"i": m, "j": n, "k": inps_types[0].constant_shape[1]}, ("P", "P", "R"),
                               (("i", "k"), ("i", "block(k)"), ("j", "k"), ("block(j)", "block(k)")), (("i", "j"),))

    def forward(self, inputs):  # type: ignore[override]
        ac, asc, bc, bsc = (i.numpy() for i in inputs)
        out = self.forward_types([i.type for i in inputs])[0].dtype
        a, b = (fp8_values(c, s, dtype=np.float64) for c, s in ((ac, asc), (bc, bsc)))
        return [self._check(XTCTensor(np.dot(a, b.T), dtype=out), inputs)]


# --------------------------------------------------------------- expert layer


class XTCOperExpertLayer(XTCOperator):
    """A whole layer of experts for a few tokens:
    l = x router^T, p = softmax(l); of the top_k largest l (ties: the lowest
    expert) y = sum p[e] down[e] act(up[e] x), with `normalize` the p divided by
    their sum.  act: "relu", or "swiglu": silu(u[:H]) u[H:] of up's 2 H rows.

    x (T, K), T <= 64, router (E, K), E <= 256, up (E, H or 2 H, K), down (E, K, H) of
    x's type, or of bfloat16 x with up and down each as two uint8 tensors, codes and
    scales: 8-bit floats (scales (E, ceil(R / 128), B)) or microscaled 4-bit floats
    (scales (E, R, B)) -> (T, K) of x's type.  p[e] act(..) is kept in hidden_dtype between
    the products, float32 or x's type.  A NaN among a token's l makes its row NaN.  On the
    GPU an infinity in down gives NaN where bfloat16 layers keep float32, and 8-bit scale
    bytes below 3 or past 246 take values out of bfloat16's range.
    Attributes top_k (2), activation ("swiglu"), normalize (True), hidden_dtype (float32).
    """

    def __init__(self, **attrs: Any) -> None:
        super().__init__("expert_layer", **attrs)

    def layer(self, inputs_types: Any) -> dict[str, Any]:
        """Sizes, activation and the type of the matrices."""
        x, router = inputs_types[:2]
        top_k = getattr(self.attrs, "top_k", 2)
        activation = getattr(self.attrs, "activation", "swiglu")
        if activation not in ("relu", "swiglu"):
            raise ValueError(f"{self.name}: activation {activation!r} is neither 'relu' nor 'swiglu'")
        xs = _rows_type(self.name, x)
        if len(xs) != 2 or len(router.constant_shape) != 2 or str(router.dtype) != str(x.dtype) or router.constant_shape[1] != xs[1]:
            raise ValueError(f"{self.name} expects x (T, K) and router (E, K) of one type: {x} {router}")
        hidden = getattr(self.attrs, "hidden_dtype", "float32")
        if hidden not in ("float32", str(x.dtype)):
            raise ValueError(f"{self.name}: hidden_dtype {hidden!r} is neither float32 nor x's type {x.dtype}")
        (t, k), e = xs, router.constant_shape[0]
        if t > MOST_TOKENS or e > MOST_EXPERTS or not isinstance(top_k, int) or not 1 <= top_k <= min(e, MOST_CHOSEN):
            raise ValueError(f"{self.name}: {t} tokens (at most {MOST_TOKENS}), {e} experts (at most {MOST_EXPERTS}), top_k "
                             f"{top_k} (from 1 to {min(e, MOST_CHOSEN)}); more tokens take the products by group")
        if len(inputs_types) == 4:
            up, down = inputs_types[2:]
            weights = "dense"
            if not str(up.dtype) == str(down.dtype) == str(x.dtype):
                raise ValueError(f"{self.name}: up {up} and down {down} must be of x's type {x.dtype}")
            shapes = [up.constant_shape, down.constant_shape]
        else:
            if str(x.dtype) != "bfloat16":
                raise ValueError(f"{self.name}: 8-bit and 4-bit matrices take bfloat16 x, got {x}")
            pairs = [(inputs_types[2], inputs_types[3]), (inputs_types[4], inputs_types[5])]
            mx4 = [len(c.constant_shape) == 3 and c.constant_shape == (*s.constant_shape[:-1], 16 * s.constant_shape[-1])
                   for c, s in pairs]
            weights = "mx4" if all(mx4) else "fp8"
            shapes = [c.constant_shape for c, _ in pairs]
            for c, s in pairs:
                shape = c.constant_shape
                if any(str(i.dtype) != "uint8" for i in (c, s)) or len(shape) != 3 or (
                        weights == "fp8" and s.constant_shape != (shape[0], blocks_of(shape[1]), shape[2] // BLOCK)):
                    raise ValueError(f"{self.name}: codes and scales must be both those of 8-bit floats in blocks of 128 x 128 "
                                     f"or both those of 4-bit floats, uint8: {[str(i) for i in inputs_types[2:]]}")
        if len(shapes[0]) != 3 or len(shapes[1]) != 3:
            raise ValueError(f"{self.name} expects up (E, R, K) and down (E, K, H): {shapes}")
        h = shapes[0][1]
        if activation == "swiglu":
            if h % 2:
                raise ValueError(f"{self.name}: up has {h} rows, an odd number, for two halves")
            h //= 2
        packed = {"dense": lambda n: n, "fp8": lambda n: BLOCK * blocks_of(n), "mx4": lambda n: 16 * mx4_blocks_of(n)}[weights]
        if h < 1 or shapes[0] != (e, shapes[0][1], packed(k)) or shapes[1] != (e, k, packed(h)):
            raise ValueError(f"{self.name}: up {shapes[0]} and down {shapes[1]} do not match {e} experts of width {k} and hidden {h}")
        return {"T": t, "E": e, "K": k, "H": h, "top_k": top_k, "activation": activation, "weights": weights, "hidden": hidden,
                "normalize": bool(getattr(self.attrs, "normalize", True))}

    def forward_types(self, inputs_types):  # type: ignore[override]
        d = self.layer(inputs_types)
        return [XTCTensorType(shape=(d["T"], d["K"]), dtype=inputs_types[0].dtype, device=self.device)]

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[override]
        d = self.layer(inps_types)
        dims = {"i": d["T"], "j": d["K"], "k": d["K"], "h": d["H"]}
        up, down = ("chosen(i)", "h", "k"), ("chosen(i)", "j", "h")
        maps = (up, down) if len(inps_types) == 4 else (up, ("chosen(i)", "h", "block(k)"), down, ("chosen(i)", "j", "block(h)"))
        return self._operation(inps_types, outs_types, dims, ("P", "P", "R", "R"), (("i", "k"), ("chosen(i)", "k"), *maps), (("i", "j"),))

    def forward(self, inputs):  # type: ignore[override]
        d = self.layer([i.type for i in inputs])
        arrays = [i.numpy() for i in inputs]
        x, router = (a.astype(np.float64) for a in arrays[:2])
        if d["weights"] == "dense":
            up, down = (a.astype(np.float64) for a in arrays[2:])
        else:
            values = mx4_values if d["weights"] == "mx4" else fp8_values
            up, down = values(*arrays[2:4], d["K"], np.float64), values(*arrays[4:6], d["H"], np.float64)
        y = np.zeros(x.shape)
        with np.errstate(invalid="ignore", over="ignore"):
            logits = np.dot(x, router.T)
            for t, row in enumerate(logits):
                if np.isnan(row).any():
                    y[t] = np.nan
                    continue
                # ties to the lowest expert; two sums of one value may differ in their last bits
                chosen = np.argsort(-row.astype(np.float32), kind="stable")[: d["top_k"]]
                p = np.exp(row - row.max())
                p = p / (p[chosen].sum() if d["normalize"] else p.sum())
                for e in chosen:
                    u = np.dot(up[e], x[t])
                    if d["activation"] == "swiglu":
                        u = u[: d["H"]] / (1 + np.exp(-u[: d["H"]])) * u[d["H"]:]
                    else:
                        u = np.where(u < 0, 0, u)
                    h = p[e] * u
                    y[t] += np.dot(down[e], round_to_bf16(h.astype(np.float32)) if is_bf16(d["hidden"]) else h)
        return [self._check(XTCTensor(y, dtype=inputs[0].type.dtype), inputs)]
