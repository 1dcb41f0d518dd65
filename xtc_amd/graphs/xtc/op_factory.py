# SPDX-License-Identifier: BSD-3-Clause
"""DSL functions: `O.tensor`, `O.matmul`, ... (src/xtc/graphs/xtc/op_factory.py:22-112)."""

from __future__ import annotations

from typing import Any

from .context import XTCGraphContext
from .data import XTCTensorType
from .expr import OP_EXPRS, XTCExpr, XTCTensorExpr

__all__ = [
    "matmul",
    "conv2d",
    "pad2d",
    "unpad",
    "pad",
    "relu",
    "reshape",
    "transpose",
    "bias_add",
    "grouped_matmul",
    "grouped_matmul_grad_w",
    "mx4_scales",
    "mx4_codes",
    "mx4_quantize",
    "mx4_dequantize",
    "mx4_matmul",
    "grouped_mx4_matmul",
    "layer_norm",
    "layer_norm_grad_x",
    "layer_norm_grad_weight",
    "layer_norm_grad_bias",
    "layer_norm_grad",
    "fp8_scales",
    "fp8_codes",
    "fp8_quantize",
    "fp8_dequantize",
    "fp8_matmul",
    "expert_layer",
    "tensor",
    "inputs",
    "outputs",
    "type",
]


def _append(op: str, *args: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return XTCGraphContext.append(OP_EXPRS[op](*args, **attrs), name=name)


def matmul(a: XTCExpr, b: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("matmul", a, b, name=name, **attrs)


def conv2d(inp: XTCExpr, weight: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("conv2d", inp, weight, name=name, **attrs)


def pad2d(inp: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("pad2d", inp, name=name, **attrs)


def unpad(inp: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("unpad", inp, name=name, **attrs)


def pad(inp: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("pad", inp, name=name, **attrs)


def relu(inp: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("relu", inp, name=name, **attrs)


def reshape(inp: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("reshape", inp, name=name, **attrs)


def transpose(inp: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    return _append("transpose", inp, name=name, **attrs)


def bias_add(inp: XTCExpr, bias: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: adds a per-last-axis bias (fused into the producing GEMM)."""
    return _append("bias_add", inp, bias, name=name, **attrs)


def grouped_matmul(x: XTCExpr, w: XTCExpr, sizes: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: rows of x (T, K), sorted by group, times their group's matrix
    of w (E, K, N); sizes (E,) int32 rows a group.  Attribute out_dtype.  With
    the stored forward w as layout [0, 2, 1]: the gradient of x."""
    return _append("grouped_matmul", x, w, sizes, name=name, **attrs)


def grouped_matmul_grad_w(x: XTCExpr, dy: XTCExpr, sizes: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: the gradient of grouped_matmul's w, (E, K, N), from x (T, K)
    and dy (T, N).  Attribute out_dtype."""
    return _append("grouped_matmul_grad_w", x, dy, sizes, name=name, **attrs)


def mx4_scales(x: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: scales of x's blocks of 32 as microscaled 4-bit floats."""
    return _append("mx4_scales", x, name=name, **attrs)


def mx4_codes(x: XTCExpr, scales: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: codes of x as microscaled 4-bit floats of the given scales."""
    return _append("mx4_codes", x, scales, name=name, **attrs)


def mx4_quantize(x: XTCExpr) -> tuple[XTCExpr, XTCExpr]:
    """Extension: x as microscaled 4-bit floats, (codes, scales): the nodes
    mx4_scales and mx4_codes, which run as one launch."""
    scales = mx4_scales(x)
    return mx4_codes(x, scales), scales


def mx4_dequantize(codes: XTCExpr, scales: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: values of microscaled 4-bit floats.  Attributes size (of a
    row, 32 a block by default) and out_dtype (float32)."""
    return _append("mx4_dequantize", codes, scales, name=name, **attrs)


def mx4_matmul(a_codes: XTCExpr, a_scales: XTCExpr, b_codes: XTCExpr, b_scales: XTCExpr, name: str | None = None,
               **attrs: Any) -> XTCExpr:
    """Extension: a (M, K) times b (N, K) transposed, both microscaled 4-bit
    floats.  Attribute out_dtype (float32)."""
    return _append("mx4_matmul", a_codes, a_scales, b_codes, b_scales, name=name, **attrs)


def grouped_mx4_matmul(a_codes: XTCExpr, a_scales: XTCExpr, b_codes: XTCExpr, b_scales: XTCExpr, sizes: XTCExpr,
                       name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: mx4_matmul by group: rows of a sorted by group, b (E, N, K),
    sizes as in grouped_matmul.  Attribute out_dtype (float32)."""
    return _append("grouped_mx4_matmul", a_codes, a_scales, b_codes, b_scales, sizes, name=name, **attrs)


def layer_norm(x: XTCExpr, weight: XTCExpr, bias: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: layer norm of x (..., K) along its last axis, weight and bias (K,).
    Attribute eps (1e-5)."""
    return _append("layer_norm", x, weight, bias, name=name, **attrs)


def layer_norm_grad_x(x: XTCExpr, weight: XTCExpr, dy: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: the gradient of layer_norm's x.  Attribute eps (1e-5)."""
    return _append("layer_norm_grad_x", x, weight, dy, name=name, **attrs)


def layer_norm_grad_weight(x: XTCExpr, dy: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: the gradient of layer_norm's weight, float32.  Attribute eps (1e-5)."""
    return _append("layer_norm_grad_weight", x, dy, name=name, **attrs)


def layer_norm_grad_bias(dy: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: the gradient of layer_norm's bias, float32."""
    return _append("layer_norm_grad_bias", dy, name=name, **attrs)


def layer_norm_grad(x: XTCExpr, weight: XTCExpr, dy: XTCExpr, **attrs: Any) -> tuple[XTCExpr, XTCExpr, XTCExpr]:
    """Extension: the gradients of layer_norm's x, weight and bias: the three nodes
    above, which run as one call.  Attribute eps (1e-5)."""
    return (layer_norm_grad_x(x, weight, dy, **attrs), layer_norm_grad_weight(x, dy, **attrs), layer_norm_grad_bias(dy))


def fp8_scales(x: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: scales of x (..., R, K) as 8-bit floats: of every 128 elements of a
    row (attribute rows 1) or every 128 x 128 (rows 128); with transpose those of
    the transposed matrices."""
    return _append("fp8_scales", x, name=name, **attrs)


def fp8_codes(x: XTCExpr, scales: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: codes of x as 8-bit floats of the given scales.  Attributes as in
    fp8_scales."""
    return _append("fp8_codes", x, scales, name=name, **attrs)


def fp8_quantize(x: XTCExpr, **attrs: Any) -> tuple[XTCExpr, XTCExpr]:
    """Extension: x as 8-bit floats, (codes, scales): the nodes fp8_scales and
    fp8_codes, which run as one launch, with those of the transposed x where the
    graph asks for both."""
    scales = fp8_scales(x, **attrs)
    return fp8_codes(x, scales, **attrs), scales


def fp8_dequantize(codes: XTCExpr, scales: XTCExpr, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: values of 8-bit floats.  Attributes size (of a row, 128 a block by
    default) and out_dtype (float32)."""
    return _append("fp8_dequantize", codes, scales, name=name, **attrs)


def fp8_matmul(a_codes: XTCExpr, a_scales: XTCExpr, b_codes: XTCExpr, b_scales: XTCExpr, name: str | None = None,
               **attrs: Any) -> XTCExpr:
    """Extension: a (M, K) times b (N, K) transposed, both 8-bit floats, a with a scale
    for every 128 elements of a row, b that or one for every 128 x 128.  The
    gradients are products of the same kind: dx = dy w and dw = dy^T x, of operands
    quantised along what is summed over (transpose).  Attributes out_dtype (float32) and
    sums ("fp32"; "fp8": those of the 8-bit matrix instructions, faster and less exact)."""
    return _append("fp8_matmul", a_codes, a_scales, b_codes, b_scales, name=name, **attrs)


def expert_layer(x: XTCExpr, router: XTCExpr, up: Any, down: Any, name: str | None = None, **attrs: Any) -> XTCExpr:
    """Extension: a whole layer of experts for at most 64 tokens: x (T, K), router (E, K),
    up (E, H or 2 H, K) and down (E, K, H) of x's type or each a pair (codes, scales) of
    8-bit floats in blocks of 128 x 128 or of microscaled 4-bit floats.  Attributes
    top_k (2), activation ("swiglu": up's first H rows are the gate; or "relu"),
    normalize (True: the chosen experts' weights sum to 1), hidden_dtype (float32: the
    activations between up and down keep it; bfloat16 for bfloat16 x: they are rounded)."""
    matrices = [m for w in (up, down) for m in (w if isinstance(w, (tuple, list)) else (w,))]
    return _append("expert_layer", x, router, *matrices, name=name, **attrs)


def tensor(*args: Any, name: str | None = None, **attrs: Any) -> XTCExpr:
    return XTCGraphContext.append(XTCTensorExpr(*args, **attrs), name=name)


def inputs(*inps: XTCExpr) -> None:
    XTCGraphContext.inputs(*inps)


def outputs(*outs: XTCExpr) -> None:
    XTCGraphContext.outputs(*outs)


def type(*args: Any, **attrs: Any) -> XTCTensorType:  # noqa: A001 - mirrors the DSL name
    return XTCTensorType(*args, **attrs)
