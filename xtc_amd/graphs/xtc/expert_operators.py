# SPDX-License-Identifier: BSD-3-Clause
"""Operators of layers of experts and of 4-bit operands, with their numpy
semantics (extensions: the reference's operators, src/xtc/graphs/xtc/
operators.py:159-804, have neither).

grouped_matmul, grouped_matmul_grad_w: products by group of rows.  `sizes`
(int32, one per group) says how many rows each group has; the groups follow one
another from row 0, sizes below zero count as zero, rows past the last group
belong to nobody and rows past the end do not exist.

mx4_scales, mx4_codes, mx4_dequantize, mx4_matmul, grouped_mx4_matmul:
microscaled 4-bit floats (xtc_amd.utils.mx4) as two uint8 tensors, codes and
scales.
"""

from __future__ import annotations

from typing import Any

import numpy as np

from ...utils.bf16 import is_bf16
from ...utils.mx4 import BLOCK, blocks_of, mx4_codes, mx4_scales, mx4_values
from .data import XTCTensor, XTCTensorType
from .operation import XTCOperation
from .operators import XTCOperator, _out_dtype

__all__ = [
    "XTCOperGroupedMatmul",
    "XTCOperGroupedMatmulGradW",
    "XTCOperMx4Scales",
    "XTCOperMx4Codes",
    "XTCOperMx4Dequantize",
    "XTCOperMx4Matmul",
    "XTCOperGroupedMx4Matmul",
    "group_bounds",
]


def group_bounds(sizes: np.ndarray, rows: int) -> list[tuple[int, int]]:
    """[begin, end) of every group's rows."""
    ends = np.minimum(np.cumsum(np.maximum(np.asarray(sizes).astype(np.int64), 0)), rows)
    return [(int(b), int(e)) for b, e in zip([0, *ends[:-1]], ends)]


def _float_operands(name: str, *types: Any) -> None:
    dtypes = {str(t.dtype) for t in types}
    if len(dtypes) != 1 or not dtypes <= {"float32", "bfloat16"}:
        raise ValueError(f"{name}: operands must both be float32 or bfloat16, got {sorted(dtypes)}")


def _float_result(name: str, in_dtype: Any, out_dtype: Any) -> str:
    if str(out_dtype) not in ("float32", "bfloat16") or (is_bf16(out_dtype) and str(in_dtype) == "float32"):
        raise ValueError(f"{name}: result dtype {out_dtype} for operands of dtype {in_dtype}")
    return str(out_dtype)


def _sizes_type(name: str, t: Any, groups: int) -> None:
    if str(t.dtype) != "int32" or t.constant_shape != (groups,):
        raise ValueError(f"{name}: sizes must be int32 of shape ({groups},), got {t}")


class XTCOperGroupedMatmul(XTCOperator):
    """y[r, :] = x[r, :] w[e] for the rows r of group e, zeros for rows of no group.

    x (T, K), w (E, K, N), sizes (E,) -> (T, N).  A w of layout [0, 2, 1] is
    stored (E, N, K), each matrix transposed.
    """

    def __init__(self, **attrs: Any) -> None:
        super().__init__("grouped_matmul", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        x, w, sizes = inputs_types
        _float_operands(self.name, x, w)
        if len(x.constant_shape) != 2 or len(w.constant_shape) != 3 or x.constant_shape[1] != w.constant_shape[1]:
            raise ValueError(f"{self.name} expects (T,K) and (E,K,N): {x.constant_shape} {w.constant_shape}")
        _sizes_type(self.name, sizes, w.constant_shape[0])
        out = _float_result(self.name, x.dtype, _out_dtype(self, x.dtype))
        return [XTCTensorType(shape=(x.constant_shape[0], w.constant_shape[2]), dtype=out, device=self.device)]

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[override]
        (t, k), n = inps_types[0].constant_shape, inps_types[1].constant_shape[2]
        return self._operation(inps_types, outs_types, {"i": t, "j": n, "k": k}, ("P", "P", "R"),
                               (("i", "k"), ("group(i)", "k", "j"), ("group(i)",)), (("i", "j"),))

    def forward(self, inputs):  # type: ignore[override]
        x, w, sizes = (i.numpy() for i in inputs)
        y = np.zeros((x.shape[0], w.shape[2]), np.float32)
        for e, (b, end) in enumerate(group_bounds(sizes, x.shape[0])):
            y[b:end] = np.dot(x[b:end], w[e])
        return [self._check(XTCTensor(y, dtype=self.forward_types([i.type for i in inputs])[0].dtype), inputs)]


class XTCOperGroupedMatmulGradW(XTCOperator):
    """dw[e] = x_e^T dy_e over the rows of group e, zeros where it has none.

    x (T, K), dy (T, N), sizes (E,) -> (E, K, N).
    """

    def __init__(self, **attrs: Any) -> None:
        super().__init__("grouped_matmul_grad_w", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        x, dy, sizes = inputs_types
        _float_operands(self.name, x, dy)
        if len(x.constant_shape) != 2 or len(dy.constant_shape) != 2 or x.constant_shape[0] != dy.constant_shape[0]:
            raise ValueError(f"{self.name} expects (T,K) and (T,N): {x.constant_shape} {dy.constant_shape}")
        if len(sizes.constant_shape) != 1:
            raise ValueError(f"{self.name}: sizes must be int32 of rank 1, got {sizes}")
        groups = sizes.constant_shape[0]
        _sizes_type(self.name, sizes, groups)
        out = _float_result(self.name, x.dtype, _out_dtype(self, x.dtype))
        shape = (groups, x.constant_shape[1], dy.constant_shape[1])
        return [XTCTensorType(shape=shape, dtype=out, device=self.device)]

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[override]
        (t, k), n = inps_types[0].constant_shape, inps_types[1].constant_shape[1]
        return self._operation(inps_types, outs_types, {"i": k, "j": n, "k": t}, ("P", "P", "R"),
                               (("k", "i"), ("k", "j"), ("group(k)",)), (("group(k)", "i", "j"),))

    def forward(self, inputs):  # type: ignore[override]
        x, dy, sizes = (i.numpy() for i in inputs)
        dw = np.zeros((sizes.shape[0], x.shape[1], dy.shape[1]), np.float32)
        for e, (b, end) in enumerate(group_bounds(sizes, x.shape[0])):
            dw[e] = np.dot(x[b:end].T, dy[b:end])
        return [self._check(XTCTensor(dw, dtype=self.forward_types([i.type for i in inputs])[0].dtype), inputs)]


class _Blocks:
    """Iteration space of the block-wise operators: rows and blocks of 32."""

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[no-untyped-def]
        shape = outs_types[0].constant_shape
        names = tuple(f"d{i}" for i in range(len(shape)))
        return self._operation(  # type: ignore[attr-defined]
            inps_types, outs_types, dict(zip(names, shape)), ("P",) * len(shape),
            tuple((*names[:-1], f"block({names[-1]})") for _ in inps_types), (names,))


def _mx4_source(name: str, t: Any) -> tuple[int, ...]:
    if str(t.dtype) not in ("float32", "bfloat16") or len(t.constant_shape) < 2:
        raise ValueError(f"{name} expects a float32 or bfloat16 tensor of rank >= 2, got {t}")
    return t.constant_shape  # type: ignore[no-any-return]


def _mx4_pair(name: str, codes: Any, scales: Any) -> tuple[int, ...]:
    """Shape of the scales of a pair of tensors."""
    c, s = codes.constant_shape, scales.constant_shape
    if str(codes.dtype) != "uint8" or str(scales.dtype) != "uint8" or len(c) < 2 or c != (*s[:-1], 16 * s[-1]):
        raise ValueError(f"{name}: codes (..., 16 B) and scales (..., B) must be uint8: {codes} {scales}")
    return s  # type: ignore[no-any-return]


class XTCOperMx4Scales(_Blocks, XTCOperator):
    """Scales of the blocks of x: (..., K) -> (..., ceil(K / 32)) uint8."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("mx4_scales", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        shape = _mx4_source(self.name, inputs_types[0])
        return [XTCTensorType(shape=(*shape[:-1], blocks_of(shape[-1])), dtype="uint8", device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        return [self._check(XTCTensor(mx4_scales(inputs[0].numpy()), dtype="uint8"), inputs)]


class XTCOperMx4Codes(_Blocks, XTCOperator):
    """Codes of x for given scales: (..., K), (..., ceil(K / 32)) -> (..., 16 ceil(K / 32)) uint8.
    0 where the scale is 255; elsewhere a NaN gives a zero of its sign."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("mx4_codes", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        shape = _mx4_source(self.name, inputs_types[0])
        scales = inputs_types[1]
        if str(scales.dtype) != "uint8" or scales.constant_shape != (*shape[:-1], blocks_of(shape[-1])):
            raise ValueError(f"{self.name}: scales {scales} do not match {inputs_types[0]}")
        return [XTCTensorType(shape=(*shape[:-1], 16 * blocks_of(shape[-1])), dtype="uint8", device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        return [self._check(XTCTensor(mx4_codes(inputs[0].numpy(), inputs[1].numpy()), dtype="uint8"), inputs)]


class XTCOperMx4Dequantize(_Blocks, XTCOperator):
    """Values of codes and scales: (..., 16 B), (..., B) -> (..., size), size
    defaulting to 32 B, of type out_dtype (float32)."""

    def __init__(self, **attrs: Any) -> None:
        super().__init__("mx4_dequantize", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        shape = _mx4_pair(self.name, *inputs_types)
        size = getattr(self.attrs, "size", None) or BLOCK * shape[-1]
        if blocks_of(size) != shape[-1]:
            raise ValueError(f"{self.name}: {shape[-1]} blocks do not hold rows of {size} elements")
        out = _float_result(self.name, "uint8", getattr(self.attrs, "out_dtype", None) or "float32")
        return [XTCTensorType(shape=(*shape[:-1], size), dtype=out, device=self.device)]

    def forward(self, inputs):  # type: ignore[override]
        t = self.forward_types([i.type for i in inputs])[0]
        values = mx4_values(inputs[0].numpy(), inputs[1].numpy(), t.constant_shape[-1])
        return [self._check(XTCTensor(values, dtype=t.dtype), inputs)]


class XTCOperMx4Matmul(XTCOperator):
    """c[i, j] = sum_k a[i, k] b[j, k] of microscaled operands.

    a codes (M, 16 B) and scales (M, B), b codes (N, 16 B) and scales (N, B)
    -> (M, N) of type out_dtype (float32).
    """

    def __init__(self, **attrs: Any) -> None:
        super().__init__("mx4_matmul", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        a = _mx4_pair(self.name, *inputs_types[:2])
        b = _mx4_pair(self.name, *inputs_types[2:4])
        if len(a) != 2 or len(b) != 2 or a[1] != b[1]:
            raise ValueError(f"{self.name} expects operands of one depth: scales {a} {b}")
        out = _float_result(self.name, "uint8", getattr(self.attrs, "out_dtype", None) or "float32")
        return [XTCTensorType(shape=(a[0], b[0]), dtype=out, device=self.device)]

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[override]
        m, n = outs_types[0].constant_shape
        k = BLOCK * inps_types[1].constant_shape[1]
        return self._operation(inps_types, outs_types, {"i": m, "j": n, "k": k}, ("P", "P", "R"),
                               (("i", "k"), ("i", "block(k)"), ("j", "k"), ("j", "block(k)")), (("i", "j"),))

    def forward(self, inputs):  # type: ignore[override]
        ac, asc, bc, bsc = (i.numpy() for i in inputs)
        out = self.forward_types([i.type for i in inputs])[0].dtype
        a, b = (mx4_values(c, s, dtype=np.float64) for c, s in ((ac, asc), (bc, bsc)))
        return [self._check(XTCTensor(np.dot(a, b.T), dtype=out), inputs)]


class XTCOperGroupedMx4Matmul(XTCOperator):
    """c[r, :] = a[r, :] b[e]^T for the rows r of group e, of microscaled operands.

    a codes (T, 16 B) and scales (T, B), b codes (E, N, 16 B) and scales
    (E, N, B), sizes (E,) -> (T, N) of type out_dtype (float32).
    """

    def __init__(self, **attrs: Any) -> None:
        super().__init__("grouped_mx4_matmul", **attrs)

    def forward_types(self, inputs_types):  # type: ignore[override]
        a = _mx4_pair(self.name, *inputs_types[:2])
        b = _mx4_pair(self.name, *inputs_types[2:4])
        if len(a) != 2 or len(b) != 3 or a[1] != b[2]:
            raise ValueError(f"{self.name} expects operands of one depth: scales {a} {b}")
        _sizes_type(self.name, inputs_types[4], b[0])
        out = _float_result(self.name, "uint8", getattr(self.attrs, "out_dtype", None) or "float32")
        return [XTCTensorType(shape=(a[0], b[1]), dtype=out, device=self.device)]

    def get_operation(self, inps_types, outs_types) -> XTCOperation:  # type: ignore[override]
        t, n = outs_types[0].constant_shape
        k = BLOCK * inps_types[1].constant_shape[1]
        return self._operation(
            inps_types, outs_types, {"i": t, "j": n, "k": k}, ("P", "P", "R"),
            (("i", "k"), ("i", "block(k)"), ("group(i)", "j", "k"), ("group(i)", "j", "block(k)"), ("group(i)",)),
            (("i", "j"),))

    def forward(self, inputs):  # type: ignore[override]
        ac, asc, bc, bsc, sizes = (i.numpy() for i in inputs)
        a, b = (mx4_values(c, s, dtype=np.float64) for c, s in ((ac, asc), (bc, bsc)))
        y = np.zeros((a.shape[0], b.shape[1]), np.float32)
        for e, (lo, hi) in enumerate(group_bounds(sizes, a.shape[0])):
            y[lo:hi] = np.dot(a[lo:hi], b[e].T)
        return [self._check(XTCTensor(y, dtype=self.forward_types([i.type for i in inputs])[0].dtype), inputs)]
