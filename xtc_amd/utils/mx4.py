# SPDX-License-Identifier: BSD-3-Clause
"""Microscaled 4-bit floats in numpy (the OCP MX format of E2M1 elements with
E8M0 scales).

Every 32 consecutive elements of a row share a power-of-two scale, stored as
its exponent plus 127; 255 marks a block that holds an infinity or a NaN and
stands for NaN as a whole.  The last block of a row is filled up with zeros.
Two codes share a byte, the even element in the low half: a sign bit above the
index of 0, .5, 1, 1.5, 2, 3, 4, 6.
"""

from __future__ import annotations

import numpy as np

__all__ = ["BLOCK", "blocks_of", "mx4_scales", "mx4_codes", "mx4_values"]

BLOCK = 32
_VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float32)
# midpoints of neighbouring values; a tie goes to the even index
_MIDS = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))


def blocks_of(size: int) -> int:
    """Blocks of a row of `size` elements."""
    return -(-size // BLOCK)


def _blocks(x: np.ndarray) -> np.ndarray:
    a = np.asarray(x, dtype=np.float32)
    out = np.zeros((*a.shape[:-1], blocks_of(a.shape[-1]) * BLOCK), np.float32)
    out[..., : a.shape[-1]] = a
    return out.reshape(*a.shape[:-1], -1, BLOCK)


def mx4_scales(x: np.ndarray) -> np.ndarray:
    """(..., K) -> (..., ceil(K / 32)) uint8."""
    exponent = (_blocks(x).view(np.uint32) >> 23) & 255
    top = exponent.max(axis=-1).astype(np.int32)
    return np.where(top == 255, 255, np.maximum(top - 2, 0)).astype(np.uint8)


def mx4_codes(x: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """(..., K) and its scales -> (..., 16 ceil(K / 32)) uint8.  Codes are 0 where
    the scale is 255; elsewhere a NaN gives a zero of its sign."""
    v = _blocks(x)
    s = np.asarray(scales).astype(np.int32)[..., None]
    # exact in double precision: 24-bit elements times a power of two
    with np.errstate(invalid="ignore"):
        y = np.abs(v.astype(np.float64)) * np.ldexp(1.0, 127 - s)
        code = np.zeros(v.shape, np.uint8)
        for mid, up in _MIDS:
            code += (y >= mid) if up else (y > mid)
    code |= np.signbit(v).astype(np.uint8) << 3
    code[np.broadcast_to(s == 255, code.shape)] = 0
    code = code.reshape(*v.shape[:-2], -1, 2)
    return code[..., 0] | (code[..., 1] << 4)


def mx4_values(codes: np.ndarray, scales: np.ndarray, size: int | None = None, dtype: object = np.float32) -> np.ndarray:
    """(..., 16 B) codes and (..., B) scales -> (..., size or 32 B) of `dtype`
    (float64 holds all of them; the largest pass float32's range)."""
    c = np.asarray(codes)
    nib = np.stack((c & 15, c >> 4), axis=-1).reshape(*c.shape[:-1], -1, BLOCK)
    v = np.where(nib & 8, -_VALUES[nib & 7], _VALUES[nib & 7])
    s = np.asarray(scales).astype(np.int32)[..., None]
    scale = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127))
    with np.errstate(over="ignore"):
        out = (v * scale).astype(dtype).reshape(*c.shape[:-1], -1)
    return out if size is None else out[..., :size]
