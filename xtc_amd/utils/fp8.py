# SPDX-License-Identifier: BSD-3-Clause
"""8-bit floats (E4M3) with E8M0 scales in numpy.

Every 128 consecutive elements of a row, or every block of 128 x 128, share a
power-of-two scale, stored as its exponent plus 127: the smallest with max|x| <=
448 scale, from 2^-127 on; 255 marks a block that holds an infinity or a NaN and
stands for NaN as a whole.  The last block of a row is filled up with zeros.  A
code is a sign, 4 exponent bits (bias 7, 0 subnormal) and 3 mantissa bits; 0x7f
is NaN, there is no infinity.
"""

from __future__ import annotations

import numpy as np

__all__ = ["BLOCK", "blocks_of", "fp8_scales", "fp8_codes", "fp8_values"]

BLOCK = 128
MOST = 448.0
_VALUES = np.array([i * 2.0**-9 for i in range(8)] + [(8 + i) * 2.0 ** (e - 10) for e in range(1, 16) for i in range(8)])
_VALUES[127] = np.nan


def blocks_of(size: int) -> int:
    """Blocks of a row of `size` elements."""
    return -(-size // BLOCK)


def _blocks(x: np.ndarray, rows: int) -> np.ndarray:
    """(..., R, K) to (..., R / rows, rows, K / 128, 128), filled up with zeros."""
    a = np.asarray(x, dtype=np.float32)
    r, k = a.shape[-2:]
    rb = -(-r // rows)
    out = np.zeros((*a.shape[:-2], rb * rows, blocks_of(k) * BLOCK), np.float32)
    out[..., :r, :k] = a
    return out.reshape(*a.shape[:-2], rb, rows, blocks_of(k), BLOCK)


def fp8_scales(x: np.ndarray, rows: int = 1) -> np.ndarray:
    """(..., R, K) -> (..., ceil(R / rows), ceil(K / 128)) uint8."""
    top = (_blocks(x, rows).view(np.uint32) & 0x7FFFFFFF).max(axis=(-3, -1)).astype(np.int64)
    e = top >> 23
    s = np.maximum(e - 8 + ((top & 0x7FFFFF) > 0x600000), 0)
    return np.where(e == 255, 255, s).astype(np.uint8)


def fp8_codes(x: np.ndarray, scales: np.ndarray, rows: int = 1) -> np.ndarray:
    """(..., R, K) and its scales -> (..., R, 128 ceil(K / 128)) uint8.  0 where the
    scale is 255; elsewhere 448 of its sign for what passes 448 scale, infinities
    among it, and the NaN code of its sign for a NaN."""
    v = _blocks(x, rows)
    s = np.asarray(scales).astype(np.int32)[..., :, None, :, None]
    with np.errstate(invalid="ignore"):
        # exact in double precision: 24-bit elements times a power of two
        y = np.minimum(np.abs(v.astype(np.float64)) * np.ldexp(1.0, 127 - s), MOST)
        nan = np.isnan(y)
        y = np.where(nan, 0, y)
        # the exponent, that of subnormals at least
        low = np.where(y < 2.0**-6, -6, np.frexp(y)[1] - 1)
        code = np.rint(np.ldexp(y, 3 - low)).astype(np.int64) + 8 * (low + 6)
    code = np.where(nan, 127, code) | (np.signbit(v).astype(np.int64) << 7)
    code = np.where(s == 255, 0, code).astype(np.uint8)
    code = code.reshape(*v.shape[:-4], v.shape[-4] * rows, v.shape[-2] * BLOCK)
    return np.ascontiguousarray(code[..., : np.shape(x)[-2], :])


def fp8_values(codes: np.ndarray, scales: np.ndarray, size: int | None = None, dtype: object = np.float32) -> np.ndarray:
    """(..., R, 128 B) codes and (..., R or ceil(R / 128), B) scales -> (..., R, size or
    128 B) of `dtype` (float64 holds all of them)."""
    c = np.asarray(codes)
    v = _VALUES[c & 127]
    v = np.where(c & 128, -v, v)
    s = np.asarray(scales).astype(np.int32)
    scale = np.where(s == 255, np.nan, np.ldexp(1.0, s - 127)).repeat(BLOCK, axis=-1)
    if s.shape[-2] != c.shape[-2]:
        scale = scale.repeat(BLOCK, axis=-2)[..., : c.shape[-2], :]
    with np.errstate(over="ignore"):
        out = (v * scale).astype(dtype)
    return out if size is None else out[..., :size]
