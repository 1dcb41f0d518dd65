# SPDX-License-Identifier: BSD-3-Clause
"""Calls of the layer norm, 8-bit and expert layer entry points on numpy arrays, the
plain float64 forms that their results are compared with, and how far off those may
be."""

from __future__ import annotations

import ctypes

import numpy as np

from expert_calls import IDS, Mem, padded
from xtc_amd.runtimes.hip import capi

U = 2.0**-24  # half a unit of fp32
HALF = {"float32": 2.0**-24, "bfloat16": 2.0**-8}  # half a step of a result


def finish(mems, outs, stream=None):
    capi.check(capi.lib().xtc_hip_stream_synchronize(stream))
    got = [o.numpy() if o else None for o in outs]
    for m in (*mems, *outs):
        if m:
            m.free()
    return got


# ------------------------------------------------------------------ layer norm


def norm_parts(x, eps):
    """mean, centred x and 1 / deviation in float64."""
    x = x.astype(np.float64)
    m = x.mean(1, keepdims=True)
    c = x - m
    return m, c, 1 / np.sqrt((c * c).mean(1, keepdims=True) + np.float64(np.float32(eps)))


def norm_adds(K):
    """Additions one after another in a sum over a row: of a thread's elements, six
    lane exchanges, at most 16 waves; rows past 16384 a thread walks 1024 apart."""
    return max(16, -(-K // 1024) + 8) + 6 + 16


def layer_norm(x, w, b, dtype, params, eps=1e-5, pad=(0, 0), shift=(0, 0), stream=None):
    """pad, shift: of x and y, in elements."""
    rows, K = x.shape
    d = capi.LayerNormDesc(dtype=IDS[dtype], param_dtype=IDS[params], rows=rows, K=K, ldx=K + pad[0], ldy=K + pad[1], eps=eps,
                           stream=stream)
    mx = Mem(padded(x, K + pad[0]), dtype, shift[0])
    mw, mb = (Mem(v, params) if v is not None else None for v in (w, b))
    out = Mem(padded(np.full((rows, K), 7.0), K + pad[1]), dtype, shift[1])
    capi.check(capi.lib().xtc_hip_layer_norm(ctypes.byref(d), mx.ptr, mw and mw.ptr, mb and mb.ptr, out.ptr))
    (y,) = finish([mx, mw, mb], [out], stream)
    assert np.isnan(y[:, K:]).all(), "written past the columns"
    return y[:, :K]


def plain_norm(x, w, b, eps):
    """y and what fp32 arithmetic may be off by: the mean by its additions, 1 /
    deviation by half of those of the variance and a few roundings, then a product
    with w and the sum with b."""
    m, c, r = norm_parts(x, eps)
    w, b = (1.0 if w is None else w.astype(np.float64)), (0.0 if b is None else b.astype(np.float64))
    y = c * r * w + b
    mean = np.abs(x).astype(np.float64).mean(1, keepdims=True)
    off = (2 * norm_adds(x.shape[1]) + 16) * U * (np.abs(w) * r * (mean + np.abs(c)) + np.abs(b) + np.abs(y))
    return y, off


def layer_norm_grad(x, w, dy, dtype, params, eps=1e-5, want=(True, True, True), pad=(0, 0), stream=None):
    """(dx, dw, db), None where not wanted; pad: of x and dx, and of dy."""
    rows, K = x.shape
    d = capi.LayerNormDesc(dtype=IDS[dtype], param_dtype=IDS[params], rows=rows, K=K, ldx=K + pad[0], ldy=K + pad[1], eps=eps,
                           stream=stream)
    mems = [Mem(padded(x, K + pad[0]), dtype), Mem(w, params) if w is not None else None, Mem(padded(dy, K + pad[1]), dtype)]
    outs = [Mem(padded(np.full((rows, K), 7.0), K + pad[0]), dtype) if want[0] else None,
            *(Mem(np.full(K, 7.0), "float32") if v else None for v in want[1:])]
    ws = Mem(np.full(2 * min(rows, 512) * K + 2 * rows, np.nan), "float32") if any(want[1:]) else None
    args = [m and m.ptr for m in (*mems, *outs, ws)]
    capi.check(capi.lib().xtc_hip_layer_norm_grad(ctypes.byref(d), *args))
    got = finish([*mems, ws], outs, stream)
    if want[0]:
        assert np.isnan(got[0][:, K:]).all(), "written past the columns"
        got[0] = got[0][:, :K]
    return got


def plain_norm_grad(x, w, dy, eps):
    """(dx, dw, db) and what each may be off by, as in plain_norm."""
    (rows, K), n = x.shape, norm_adds(x.shape[1])
    m, c, r = norm_parts(x, eps)
    xh, dy = c * r, dy.astype(np.float64)
    g = dy * (1.0 if w is None else w.astype(np.float64))
    c1, c2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    dx = r * (g - c1 - xh * c2)
    mean, ga = np.abs(x).astype(np.float64).mean(1, keepdims=True), np.abs(g).mean(1, keepdims=True)
    f = (4 * n + 16) * U
    off_xh = r * mean + np.abs(xh)
    off_c2 = r * (np.abs(g * c).mean(1, keepdims=True) + mean * ga)
    off_dx = f * r * (np.abs(g) + ga + np.abs(xh) * off_c2 + off_xh * np.abs(c2))
    # a workgroup's rows, those side by side, then at most 512 parts by four waves
    adds = -(-rows // 512) + 4 + 128 + 4
    off_dw = (adds * U + f) * (np.abs(dy) * off_xh).sum(0)
    return (dx, (dy * xh).sum(0), dy.sum(0)), (off_dx, off_dw, adds * U * np.abs(dy).sum(0))


def check_close(got, want, off, dtype):
    over = np.abs(got - want) - (off + HALF[dtype] * np.abs(want))
    assert got.shape == want.shape and np.all(over <= 0), (np.unravel_index(np.nanargmax(over), over.shape), np.nanmax(over))


# ---------------------------------------------------------------------- 8-bit


def _fp8_desc(dtype, shape, rows, transpose=0, pad=0, stream=None):
    e, r, k = shape
    return capi.Fp8Desc(dtype=IDS[dtype], matrices=e, rows=r, K=k, ld=k + pad, block_rows=rows, transpose=int(transpose), stream=stream)


def _fp8_shapes(shape, rows, transpose):
    e, r, k = shape
    if transpose:
        r, k = k, r
    nb = -(-k // 128)
    return (e, r, 128 * nb), (e, -(-r // rows), nb)


def fp8_quantize(x, dtype, rows=1, transpose=False, values=True, pad=0, shift=0, stream=None):
    """x (E, R, K) -> codes, scales and values (None where transposed)."""
    cs, ss = _fp8_shapes(x.shape, rows, transpose)
    d = _fp8_desc(dtype, x.shape, rows, transpose, pad, stream)
    src = Mem(padded(x, x.shape[2] + pad), dtype, shift)
    outs = [Mem(np.zeros(cs), "uint8"), Mem(np.zeros(ss), "uint8"), Mem(np.zeros(x.shape), dtype) if values and not transpose else None]
    capi.check(capi.lib().xtc_hip_fp8_quantize(ctypes.byref(d), src.ptr, *[o and o.ptr for o in outs]))
    return finish([src], outs, stream)


def fp8_quantize_both(x, dtype, rows=1):
    """Codes and scales of x (E, R, K) and of its transpose."""
    d = _fp8_desc(dtype, x.shape, rows)
    src = Mem(x, dtype)
    outs = [Mem(np.zeros(s), "uint8") for t in (False, True) for s in _fp8_shapes(x.shape, rows, t)]
    capi.check(capi.lib().xtc_hip_fp8_quantize_both(ctypes.byref(d), src.ptr, *[o.ptr for o in outs]))
    return finish([src], outs)


def fp8_encode(x, scales, dtype, rows=1, transpose=False):
    cs, _ = _fp8_shapes(x.shape, rows, transpose)
    d = _fp8_desc(dtype, x.shape, rows, transpose)
    mems = [Mem(x, dtype), Mem(scales, "uint8")]
    out = Mem(np.zeros(cs), "uint8")
    capi.check(capi.lib().xtc_hip_fp8_encode(ctypes.byref(d), *[m.ptr for m in mems], out.ptr))
    return finish(mems, [out])[0]


def fp8_dequantize(codes, scales, size, dtype, pad=0):
    e, r, _ = codes.shape
    d = _fp8_desc(dtype, (e, r, size), 1 if scales.shape[1] == r else 128, 0, pad)
    mems = [Mem(codes, "uint8"), Mem(scales, "uint8")]
    out = Mem(np.full((e, r, size + pad), np.nan, np.float32), dtype)
    capi.check(capi.lib().xtc_hip_fp8_dequantize(ctypes.byref(d), *[m.ptr for m in mems], out.ptr))
    got = finish(mems, [out])[0]
    assert np.isnan(got[..., size:]).all(), "written past the columns"
    return got[..., :size]


def fp8_matmul(ac, asc, bc, bsc, out_dtype="float32", pad=0, shift=0, stream=None):
    (M, nb), N = asc.shape, bc.shape[0]
    d = capi.Fp8MatmulDesc(out_dtype=IDS[out_dtype], M=M, N=N, blocks=nb, b_block_rows=1 if len(bsc) == N else 128, ldc=N + pad,
                           stream=stream)
    # scales start off every boundary, one byte past one
    mems = [Mem(ac, "uint8"), Mem(asc, "uint8", 1), Mem(bc, "uint8"), Mem(bsc, "uint8", 1)]
    out = Mem(padded(np.full((M, N), 7.0), N + pad), out_dtype, shift)
    capi.check(capi.lib().xtc_hip_fp8_matmul(ctypes.byref(d), *[m.ptr for m in mems], out.ptr))
    (got,) = finish(mems, [out], stream)
    assert np.isnan(got[:, N:]).all(), "written past the columns"
    return got[:, :N]


# --------------------------------------------------------------- expert layer


def layer_desc(x, router, h, top_k, dtype, weights="dense", activation="swiglu", normalize=True, pad=(0, 0), stream=None):
    (T, K), E = x.shape, router.shape[0]
    return capi.ExpertLayerDesc(dtype=IDS[dtype], weights=("dense", "fp8", "mx4").index(weights),
                                activation=("relu", "swiglu").index(activation), T=T, E=E, K=K, H=h, top_k=top_k,
                                normalize=int(normalize), ldx=K + pad[0], ldy=K + pad[1], stream=stream)


def expert_layer(x, router, up, down, top_k, dtype, weights="dense", activation="swiglu", normalize=True, pad=(0, 0), shift=0,
                 stream=None):
    """up, down: arrays, or (codes, scales) of 8-bit or 4-bit matrices."""
    T, K = x.shape
    ups, downs = ((up, None), (down, None)) if weights == "dense" else (up, down)
    h = ups[0].shape[1] // (2 if activation == "swiglu" else 1)
    d = layer_desc(x, router, h, top_k, dtype, weights, activation, normalize, pad, stream)
    need = capi.lib().xtc_hip_expert_layer_workspace(ctypes.byref(d))
    assert need > 0 or T == 0, capi.last_error()
    kind = dtype if weights == "dense" else "uint8"
    mems = [Mem(padded(x, K + pad[0]), dtype, shift), Mem(router, dtype),
            *(m for c, s in (ups, downs) for m in (Mem(c, kind, shift if weights == "dense" else 0), Mem(s, "uint8", 1) if s is not None else None))]
    ws = Mem(np.full(need, 0xFF), "uint8")
    out = Mem(padded(np.full((T, K), 7.0), K + pad[1]), dtype)
    capi.check(capi.lib().xtc_hip_expert_layer(ctypes.byref(d), *[m and m.ptr for m in mems], ws.ptr, need, out.ptr))
    ws.numpy()  # nothing around it was written
    (y,) = finish([*mems, ws], [out], stream)
    assert np.isnan(y[:, K:]).all(), "written past the columns"
    return y[:, :K]


def logits_of(x, router):
    """Logits in float64, and twice what K additions in fp32 may be off by, at most."""
    x, router = x.astype(np.float64), router.astype(np.float64)
    return x @ router.T, (x.shape[1] + 16) * 2 * U * (np.abs(x) @ np.abs(router).T)


def unclear(x, router, top_k):
    """Tokens whose choice rounding could change."""
    logits, off = logits_of(x, router)
    if top_k >= len(router):
        return np.zeros(len(x), bool)
    order = np.sort(logits, axis=1)[:, ::-1]
    gap = order[:, top_k - 1] - order[:, top_k]
    return (gap <= 2 * off.max(1)) & (gap != 0)


def plain_layer(x, router, up, down, top_k, activation="swiglu", normalize=True, mid=0.0):
    """y in float64 and what fp32 sums of K and H products may be off by: additions of
    the logits (which the weights follow), of up, of down, the activation's few
    roundings and `mid`, what the down product's operand is rounded by.  Inputs whose
    choice that could change are refused."""
    assert not unclear(x, router, top_k).any(), "a choice that rounding could change"
    logits, off_l = logits_of(x, router)
    x = x.astype(np.float64)
    (T, K), h = x.shape, down.shape[2]
    y, off = np.zeros((T, K)), np.zeros((T, K))
    for t, row in enumerate(logits):
        order = np.argsort(-row, kind="stable")
        top = off_l[t].max()
        order = order[:top_k]
        p = np.exp(row - row.max())
        p = p / (p[order].sum() if normalize else p.sum())
        off_p = 4 * top + (len(row) + 32) * U
        for e in order:
            u, off_u = up[e] @ x[t], (K + 16) * 2 * U * (np.abs(up[e]) @ np.abs(x[t]))
            if activation == "swiglu":
                g, v = u[:h], u[h:]
                s = g / (1 + np.exp(-g))
                a, off_a = s * v, 1.1 * off_u[:h] * (np.abs(v) + off_u[h:]) + np.abs(s) * off_u[h:] + 16 * U * np.abs(s * v)
            else:
                a, off_a = np.maximum(u, 0), off_u
            z, d = down[e] @ a, np.abs(down[e])
            y[t] += p[e] * z
            off[t] += p[e] * (d @ (off_a + (mid + (h + 16) * 2 * U) * np.abs(a)) + (off_p + 4 * U) * (d @ np.abs(a)))
    return y, off + (top_k + 2) * U * np.abs(y)
