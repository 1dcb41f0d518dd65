# SPDX-License-Identifier: BSD-3-Clause
"""Calls of the expert and 4-bit entry points on numpy arrays, and the plain
float64 forms that their results are compared with."""

from __future__ import annotations

import ctypes

import numpy as np

from xtc_amd.runtimes.hip import capi
from xtc_amd.runtimes.hip.device import HipDevice
from xtc_amd.utils.bf16 import bf16_bits_to_f32, f32_to_bf16_bits, round_to_bf16

IDS = {"float32": capi.XTC_HIP_F32, "bfloat16": capi.XTC_HIP_BF16}
ESZ = {"float32": 4, "bfloat16": 2}


def bounds(sizes, rows):
    """[begin, end) of every group, in Python integers."""
    out, at = [], 0
    for s in sizes:
        end = min(rows, at + max(int(s), 0))
        out.append((at, end))
        at = end
    return out


def plain_grouped(x, w, sizes):
    y = np.zeros((x.shape[0], w.shape[2]))
    for e, (b, end) in enumerate(bounds(sizes, x.shape[0])):
        y[b:end] = x[b:end].astype(np.float64) @ w[e].astype(np.float64)
    return y


def plain_grad_w(x, dy, sizes):
    return np.stack([x[b:e].astype(np.float64).T @ dy[b:e].astype(np.float64) for b, e in bounds(sizes, x.shape[0])])


class Mem:
    """Device memory holding `array` as `dtype` words, `shift` elements past a
    256-byte boundary, `guard` untouched bytes of 0xff (NaN) on both sides."""

    GUARD = 4096

    def __init__(self, array, dtype, shift=0):
        self.dev = HipDevice()
        self.dev.init_device()
        self.dtype, self.shape = dtype, array.shape
        raw = f32_to_bf16_bits(array) if dtype == "bfloat16" else np.ascontiguousarray(array, dtype)
        self.nbytes = raw.nbytes
        self.total = 2 * self.GUARD + raw.nbytes + 512
        self.at = self.GUARD + shift * (2 if dtype == "bfloat16" else raw.itemsize)
        self.base = self.dev.memory_allocate(self.total)
        host = np.full(self.total, 0xFF, np.uint8)
        host[self.at : self.at + raw.nbytes] = raw.reshape(-1).view(np.uint8)
        self.dev.memory_copy_to(self.base, host.ctypes.data_as(ctypes.c_void_p), self.total)

    @property
    def ptr(self):
        return ctypes.c_void_p(self.base + self.at)

    def numpy(self):
        """The values, after checking that nothing around them was written."""
        host = np.empty(self.total, np.uint8)
        self.dev.memory_copy_from(self.base, host.ctypes.data_as(ctypes.c_void_p), self.total)
        assert (host[: self.at] == 0xFF).all() and (host[self.at + self.nbytes :] == 0xFF).all(), "written outside"
        raw = host[self.at : self.at + self.nbytes]
        if self.dtype == "bfloat16":
            return bf16_bits_to_f32(raw.view(np.uint16)).reshape(self.shape)
        return raw.view(self.dtype).reshape(self.shape)

    def free(self):
        self.dev.memory_free(self.base)


def padded(a, ld):
    """Rows of `ld` elements, the added ones NaN."""
    out = np.full((*a.shape[:-1], ld), np.nan, np.float32)
    out[..., : a.shape[-1]] = a
    return out


def _call(fn, desc, mems, out, stream):
    desc.stream = stream
    capi.check(fn(ctypes.byref(desc), *[m.ptr for m in mems], out.ptr))
    capi.check(capi.lib().xtc_hip_stream_synchronize(stream))
    got = out.numpy()
    for m in (*mems, out):
        m.free()
    return got


def grouped(x, w, sizes, dtype, out_dtype=None, trans_w=False, pad=(0, 0, 0), shift=(0, 0, 0), stream=None):
    """pad, shift: of x, w and y, in elements."""
    out_dtype = out_dtype or dtype
    T, K = x.shape
    E, _, N = w.shape
    ws = w.swapaxes(1, 2) if trans_w else w
    ldx, ldw, ldy = K + pad[0], ws.shape[2] + pad[1], N + pad[2]
    d = capi.GroupedMatmulDesc(dtype=IDS[dtype], out_dtype=IDS[out_dtype], E=E, T=T, N=N, K=K, ldx=ldx, ldw=ldw, ldy=ldy,
                               trans_w=int(trans_w))
    mems = [Mem(padded(x, ldx), dtype, shift[0]), Mem(padded(ws, ldw), dtype, shift[1]), Mem(np.asarray(sizes), "int32")]
    y = _call(capi.lib().xtc_hip_grouped_matmul, d, mems, Mem(padded(np.full((T, N), 7.0), ldy), out_dtype, shift[2]), stream)
    assert np.isnan(y[:, N:]).all(), "written past the columns"
    return y[:, :N]


def grad_w(x, dy, sizes, dtype, out_dtype=None, pad=(0, 0, 0), shift=(0, 0, 0), stream=None):
    """pad, shift: of x, dy and dw, in elements."""
    out_dtype = out_dtype or dtype
    (T, K), N, E = x.shape, dy.shape[1], len(sizes)
    ldx, ldy, ldw = K + pad[0], N + pad[1], N + pad[2]
    d = capi.GroupedMatmulDesc(dtype=IDS[dtype], out_dtype=IDS[out_dtype], E=E, T=T, N=N, K=K, ldx=ldx, ldw=ldw, ldy=ldy)
    mems = [Mem(padded(x, ldx), dtype, shift[0]), Mem(padded(dy, ldy), dtype, shift[1]), Mem(np.asarray(sizes), "int32")]
    dw = _call(capi.lib().xtc_hip_grouped_matmul_grad_w, d, mems,
               Mem(padded(np.full((E, K, N), 7.0), ldw), out_dtype, shift[2]), stream)
    assert np.isnan(dw[..., N:]).all(), "written past the columns"
    return dw[..., :N]


def quantize(x, dtype, pad=0, shift=0, stream=None):
    """(codes, scales, values) of a 2-D x."""
    rows, K = x.shape
    nb = -(-K // 32)
    d = capi.Mx4Desc(dtype=IDS[dtype], rows=rows, K=K, ld=K + pad, stream=stream)
    src = Mem(padded(x, K + pad), dtype, shift)
    outs = [Mem(np.zeros((rows, 16 * nb)), "uint8"), Mem(np.zeros((rows, nb)), "uint8"), Mem(np.zeros((rows, K)), dtype)]
    capi.check(capi.lib().xtc_hip_mx4_quantize(ctypes.byref(d), src.ptr, *[o.ptr for o in outs]))
    capi.check(capi.lib().xtc_hip_stream_synchronize(stream))
    got = [o.numpy() for o in outs]
    for m in (src, *outs):
        m.free()
    return got


def encode(x, scales, dtype):
    rows, K = x.shape
    d = capi.Mx4Desc(dtype=IDS[dtype], rows=rows, K=K)
    mems = [Mem(x, dtype), Mem(scales, "uint8")]
    return _call(capi.lib().xtc_hip_mx4_encode, d, mems, Mem(np.zeros((rows, 16 * scales.shape[1])), "uint8"), None)


def dequantize(codes, scales, size, dtype):
    d = capi.Mx4Desc(dtype=IDS[dtype], rows=codes.shape[0], K=size)
    mems = [Mem(codes, "uint8"), Mem(scales, "uint8")]
    return _call(capi.lib().xtc_hip_mx4_dequantize, d, mems, Mem(np.zeros((codes.shape[0], size)), dtype), None)


def mx4_matmul(ac, asc, bc, bsc, sizes=None, out_dtype="float32", pad=0, shift=0, stream=None):
    M, nb = asc.shape
    N = bsc.shape[-2]
    d = capi.Mx4MatmulDesc(out_dtype=IDS[out_dtype], E=0 if sizes is None else len(sizes), M=M, N=N, blocks=nb, ldc=N + pad,
                           stream=stream)
    mems = [Mem(a, "uint8") for a in (ac, asc, bc, bsc)]
    sz = None if sizes is None else Mem(np.asarray(sizes), "int32")
    out = Mem(padded(np.full((M, N), 7.0), N + pad), out_dtype, shift)
    capi.check(capi.lib().xtc_hip_mx4_matmul(ctypes.byref(d), *[m.ptr for m in mems], sz.ptr if sz else None, out.ptr))
    capi.check(capi.lib().xtc_hip_stream_synchronize(stream))
    got = out.numpy()
    for m in (*mems, out, *([sz] if sz else [])):
        m.free()
    assert np.isnan(got[:, N:]).all(), "written past the columns"
    return got[:, :N]


def mx4_quantize_matmul(x, dtype, bc, bsc, sizes=None, out_dtype="float32", pad=0, ldx=0, shift=0):
    """The product with x quantised by the same call."""
    (M, K), nb, N = x.shape, bsc.shape[-1], bsc.shape[-2]
    r = capi.Mx4Desc(dtype=IDS[dtype], rows=M, K=K, ld=K + ldx)
    d = capi.Mx4MatmulDesc(out_dtype=IDS[out_dtype], E=0 if sizes is None else len(sizes), M=M, N=N, blocks=nb, ldc=N + pad)
    mx = Mem(padded(x, K + ldx), dtype, shift)
    mems = [mx, Mem(np.zeros((M, 16 * nb)), "uint8"), Mem(np.zeros((M, nb)), "uint8"), Mem(bc, "uint8"), Mem(bsc, "uint8")]
    sz = None if sizes is None else Mem(np.asarray(sizes), "int32")
    out = Mem(padded(np.full((M, N), 7.0), N + pad), out_dtype)
    capi.check(capi.lib().xtc_hip_mx4_quantize_matmul(ctypes.byref(r), ctypes.byref(d), *[m.ptr for m in mems],
                                                      sz.ptr if sz else None, out.ptr))
    capi.check(capi.lib().xtc_hip_synchronize())
    got = out.numpy()
    for m in (*mems, out, *([sz] if sz else [])):
        m.free()
    assert np.isnan(got[:, N:]).all(), "written past the columns"
    return got[:, :N]


def ints(seed, shape, top=4):
    """Whole numbers: sums below 2^24 are exact in fp32, in any order."""
    return np.random.default_rng(seed).integers(-top, top + 1, shape).astype(np.float32)


def rounded(a, dtype):
    return round_to_bf16(a.astype(np.float32)) if dtype == "bfloat16" else a.astype(np.float32)
