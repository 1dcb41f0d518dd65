# SPDX-License-Identifier: BSD-3-Clause
"""Calls of the expert and 4-bit entry points by the kernel that each is meant to
reach: the GPU compares their results with plain forms, the CPU checks that the
call does launch that kernel."""

from __future__ import annotations

F, B = "float32", "bfloat16"
TYPES = [(F, F), (B, F), (B, B)]
_C = {F: "float", B: "__bf16"}


def _bool(*flags):
    return ", ".join("true" if f else "false" for f in flags)


# ---- products by group: (kernel, operands, result, transposed, T, K, N, sizes)

# 64 x 64 slabs of any operands: one slab, as many as a register ring holds, one more,
# many; the last one cut; ragged groups, one of a row, an empty one, rows of nobody
_SLABS = [(1500, k, 2057, [400, 0, 1, 700, 64, 300]) for k in (20, 95, 127, 201)]
GROUPED_ANY = [(f"grouped_any<{_C[d]}, {_C[o]}, {_bool(t, False)}>", d, o, t, *size)
               for d, o in TYPES for t in (False, True) for size in _SLABS]
# whole vectors too in fp32, which has no other kernel of many tiles
GROUPED_ANY += [(f"grouped_any<float, float, {_bool(t, False)}>", F, F, t, 1500, 264, 2056, [400, 0, 1, 700, 64, 300])
                for t in (False, True)]

# waves that share out the depth: 16 rows by 16, 32 or 64 columns, cut in both; depths of
# one step of one wave, of every wave's, and of more than a register ring holds
_SMALL = [(16, True, 9, 3, 2), (16, True, 9, 777, 50), (16, True, 5, 2500, 37), (32, False, 200, 45, 300),
          (32, False, 200, 1300, 70), (32, True, 200, 45, 300), (32, True, 200, 1300, 70), (64, False, 20, 9, 3),
          (64, False, 20, 2500, 130), (64, False, 700, 300, 723), (64, True, 700, 300, 723)]
GROUPED_SMALL = [(f"grouped_small<{_C[d]}, {_C[o]}, {_bool(t, False)}, 1, {n // 16}>", d, o, t, T, k, N,
                  [T // 2, 0, T // 3 + 1] if n != 64 or T > 20 else [T // 2, 0, T // 3])
                 for d, o in TYPES for n, t, T, k, N in _SMALL]


def _dma(grad, t, tile):
    return f"grouped_dma<false, {_bool(grad, t)}, {tile}>"


TILE64, TILE128, TILE256 = "2, 2, 2, 2, 4, false", "2, 2, 4, 4, 4, false", "2, 4, 8, 4, 4, true"
# LDS-DMA tiles cut in rows, columns and depth; K of fewer slabs than the three that
# are in flight where the call takes the tile (256 x 256 ones start at deeper sums)
_DMA = [(TILE64, B, 1500, 32, 2056, [500, 1, 0, 300, 257, 375]), (TILE64, B, 1500, 72, 2056, [500, 1, 0, 300, 257, 375]),
        (TILE64, F, 1500, 200, 2056, [500, 1, 0, 300, 257, 375]),
        (TILE128, B, 4100, 40, 3336, [1300, 1, 0, 800, 257, 1025]), (TILE128, F, 4100, 72, 3336, [1300, 1, 0, 800, 257, 1025]),
        (TILE128, F, 4100, 264, 3336, [1300, 1, 0, 800, 257, 1025]),
        (TILE256, B, 3300, 200, 4104, [1700, 0, 1, 1500]), (TILE256, F, 3300, 264, 4104, [1700, 0, 1, 1500]),
        (TILE256, F, 3300, 520, 4104, [1, 257, 2900, 0]), (TILE256, B, 5000, 264, 2312, [2000, 1, 0, 1300, 257, 900]),
        (TILE256, F, 2300, 1032, 3336, [100, 2100, 0])]
# one slab and less of it, with results of either type
_DMA += [(tile, o, T, K, N, sizes) for o in (F, B) for K in (8, 32) for tile, T, N, sizes in (
    (TILE64, 1500, 2056, [500, 1, 0, 300, 257, 375]), (TILE128, 4100, 3336, [1300, 1, 0, 800, 257, 1025]))
    if (tile, o, T, K) != (TILE64, B, 1500, 32)]
GROUPED_DMA = [(_dma(False, t, tile), B, o, t, *size) for tile, o, *size in _DMA for t in (False, True)]

# ---- gradients: (kernel, in parts, operands, result, T, K, N, sizes)

GRAD_ANY = [(f"grouped_any<{_C[d]}, {_C[o]}, false, true>", False, d, o, *size) for d, o in TYPES
            for size in ((400, 905, 777, [200, 0, 33, 1, 96, 60]), (900, 1001, 721, [32, 700, 0, 160]))]
GRAD_SMALL = [(f"grouped_small<{_C[d]}, {_C[o]}, false, true, 2, 2>", False, d, o, *size) for d, o in TYPES
              for size in ((30, 19, 23, [1, 0, 29]), (2600, 77, 45, [300, 0, 2298, 1]), (900, 333, 250, [450, 33, 0, 417]))]
GRAD_DMA = [(_dma(True, False, tile), parts, B, o, *size) for o in (F, B) for tile, parts, *size in (
    (TILE64, False, 420, 264, 520, [200, 0, 33, 1, 96, 60]),
    (TILE128, False, 600, 648, 520, [16] * 20 + [33, 0, 1, 96] + [5] * 8),
    (TILE256, False, 1500, 1544, 1800, [32, 300, 0, 5, 97, 1000]),
    (TILE256, False, 900, 2056, 2312, [1, 96, 800, 0]),
    # summed in parts: a group of fewer slabs than parts, one of a single slab, an empty
    # one, next to groups that are split; tiles cut by K and N
    (TILE64, True, 9000, 128, 136, [8600, 100, 20, 0]),
    (TILE64, True, 16000, 72, 136, [0, 33, 6000, 9000, 900]),
    (TILE64, True, 6000, 264, 520, [100, 5000, 32]),
    (TILE128, True, 24000, 264, 520, [14000, 33, 0, 9000]),
    (TILE128, True, 30000, 776, 520, [20, 20000, 9000]),
)]

# ---- 4-bit products: (kernel, result, M, N, blocks, sizes or None, bytes that the
# scales of a and b lie past a 16-byte boundary)

_GROUPS = [700, 1, 0, 420, 257, 700]
MX4 = [(f"{kernel}{_C[o]}{rest}", o, *call) for o in (F, B) for kernel, rest, *call in (
    # one step, two, more than the ring; the last run of blocks cut to 1, 2 and 3
    ("mx4_any<", ">", 2100, 2056, 13, None, (0, 0)), ("mx4_any<", ">", 2100, 2056, 33, None, (0, 0)),
    ("mx4_any<", ">", 700, 1000, 50, None, (0, 0)), ("mx4_any<", ">", 700, 1000, 103, None, (0, 0)),
    ("mx4_any<", ">", 2100, 2056, 13, _GROUPS, (0, 0)), ("mx4_any<", ">", 700, 1500, 7, [300, 0, 399], (0, 0)),
    # whole slabs whose scales cannot be staged in dwords
    ("mx4_any<", ">", 2100, 2056, 12, None, (1, 0)), ("mx4_any<", ">", 2100, 2056, 36, _GROUPS, (0, 2)),
    ("mx4_rows<", ", 1, 2, false>", 16, 1000, 12, None, (1, 3)), ("mx4_rows<", ", 1, 2, false>", 20, 200, 16, [9, 0, 10], (3, 1)),
    ("mx4_rows<", ", 2, 2, false>", 32, 8192, 20, None, (2, 1)),
)] + [(f"grouped_dma<true, false, true, {tile}>", o, *call, (0, 0)) for o in (F, B) for tile, *call in (
    ("2, 2, 2, 2, 4, false", 700, 1000, 12, [300, 0, 1, 390]), ("2, 2, 4, 4, 2, false", 2100, 2056, 68, _GROUPS),
    ("2, 4, 8, 4, 2, true", 2000, 4104, 68, [900, 1, 0, 600, 257]), ("2, 4, 8, 4, 2, true", 4100, 3336, 36, None),
)]

# ---- operands whose rows or matrices lie more than 2^32 bytes apart:
# (kernel, T, K, N, sizes, row strides of x, y and (gradients) dy, between matrices)

FAR = [(_dma(False, False, TILE64), 700, 264, 2056, [300, 0, 390], 2**22 - 16, 2**21 + 8, 2**30 + 16),
       (_dma(False, True, TILE64), 700, 264, 2056, [300, 0, 390], 2**22 - 16, 2**21 + 8, 2**30 + 16),
       (f"grouped_any<__bf16, float, {_bool(False, False)}>", 1100, 201, 2057, [500, 0, 590], 2**21 + 5, 2**20 + 3, 2**30 + 15),
       (f"grouped_any<__bf16, float, {_bool(True, False)}>", 1100, 201, 2057, [500, 0, 590], 2**21 + 5, 2**20 + 3, 2**30 + 15)]
FAR_GRAD = [(_dma(True, False, TILE64), 700, 264, 520, [300, 0, 390], 2**22 - 16, 2**22 - 24, 2**30 + 16),
            ("grouped_any<__bf16, float, false, true>", 1100, 1001, 721, [500, 0, 590], 2**21 + 5, 2**21 + 7, 2**30 + 15)]
# (kernel, M, N, blocks, sizes or None, row stride of c or 0)
FAR_MX4 = [("grouped_dma<true, false, true, 2, 2, 2, 2, 4, false>", 40, 400000, 256, [15, 0, 25], 2**25 + 4),
           ("grouped_dma<true, false, true, 2, 2, 2, 2, 4, false>", 2**20 + 40, 64, 256, None, 0),
           ("mx4_any<float>", 40, 2**20 + 72, 257, None, 2**25 + 1), ("mx4_any<float>", 2**20 + 40, 64, 257, None, 0),
           ("mx4_rows<float, 1, 2, false>", 16, 2**20 + 72, 257, None, 0)]


def transposed(kernel):
    """Whether a kernel of FAR takes transposed matrices."""
    return kernel.startswith(("grouped_dma<false, false, true", "grouped_any<__bf16, float, true"))
