# SPDX-License-Identifier: BSD-3-Clause
"""Sizes (M, N, blocks of k) of 8-bit products that reach every kernel, by how they add up
and their result's type.  test_fp8_sums checks on the CPU that they do."""

FP32, FP8 = 1, 2  # XTC_HIP_SUMS_..

# kernel: a size that takes it
ROWS = {"rows16": (5, 70, 3), "rows32": (30, 4200, 9)}
TILES = {"64": (500, 1100, 5), "128": (2000, 4096, 9), "256": (4000, 3904, 65)}
# (sums, out dtype, kernel, size)
CASES = [(sums, out, kernel, size) for sums in (FP32, FP8) for out in ("float32", "bfloat16")
         for kernel, size in ({**ROWS, **TILES} if sums == FP32 else TILES).items()]
