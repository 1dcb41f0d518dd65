# SPDX-License-Identifier: BSD-3-Clause
"""Where an 8-bit product's kernel reads its scales in LDS (xtc_amd/csrc/fp8_scales.hpp),
on the CPU: every row of the largest tile and every slab that a schedule asks for, the one
past a full walk's last among them."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "xtc_amd" / "csrc"

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")

# blocks of a walk, then a line a slab: the offset of every row's four bytes
HARNESS = r"""
#include "fp8_scales.hpp"
#include <cstdio>
int main() {
  using namespace xtc_hip::fp8;
  printf("%d\n", SCALES);
  for (int slab = 0; slab <= 2 * SCALES; ++slab) {
    for (int r = 0; r < 512; ++r) printf("%d ", scales_at(r, slab));
    printf("\n");
  }
}
"""


@pytest.fixture(scope="module")
def offsets(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("fp8_scales")
    (tmp / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(tmp / "h.cpp"), "-o", str(tmp / "h")], check=True)
    head, *lines = subprocess.run([str(tmp / "h")], check=True, capture_output=True, text=True).stdout.splitlines()
    return int(head), [[int(v) for v in line.split()] for line in lines]


@pytest.mark.parametrize("rows", [128, 256, 512])
def test_every_read_stays_in_its_row(offsets, rows):
    """A tile's A and B rows, SCALES bytes each: no read leaves them, nor the row itself."""
    scales, table = offsets
    assert len(table) == 2 * scales + 1
    for slab, line in enumerate(table):
        for r, at in enumerate(line[:rows]):
            assert r * scales <= at and at + 4 <= (r + 1) * scales <= rows * scales, (r, slab, at)


def test_slabs_find_their_blocks(offsets):
    """The bytes of a block are where they were put: chunk c of row r at c ^ (r / 8 % 4)."""
    scales, table = offsets
    for slab, line in enumerate(table[:-1]):
        block = slab // 2
        for r, at in enumerate(line):
            assert at + block % 4 == r * scales + 16 * (block // 16 ^ r // 8 % 4) + block % 16, (r, slab)
