// SPDX-License-Identifier: BSD-3-Clause
// Where the scales of an 8-bit product's tile lie in LDS (fp8_dma.hpp): plain C++, so
// that a CPU test walks over all of it.
//
// SCALES bytes a row, the blocks of a walk, in 16-byte chunks of which chunk c of row r
// stands at c ^ swz(r).  A slab is half a block, and a lane reads the four bytes of eight
// slabs at once.
#pragma once

namespace xtc_hip {
namespace fp8 {

constexpr int SCALES = 64;  // blocks of a walk

constexpr int swz(int r) { return (r >> 3) & 3; }

// Offset of the four bytes of row r that hold slab `slab`'s, 0 .. 2 SCALES.  The slab
// past the last one, which a schedule without a branch round the read asks for, wraps to
// the row's first bytes: in bounds, and used by no one.
constexpr int scales_at(int r, int slab) {
  return r * SCALES + 16 * ((slab >> 5 & (SCALES / 16 - 1)) ^ swz(r)) + (slab >> 1 & 12);
}

}  // namespace fp8
}  // namespace xtc_hip
