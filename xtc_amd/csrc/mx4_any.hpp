// SPDX-License-Identifier: BSD-3-Clause
// Products of microscaled 4-bit operands of any size, one matrix or one per
// group of rows:
//   c[m, n] = sum over blocks b of 2^(sa[m, b] - 127) 2^(sb[n, b] - 127)
//             sum_{k < 32} a[m, b, k] w[n, b, k]
// on v_mfma_scale_f32_16x16x128_f8f6f4, whose lane takes 32 consecutive 4-bit
// elements (16 bytes) and their scale: exactly one block of a row of the codes.
//
// A workgroup of 2 x 2 waves computes a 64 x 64 tile; the waves read their
// fragments straight from global memory, a step of 16 blocks ahead.  k may be
// summed in any order as long as a and b agree: a lane takes 4 neighbouring blocks
// of its row, 64 bytes of codes and 4 scales in one load of any alignment, and feeds
// them to four MFMAs that each pick their byte of the scales.  Blocks past the last
// one count as zeros of scale 1.
// Bound by the loads that a tile waits for and, for few blocks, by writing c:
// 2253 rows over 32 experts of 672 x 2560 in 26.6 us (a block a lane and step: 38.5),
// 2747 x 1120 x 256 in 6.5 (12.5), 8145 rows over 24 of 160 x 1280, 42 MB of fp32
// out, in 26 (33.7).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "groups.hpp"
#include "mx4.hpp"

namespace xtc_hip {

struct Mx4Args {
  const uint8_t* a_codes;   // [M][16 blocks]
  const uint8_t* a_scales;  // [M][blocks]
  const uint8_t* b_codes;   // [E][N][16 blocks]
  const uint8_t* b_scales;  // [E][N][blocks]
  const int* sizes;         // [E], or null: one product
  void* c;                  // [M][ldc]
  int E, M, N, blocks, ldc;
  int tiles_n;
  const __bf16* x;          // mx4_rows with QUANTIZE: [M][ldx] of K elements, in place of a
  int K, ldx;
};

namespace mx4 {

constexpr int BM = 64, BN = 64;
constexpr int STEP = 16, RING = 2;  // blocks of a step, steps in registers

// one step's part of a row: 4 blocks and their scales
struct Run {
  u32x4 codes[4];
  unsigned scales;
};

// `left` of the 4 blocks at `codes` exist; the others are zeros of scale 1
__device__ __forceinline__ void load_run(Run& r, const uint8_t* codes, const uint8_t* scales, int left) {
  if (left >= 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.codes[j] = *(const u32x4*)(codes + 16 * j);
    __builtin_memcpy(&r.scales, scales, 4);
  } else {
    r.scales = 0x7f7f7f7fu;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.codes[j] = u32x4{0, 0, 0, 0};
      if (j < left) {
        r.codes[j] = *(const u32x4*)(codes + 16 * j);
        r.scales ^= (0x7fu ^ scales[j]) << (8 * j);
      }
    }
  }
}

template <int BYTE>
__device__ __forceinline__ f32x4 mfma_byte(u32x4 a, unsigned sa, u32x4 b, unsigned sb, f32x4 c) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, BYTE, (int)sa, BYTE, (int)sb);
}
__device__ __forceinline__ f32x4 mfma_run(const Run& a, const Run& b, f32x4 c) {
  c = mfma_byte<0>(a.codes[0], a.scales, b.codes[0], b.scales, c);
  c = mfma_byte<1>(a.codes[1], a.scales, b.codes[1], b.scales, c);
  c = mfma_byte<2>(a.codes[2], a.scales, b.codes[2], b.scales, c);
  return mfma_byte<3>(a.codes[3], a.scales, b.codes[3], b.scales, c);
}

// columns n .. n+3 of a row, the first `left` of them
__device__ __forceinline__ void put(float* p, f32x4 v, int left, bool whole) {
  if (whole && left >= 4) *(f32x4*)p = v;
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = v[i];
}
__device__ __forceinline__ void put(__bf16* p, f32x4 v, int left, bool whole) {
  const bf16x4 h = __builtin_convertvector(v, bf16x4);
  if (whole && left >= 4) *(bf16x4*)p = h;
  else
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = h[i];
}

}  // namespace mx4

template <typename U>
__global__ void __launch_bounds__(256) mx4_any(Mx4Args p) {
  using namespace mx4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int mt = blockIdx.x / p.tiles_n, n0 = blockIdx.x % p.tiles_n * BN;
  RowGroup gr{0, mt * BM, p.M};
  if (p.sizes) gr = find_tile<BM>(p.sizes, p.E, p.M, mt);
  if (gr.e < 0) return;
  const int blocks = gr.e < p.E ? p.blocks : 0;  // rows of no group: zeros
  const int e = gr.e < p.E ? gr.e : 0;
  // the lane's first block of each of its rows; rows past the tile's edge repeat
  // the last one and are not stored
  int64_t at_a[2], at_b[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    at_a[i] = (int64_t)min(gr.begin + (wave >> 1) * 32 + i * 16 + l16, gr.end - 1) * p.blocks + 4 * g;
    at_b[i] = ((int64_t)e * p.N + min(n0 + (wave & 1) * 32 + i * 16 + l16, p.N - 1)) * p.blocks + 4 * g;
  }
  Run a[RING][2], b[RING][2];
  int left = blocks - 4 * g;
  auto load = [&](int buf) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load_run(b[buf][i], p.b_codes + at_b[i] * 16, p.b_scales + at_b[i], left);
      load_run(a[buf][i], p.a_codes + at_a[i] * 16, p.a_scales + at_a[i], left);
      at_a[i] += STEP, at_b[i] += STEP;
    }
    left -= STEP;
  };
  f32x4 acc[2][2] = {};
  if (blocks > 0) load(0);
  for (int b0 = 0; b0 < blocks; b0 += RING * STEP) {
#pragma unroll
    for (int q = 0; q < RING; ++q) {
      const int now = b0 + q * STEP;
      if (now >= blocks) break;
      if (now + STEP < blocks) load((q + 1) % RING);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma_run(b[q][j], a[q][i], acc[i][j]);
    }
  }
  const bool whole = (p.ldc & 3) == 0 && ((uintptr_t)p.c & (4 * sizeof(U) - 1)) == 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = gr.begin + (wave >> 1) * 32 + i * 16 + l16;
    if (m >= gr.end) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + (wave & 1) * 32 + j * 16 + 4 * g;
      put((U*)p.c + (int64_t)m * p.ldc + n, acc[i][j], p.N - n, whole);
    }
  }
}

}  // namespace xtc_hip
