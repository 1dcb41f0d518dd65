// SPDX-License-Identifier: BSD-3-Clause
// Products of 8-bit floats (fp8.hpp) of few rows, where the cost is reading b once:
//   c[m, n] = sum_k a[m, k] b[n, k]
//
// A workgroup computes 16 TM rows x 16 TN columns with 8 waves that share out k in
// steps of two blocks in turn, load their fragments straight into registers, a step
// ahead, and add their sums up in LDS, in order.  A lane holds two times 16 bytes of its
// row's block, so that the four lanes of a row read 64 neighbouring ones, and brings them
// to bf16, scale and all, for four v_mfma_f32_16x16x32_bf16: k may be summed in any order as
// long as a and b agree.
// Bound by the stream of b: 16 rows by 8192 x 8192 18 us (3.7 TB/s).
// The sums are fp32 whatever the result's type (fp8_dma.hpp), as memory leaves the time.
#pragma once
#include "fp8_dma.hpp"

namespace xtc_hip {

namespace fp8 {

constexpr int RWAVES = 8, RING = 2, STEP = 2;  // blocks of a step

// A lane's bytes of two blocks of a row and their scales
struct Run {
  gdma::u32x4 codes[2 * STEP];
  unsigned scale[STEP];
};

// `left` of the blocks at `scale` exist; zeros for the others
__device__ __forceinline__ void load_run(Run& r, const uint8_t* codes, const uint8_t* scale, int left) {
#pragma unroll
  for (int h = 0; h < STEP; ++h)
    if (h < left) {
      r.codes[2 * h] = *(const gdma::u32x4*)(codes + 128 * h);
      r.codes[2 * h + 1] = *(const gdma::u32x4*)(codes + 128 * h + 64);
      r.scale[h] = scale[h];
    } else {
      r.codes[2 * h] = r.codes[2 * h + 1] = gdma::u32x4{0, 0, 0, 0};
      r.scale[h] = 127;
    }
}

// 8 of a lane's elements of block h
__device__ __forceinline__ bf16x8 elements(const Run& r, int h, int i) {
  const gdma::u32x4 v = r.codes[2 * h + (i >> 1)];
  return values_bf16(v[2 * (i & 1)], v[2 * (i & 1) + 1], scale_of_byte(r.scale[h]));
}

template <int TM, int TN>
__device__ __forceinline__ void multiply(gdma::f32x4 (&acc)[TM][TN], const Run (&a)[TM], const Run (&b)[TN]) {
#pragma unroll
  for (int h = 0; h < STEP; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x8 av[TM], bv[TN];
#pragma unroll
      for (int m = 0; m < TM; ++m) av[m] = elements(a[m], h, i);
#pragma unroll
      for (int n = 0; n < TN; ++n) bv[n] = elements(b[n], h, i);
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv[n], av[m], acc[m][n], 0, 0, 0);
    }
}

}  // namespace fp8

template <typename U, int TM, int TN>
__global__ void __launch_bounds__(64 * fp8::RWAVES) fp8_rows(Fp8Args p) {
  using namespace fp8;
  using gdma::f32x4;
  constexpr int SM = 16 * TM, SN = 16 * TN;
  __shared__ float sums[RWAVES][SM][SN + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.x / p.tiles_n * SM, n0 = blockIdx.x % p.tiles_n * SN;
  const int rows = min(p.M - m0, SM), cols = min(p.N - n0, SN);
  const int first = wave * STEP;  // the wave's first block
  // rows past the tile's edge repeat the last one and are not stored
  const uint8_t *a[TM], *b[TN], *sa[TM], *sb[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t at = (int64_t)(m0 + min(16 * i + l16, rows - 1)) * p.blocks + first;
    a[i] = p.a + 128 * at + 16 * g, sa[i] = p.sa + at;
  }
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int64_t n = n0 + min(16 * j + l16, cols - 1);
    b[j] = p.b + 128 * (n * p.blocks + first) + 16 * g, sb[j] = p.sb + (n >> p.b_shift) * p.blocks + first;
  }
  Run fa[RING][TM], fb[RING][TN];
  int left = p.blocks - first;
  auto load = [&](int buf) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      load_run(fb[buf][j], b[j], sb[j], left);
      b[j] += 128 * RWAVES * STEP, sb[j] += RWAVES * STEP;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      load_run(fa[buf][i], a[i], sa[i], left);
      a[i] += 128 * RWAVES * STEP, sa[i] += RWAVES * STEP;
    }
    left -= RWAVES * STEP;
  };
  f32x4 acc[TM][TN] = {};
  const int steps = (p.blocks - wave * STEP + RWAVES * STEP - 1) / (RWAVES * STEP);  // of this wave
#pragma unroll
  for (int s = 0; s < RING - 1; ++s)
    if (s < steps) load(s);
  for (int s = 0; s < steps; s += RING) {
#pragma unroll
    for (int q = 0; q < RING; ++q) {
      if (s + q >= steps) break;
      if (s + q + RING - 1 < steps) load((q + RING - 1) % RING);
      multiply(acc, fa[q], fb[q]);
    }
  }
  // the sums are read behind branches: their wait states are spelled out
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15");
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) *(f32x4*)&sums[wave][16 * i + l16][16 * j + 4 * g] = acc[i][j];
  __syncthreads();
  for (int t = threadIdx.x; t < SM * SN; t += 64 * RWAVES) {
    const int m = t / SN, n = t % SN;
    if (m >= rows || n >= cols) continue;
    float v = sums[0][m][n];
#pragma unroll
    for (int w = 1; w < RWAVES; ++w) v += sums[w][m][n];
    ((U*)p.c)[(int64_t)(m0 + m) * p.ldc + n0 + n] = (U)v;
  }
}

}  // namespace xtc_hip
