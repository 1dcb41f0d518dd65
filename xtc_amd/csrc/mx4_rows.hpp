// SPDX-License-Identifier: BSD-3-Clause
// Microscaled 4-bit products of few rows, where the cost is reading b once:
//   c[m, n] = sum_k a[m, k] b[n, k], the rows of a by group as in mx4_any.hpp.
//
// A workgroup computes 16 TM rows x 16 TN columns with 8 waves that share out
// the blocks of k in turn, load their fragments straight into registers, a step
// ahead, and add their sums up in LDS, in order.  k may be summed in any order as
// long as a and b agree, so a lane takes 4 neighbouring blocks of its row (64
// bytes of codes, 4 scales in one load) and feeds them to four
// v_mfma_scale_f32_16x16x128_f8f6f4 one after the other, each picking its byte of
// the scales: a step reads 256 bytes of every row (a block a lane and step: 16 x
// 8192 x 8192 17 us).
// Bound by memory: 16 x 8192 x 8192 reads 36 MB in 9.9 us.
//
// QUANTIZE takes a in bf16 and brings it to 4 bits on the way, every workgroup for
// itself: what mx4_quantize would write, without its launch.
// Bound by the launch and one walk of loads: 16 x 1024 x 2048 4.9 us.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4_any.hpp"

namespace xtc_hip {

namespace mx4 {

constexpr int RWAVES = 8;

// A run of a row of bf16 numbers before its quantisation
struct RawRun {
  QuarterBf16 quarters[16];
};

// `left` of the elements at x exist, whole quarters of blocks; zeros for the others
__device__ __forceinline__ void load_raw(RawRun& r, const __bf16* x, int left) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (8 * i < left) __builtin_memcpy(&r.quarters[i], x + 8 * i, 16);
    else r.quarters[i].v = u32x4{0, 0, 0, 0};
  }
}

__device__ __forceinline__ void quantize_run(Run& r, const RawRun& x) {
  r.scales = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const QuarterBf16* const q = x.quarters + 4 * b;
    const int s = scale_of(max(max(q[0].top(), q[1].top()), max(q[2].top(), q[3].top())));
    const float scale = scale_value(s);
    r.scales |= (unsigned)s << (8 * b);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.codes[b][i] = s == 255 ? 0u : q[i].codes(scale);
  }
}

}  // namespace mx4

template <typename U, int TM, int TN, bool QUANTIZE>
__global__ void __launch_bounds__(64 * mx4::RWAVES) mx4_rows(Mx4Args p) {
  using namespace mx4;
  constexpr int SM = 16 * TM, SN = 16 * TN;
  static_assert(RING == 2, "a run is quantised a step ahead");
  __shared__ float sums[RWAVES][SM][SN + 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int mt = blockIdx.x / p.tiles_n, n0 = blockIdx.x % p.tiles_n * SN;
  RowGroup gr{0, mt * SM, p.M};
  if (p.sizes) gr = find_tile<SM>(p.sizes, p.E, p.M, mt);
  if (gr.e < 0) return;
  const int blocks = gr.e < p.E ? p.blocks : 0;  // rows of no group: zeros
  const int e = gr.e < p.E ? gr.e : 0;
  const int rows = min(gr.end - gr.begin, SM), cols = min(p.N - n0, SN);

  // the lane's first block of each of its rows; rows past the tile's edge repeat
  // the last one and are not stored
  const int first = wave * STEP + g * 4;
  int64_t at_a[TM], at_b[TN];
#pragma unroll
  for (int i = 0; i < TM; ++i) at_a[i] = (int64_t)(gr.begin + min(16 * i + l16, rows - 1)) * p.blocks + first;
#pragma unroll
  for (int j = 0; j < TN; ++j) at_b[j] = ((int64_t)e * p.N + n0 + min(16 * j + l16, cols - 1)) * p.blocks + first;
  constexpr int A_RING = QUANTIZE ? 1 : RING;
  Run a[A_RING][TM], b[RING][TN];
  RawRun raw[TM];
  const __bf16* at_x[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i)
    if constexpr (QUANTIZE) at_x[i] = p.x + (int64_t)(gr.begin + min(16 * i + l16, rows - 1)) * p.ldx + 32 * first;
  int left = blocks - first, left_x = blocks > 0 ? p.K - 32 * first : 0;
  auto load = [&](int buf) {
    if constexpr (QUANTIZE) {
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        load_raw(raw[i], at_x[i], left_x);
        at_x[i] += 32 * RWAVES * STEP;
      }
      left_x -= 32 * RWAVES * STEP;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      load_run(b[buf][j], p.b_codes + at_b[j] * 16, p.b_scales + at_b[j], left);
      at_b[j] += RWAVES * STEP;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if constexpr (!QUANTIZE) load_run(a[buf][i], p.a_codes + at_a[i] * 16, p.a_scales + at_a[i], left);
      at_a[i] += RWAVES * STEP;
    }
    left -= RWAVES * STEP;
  };
  auto quantize = [&] {
#pragma unroll
    for (int i = 0; i < TM; ++i) quantize_run(a[0][i], raw[i]);
  };
  f32x4 acc[TM][TN] = {};
  const int steps = (blocks - wave * STEP + RWAVES * STEP - 1) / (RWAVES * STEP);  // of this wave
#pragma unroll
  for (int s = 0; s < RING - 1; ++s)
    if (s < steps) load(s);
  if (QUANTIZE && steps > 0) quantize();
  for (int s = 0; s < steps; s += RING) {
#pragma unroll
    for (int q = 0; q < RING; ++q) {
      if (s + q >= steps) break;
      if (s + q + RING - 1 < steps) load((q + RING - 1) % RING);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma_run(b[q][j], a[q % A_RING][i], acc[i][j]);
      if (QUANTIZE && s + q + 1 < steps) quantize();  // the step just loaded: one step ahead
    }
  }
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
    ((U*)p.c)[(int64_t)(gr.begin + m) * p.ldc + n0 + n] = (U)v;
  }
}

}  // namespace xtc_hip
