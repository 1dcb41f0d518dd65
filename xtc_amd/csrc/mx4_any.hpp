// SPDX-License-Identifier: BSD-3-Clause
// Products of microscaled 4-bit operands of any size, one matrix or one per
// group of rows:
//   c[m, n] = sum over blocks b of 2^(sa[m, b] - 127) 2^(sb[n, b] - 127)
//             sum_{k < 32} a[m, b, k] w[n, b, k]
// on v_mfma_scale_f32_16x16x128_f8f6f4, whose lane takes 32 consecutive 4-bit
// elements (16 bytes) and their scale: exactly one block of a row of the codes.
//
// A workgroup of 2 x 2 waves computes a 64 x 64 tile; the waves read their
// fragments straight from global memory.  Blocks past the last one count as
// zeros of scale 1.
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
};

namespace mx4 {

constexpr int BM = 64, BN = 64;

__device__ __forceinline__ f32x4 mfma(u32x4 a, int sa, u32x4 b, int sb, f32x4 c) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, sa, 0, sb);
}

__device__ __forceinline__ void put(float* p, f32x4 v, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = v[i];
}
__device__ __forceinline__ void put(__bf16* p, f32x4 v, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = (__bf16)v[i];
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
  int64_t arow[2], brow[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    arow[i] = min(gr.begin + (wave >> 1) * 32 + i * 16 + l16, gr.end - 1);
    brow[i] = (int64_t)e * p.N + min(n0 + (wave & 1) * 32 + i * 16 + l16, p.N - 1);
  }
  f32x4 acc[2][2] = {};
  for (int b0 = 0; b0 < blocks; b0 += 4) {
    const int b = b0 + g;
    u32x4 av[2] = {}, bv[2] = {};
    int sa[2] = {127, 127}, sb[2] = {127, 127};
    if (b < blocks) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        av[i] = *(const u32x4*)(p.a_codes + (arow[i] * p.blocks + b) * 16);
        bv[i] = *(const u32x4*)(p.b_codes + (brow[i] * p.blocks + b) * 16);
        sa[i] = p.a_scales[arow[i] * p.blocks + b];
        sb[i] = p.b_scales[brow[i] * p.blocks + b];
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = mfma(bv[j], sb[j], av[i], sa[i], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = gr.begin + (wave >> 1) * 32 + i * 16 + l16;
    if (m >= gr.end) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + (wave & 1) * 32 + j * 16 + 4 * g;
      put((U*)p.c + (int64_t)m * p.ldc + n, acc[i][j], p.N - n);
    }
  }
}

}  // namespace xtc_hip
