// SPDX-License-Identifier: BSD-3-Clause
// 8-bit floats (E4M3) in blocks of 128 elements of a row, or of 128 x 128, that
// share a power-of-two scale:
//   scale   2^(s - 127), the smallest with max|x| <= 448 scale, s >= 0: nothing
//           saturates, and an element is off by at most 2^-4 of itself or 2^-10
//           scale.  s = 255 marks a block that holds an infinity or a NaN, all of
//           it stands for NaN
//   code    x / scale to the nearest of sign, 4 exponent bits (bias 7, 0 subnormal)
//           and 3 mantissa bits, ties to even; 0x7f is NaN, there is no infinity
// A row of K elements has ceil(K / 128) blocks, the last one filled up with zeros.
// A power of two loses no bits of an element and is what the matrix instructions
// apply by themselves: products need no arithmetic beside them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx4.hpp"

namespace xtc_hip {

struct Fp8QuantArgs {
  const void* x;              // [matrices][rows][ldx]
  const uint8_t* scales_in;   // codes are made for these scales (of the one result asked for), or null
  uint8_t *codes, *scales;    // each result may be null
  void* values;               // [matrices][rows][ldv]
  uint8_t *codes_t, *scales_t;  // of the transposed matrices
  const uint8_t* codes_in;
  int64_t rows;               // of a matrix
  int64_t matrices;
  int K, blocks, ldx, ldv;    // blocks of a row
  int square;                 // a scale for every 128 x 128 block
};

namespace fp8 {

using mx4::f32x2;
typedef short i16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// s of a block whose largest magnitude has the bits `top`: 448 is 1.75 x 2^8
__device__ __forceinline__ int scale_of(unsigned top) {
  const int e = (int)(top >> 23);
  return e == 255 ? 255 : max(e - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
}

// A scale as the conversion instructions take it: they look at the exponent bits alone, 0
// is 2^-127 and 255 makes everything NaN
__device__ __forceinline__ float scale_of_byte(unsigned s) { return __uint_as_float(s << 23); }

// Codes of two pairs for a scale, by the conversion instruction (which divides by the
// scale's exponent and rounds to nearest even).
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d, float scale) {
  i16x2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, scale, true);
  return __builtin_bit_cast(unsigned, w);
}

// The sign bits of four codes: the conversion instruction sets a NaN's
__device__ __forceinline__ unsigned signs4(float a, float b, float c, float d) {
  return (__float_as_uint(a) >> 24 & 0x80u) | (__float_as_uint(b) >> 16 & 0x8000u) | (__float_as_uint(c) >> 8 & 0x800000u) |
         (__float_as_uint(d) & 0x80000000u);
}
__device__ __forceinline__ u32x2 signs8(const float (&v)[8]) { return u32x2{signs4(v[0], v[1], v[2], v[3]), signs4(v[4], v[5], v[6], v[7])}; }

// x / 2^(s - 127) within 448; a NaN stays.  What the division rounds (below 2^-126) is
// far below the smallest code.
__device__ __forceinline__ float scaled(float x, int s) {
  const float y = ldexpf(x, 127 - s);
  return (__float_as_uint(y) & 0x7fffffffu) > 0x7f800000u ? y : fminf(fmaxf(y, -448.f), 448.f);
}

__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the 4 values of a dword of codes
__device__ __forceinline__ void values4(float* v, unsigned word, unsigned s) {
  const float scale = scale_of_byte(s);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, scale, true);
  v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// The values of 8 codes as bf16 numbers: exact, as scales are powers of two.
__device__ __forceinline__ bf16x8 values_bf16(unsigned lo, unsigned hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
               c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, int n) {
  T raw[8];
  if (n >= 8) {
    __builtin_memcpy(raw, p, sizeof(raw));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = i < n ? p[i] : (T)0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)raw[i];
}

// The larger of the 16 lanes of a row of lanes
__device__ __forceinline__ unsigned max16(unsigned v) {
  v = mx4::quad_max(v);
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true));  // row_ror:4
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true));  // row_ror:8
}

}  // namespace fp8

// Quantisation by rows: a lane takes RUNS runs of 8 elements, a workgroup's width
// apart, all loads first; 16 lanes share a block.  `dense` says that run q of all
// rows starts at element 8 q.
template <typename T, int RUNS>
__global__ void __launch_bounds__(256) fp8_quantize_rows(Fp8QuantArgs p, int64_t runs, int dense) {
  using namespace fp8;
  const unsigned per_row = 16u * (unsigned)p.blocks;
  const int64_t rows = p.rows * p.matrices;
  for (int64_t base = (int64_t)blockIdx.x * (256 * RUNS); base < runs; base += (int64_t)gridDim.x * (256 * RUNS)) {
    float x[RUNS][8];
    int64_t row[RUNS];
    int at[RUNS];  // the run's first element in its row
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int64_t q = base + i * 256 + threadIdx.x;
      row[i] = 0, at[i] = 0;
      int64_t from = 8 * q;
      int n = q < runs ? 8 : 0;
      if (!dense) {
        row[i] = q / per_row, at[i] = (int)(q - row[i] * per_row) * 8;
        from = row[i] * p.ldx + at[i], n = row[i] < rows ? min(p.K - at[i], 8) : 0;
      }
      load8(x[i], (const T*)p.x + from, n);
    }
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int64_t q = base + i * 256 + threadIdx.x;
      if (q >= runs) break;  // whole blocks: never inside 16 lanes
      int s;
      u32x2 signs = {0, 0};
      if (p.scales_in) {
        signs = signs8(x[i]);
        s = p.scales_in[q >> 4];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = scaled(x[i][j], s);
      } else {
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude(x[i][j]));
        s = scale_of(max16(top));
      }
      const float scale = p.scales_in ? 1.f : scale_of_byte(s);
      u32x2 w = {codes4(x[i][0], x[i][1], x[i][2], x[i][3], scale), codes4(x[i][4], x[i][5], x[i][6], x[i][7], scale)};
      if (p.scales_in) w = (w & 0x7f7f7f7fu) | signs;
      if (s == 255) w = u32x2{0, 0};
      if (p.codes) *(u32x2*)(p.codes + 8 * q) = w;
      if (p.scales && (threadIdx.x & 15) == 0) p.scales[q >> 4] = (uint8_t)s;
      if (p.values) {
        float v[8];
        values4(v, (unsigned)w[0], s), values4(v + 4, (unsigned)w[1], s);
        if (dense) mx4::store8((T*)p.values + 8 * q, v, 8);
        else mx4::store8((T*)p.values + row[i] * p.ldv + at[i], v, p.K - at[i]);
      }
    }
  }
}

// Quantisation by 128 x 128 blocks, of the transposed matrix, or of both: a workgroup
// takes a 128 x 128 piece, a thread 8 x 8 of it, so that the lanes next to one another
// read 256 (bf16) bytes of a row, and the transposed codes leave through LDS as whole
// lines of 128 bytes.
template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_tiles(Fp8QuantArgs p) {
  using namespace fp8;
  __shared__ unsigned col_top[4][128];
  __shared__ unsigned all_top[4];
  __shared__ __attribute__((aligned(16))) unsigned char turned[128][144];
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15, wave = threadIdx.x >> 6;
  const int64_t row_tiles = (p.rows + 127) / 128, tiles = row_tiles * p.blocks * p.matrices;
  const int64_t scale_rows = p.square ? row_tiles : p.rows;                    // of one matrix
  const int64_t scale_rows_t = p.square ? (int64_t)p.blocks : (int64_t)p.K;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int cb = (int)(tile % p.blocks);
    const int64_t rb = tile / p.blocks % row_tiles, e = tile / p.blocks / row_tiles;
    const int64_t r0 = rb * 128 + tr * 8;
    const int c0 = cb * 128 + tc * 8;
    const T* const x = (const T*)p.x + (e * p.rows + r0) * p.ldx + c0;
    float v[8][8];  // row, column
#pragma unroll
    for (int i = 0; i < 8; ++i) load8(v[i], x + (int64_t)i * p.ldx, r0 + i < p.rows ? p.K - c0 : 0);
    unsigned row_top[8], ct[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      row_top[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) row_top[i] = max(row_top[i], magnitude(v[i][j])), ct[j] = max(ct[j], magnitude(v[i][j]));
    }
    int s = 0;  // of the whole piece
    if (p.square) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, row_top[i]);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) top = max(top, (unsigned)__shfl_xor((int)top, d));
      __syncthreads();  // the last piece's readers are done
      if ((threadIdx.x & 63) == 0) all_top[wave] = top;
      __syncthreads();
      s = scale_of(max(max(all_top[0], all_top[1]), max(all_top[2], all_top[3])));
    } else if (p.codes_t || p.scales_t) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        ct[j] = max(ct[j], (unsigned)__shfl_xor((int)ct[j], 16));
        ct[j] = max(ct[j], (unsigned)__shfl_xor((int)ct[j], 32));
      }
      __syncthreads();
      if ((threadIdx.x & 48) == 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) col_top[wave][tc * 8 + j] = ct[j];
      __syncthreads();
    }
    if (p.codes || p.scales || p.values) {
      const int64_t scales = (e * scale_rows + (p.square ? rb : r0)) * p.blocks + cb;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        int si = p.square ? s : scale_of(max16(row_top[i]));
        float in[8];
        u32x2 signs = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) in[j] = v[i][j];
        if (p.scales_in && r0 + i < p.rows) {
          si = p.scales_in[p.square ? scales : scales + (int64_t)i * p.blocks];
          signs = signs8(in);
#pragma unroll
          for (int j = 0; j < 8; ++j) in[j] = scaled(in[j], si);
        }
        const float scale = p.scales_in ? 1.f : scale_of_byte(si);
        u32x2 w = {codes4(in[0], in[1], in[2], in[3], scale), codes4(in[4], in[5], in[6], in[7], scale)};
        if (p.scales_in) w = (w & 0x7f7f7f7fu) | signs;
        if (si == 255) w = u32x2{0, 0};
        if (r0 + i >= p.rows) continue;
        if (p.codes) *(u32x2*)(p.codes + ((e * p.rows + r0 + i) * p.blocks + cb) * 128 + tc * 8) = w;
        if (p.scales && tc == 0 && (!p.square || (tr == 0 && i == 0))) p.scales[p.square ? scales : scales + (int64_t)i * p.blocks] = (uint8_t)si;
        if (p.values) {
          float out[8];
          values4(out, (unsigned)w[0], si), values4(out + 4, (unsigned)w[1], si);
          mx4::store8((T*)p.values + (e * p.rows + r0 + i) * p.ldv + c0, out, p.K - c0);
        }
      }
    }
    if (p.codes_t || p.scales_t) {
      const int64_t scales = (e * scale_rows_t + (p.square ? cb : c0)) * row_tiles + rb;
      // the last piece's readers of `turned` have passed the barriers above
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        int sj = p.square ? s : scale_of(max(max(col_top[0][tc * 8 + j], col_top[1][tc * 8 + j]), max(col_top[2][tc * 8 + j], col_top[3][tc * 8 + j])));
        float in[8];
        u32x2 signs = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) in[i] = v[i][j];
        if (p.scales_in && c0 + j < p.K) {
          sj = p.scales_in[p.square ? scales : scales + j * row_tiles];
          signs = signs8(in);
#pragma unroll
          for (int i = 0; i < 8; ++i) in[i] = scaled(in[i], sj);
        }
        const float scale = p.scales_in ? 1.f : scale_of_byte(sj);
        u32x2 w = {codes4(in[0], in[1], in[2], in[3], scale), codes4(in[4], in[5], in[6], in[7], scale)};
        if (p.scales_in) w = (w & 0x7f7f7f7fu) | signs;
        if (sj == 255) w = u32x2{0, 0};
        *(u32x2*)&turned[tc * 8 + j][tr * 8] = w;
        if (p.scales_t && tr == 0 && c0 + j < p.K && (!p.square || (tc == 0 && j == 0)))
          p.scales_t[p.square ? scales : scales + j * row_tiles] = (uint8_t)sj;
      }
      __syncthreads();
      if (p.codes_t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = i * 32 + (threadIdx.x >> 3);
          if (cb * 128 + c < p.K)
            *(mx4::u32x4*)(p.codes_t + ((e * p.K + cb * 128 + c) * row_tiles + rb) * 128 + (threadIdx.x & 7) * 16) =
                *(const mx4::u32x4*)&turned[c][(threadIdx.x & 7) * 16];
        }
    }
  }
}

// The values of codes and scales: a lane 8 elements.
template <typename T>
__global__ void __launch_bounds__(256) fp8_dequantize(Fp8QuantArgs p, int64_t runs) {
  using namespace fp8;
  const unsigned per_row = 16u * (unsigned)p.blocks;
  const int64_t row_tiles = (p.rows + 127) / 128;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < runs; q += (int64_t)gridDim.x * 256) {
    const int64_t row = q / per_row;
    const int at = (int)(q - row * per_row) * 8;
    const u32x2 w = *(const u32x2*)(p.codes_in + 8 * q);
    int64_t scale = q >> 4;
    if (p.square) {
      const int64_t e = row / p.rows;
      scale = (e * row_tiles + (row - e * p.rows) / 128) * p.blocks + at / 128;
    }
    float v[8];
    const int s = p.scales_in[scale];
    values4(v, (unsigned)w[0], s), values4(v + 4, (unsigned)w[1], s);
    mx4::store8((T*)p.values + row * p.ldv + at, v, p.K - at);
  }
}

}  // namespace xtc_hip
