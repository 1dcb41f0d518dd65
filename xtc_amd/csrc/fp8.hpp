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
#include "stream.hpp"

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
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
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

// The values of 8 codes as bf16 numbers: exact for scale bytes from 3 to 246.  Below, a
// code's last bits lie under bf16's smallest number, 2^-133; above, 448 scale lies past its
// largest, below 2^128.
__device__ __forceinline__ bf16x8 values_bf16(unsigned lo, unsigned hi, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true),
               c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 8 neighbours of a row as stored
template <typename T>
struct Run8 {
  T v[8];
  // the first n of the 8 elements at p, zeros for the others
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= 8) {
      stream::load(v, p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0.f;
    }
  }
  __device__ __forceinline__ void widen(float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (float)v[i];
  }
};

// The larger of the 16 lanes of a row of lanes
__device__ __forceinline__ unsigned max16(unsigned v) {
  v = mx4::quad_max(v);
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, true));  // row_ror:4
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true));  // row_ror:8
}

// Largest magnitudes of pairs (bf16) or single elements (fp32) of 8 neighbours, kept as
// words: bf16 numbers order by their bits, two a word.
template <typename T>
struct Tops {
  static constexpr int WORDS = 8;
  unsigned w[WORDS] = {};
  __device__ __forceinline__ void add(const Run8<T>& x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = max(w[j], magnitude(x.v[j]));
  }
  __device__ __forceinline__ unsigned all() const {
    unsigned top = w[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = max(top, w[j]);
    return top;
  }
  static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return max(a, b); }
  // of column j, from words of all the columns
  static __device__ __forceinline__ unsigned column(const unsigned* words, int j) { return words[j]; }
};
template <>
struct Tops<__bf16> {
  static constexpr int WORDS = 4;
  unsigned w[WORDS] = {};
  static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
  }
  __device__ __forceinline__ void add(const Run8<__bf16>& x) {
    unsigned raw[4];
    __builtin_memcpy(raw, &x, sizeof(raw));
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = larger(w[j], raw[j] & 0x7fff7fffu);
  }
  __device__ __forceinline__ unsigned all() const {
    const unsigned top = larger(larger(w[0], w[1]), larger(w[2], w[3]));
    return max(top & 0xffff0000u, top << 16);
  }
  static __device__ __forceinline__ unsigned column(const unsigned* words, int j) {
    const unsigned top = words[j / 2];
    return j % 2 ? top & 0xffff0000u : top << 16;
  }
};

// 4 codes for a scale.  ENCODE: a scale that somebody chose, which elements may pass.
template <bool ENCODE>
__device__ __forceinline__ unsigned codes_for(float a, float b, float c, float d, int s) {
  unsigned w;
  if constexpr (ENCODE) {
    w = codes4(scaled(a, s), scaled(b, s), scaled(c, s), scaled(d, s), 1.f);
    w = (w & 0x7f7f7f7fu) | signs4(a, b, c, d);
  } else {
    w = codes4(a, b, c, d, scale_of_byte(s));
  }
  return s == 255 ? 0u : w;
}
template <bool ENCODE>
__device__ __forceinline__ u32x2 codes8(const float (&x)[8], int s) {
  return u32x2{codes_for<ENCODE>(x[0], x[1], x[2], x[3], s), codes_for<ENCODE>(x[4], x[5], x[6], x[7], s)};
}

}  // namespace fp8

// Quantisation by rows: a lane takes RUNS runs of 8 elements, a workgroup's width
// apart, all loads first; 16 lanes share a block.  `dense` says that run q of all
// rows starts at element 8 q.  Bound by memory: 8192 x 8192 bf16 40 us (5.0 TB/s).
template <typename T, int RUNS, bool ENCODE>
__global__ void __launch_bounds__(256) fp8_quantize_rows(Fp8QuantArgs p, int64_t runs, int dense) {
  using namespace fp8;
  const unsigned per_row = 16u * (unsigned)p.blocks;
  const int64_t rows = p.rows * p.matrices;
  for (int64_t base = (int64_t)blockIdx.x * (256 * RUNS); base < runs; base += (int64_t)gridDim.x * (256 * RUNS)) {
    Run8<T> raw[RUNS];
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
      raw[i].load((const T*)p.x + from, n);
    }
#pragma unroll
    for (int i = 0; i < RUNS; ++i) {
      const int64_t q = base + i * 256 + threadIdx.x;
      if (q >= runs) break;  // whole blocks: never inside 16 lanes
      float x[8];
      raw[i].widen(x);
      int s;
      if constexpr (ENCODE) {
        s = p.scales_in[q >> 4];
      } else {
        Tops<T> tops;
        tops.add(raw[i]);
        s = scale_of(max16(tops.all()));
      }
      const u32x2 w = codes8<ENCODE>(x, s);
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

// Quantisation by 128 x 128 blocks, of the transposed matrix, or of both: a workgroup of
// 512 threads takes a 128 x 128 piece, a thread 4 rows x 8 columns of it, so that 16 lanes
// read 256 (bf16) neighbouring bytes of a row, and the transposed codes leave through LDS
// as whole lines of 128 bytes.  Bound by memory: 8192 x 8192 bf16 to codes and back 69 us
// (4.9 TB/s); with 256 threads of 8 x 8 elements, whose registers left two workgroups a
// CU, 101.
template <typename T, bool ENCODE>
__global__ void __launch_bounds__(512) fp8_quantize_tiles(Fp8QuantArgs p) {
  using namespace fp8;
  constexpr int WORDS = Tops<T>::WORDS;
  __shared__ unsigned col_top[8][16 * WORDS];
  __shared__ unsigned all_top[8];
  __shared__ uint8_t col_scale[128];
  // rows of 33 words: the 16 lanes side by side write columns that lie 8 rows apart
  __shared__ unsigned turned[128][33];
  const int tr = threadIdx.x >> 4, tc = threadIdx.x & 15, wave = threadIdx.x >> 6;
  const int64_t row_tiles = (p.rows + 127) / 128, tiles = row_tiles * p.blocks * p.matrices;
  const int64_t scale_rows = p.square ? row_tiles : p.rows;                    // of one matrix
  const int64_t scale_rows_t = p.square ? (int64_t)p.blocks : (int64_t)p.K;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int cb = (int)(tile % p.blocks);
    const int64_t rb = tile / p.blocks % row_tiles, e = tile / p.blocks / row_tiles;
    const int64_t r0 = rb * 128 + tr * 4;
    const int c0 = cb * 128 + tc * 8;
    const T* const x = (const T*)p.x + (e * p.rows + r0) * p.ldx + c0;
    Run8<T> raw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i].load(x + (int64_t)i * p.ldx, r0 + i < p.rows ? p.K - c0 : 0);
    int s = 0;  // of the whole piece
    if constexpr (!ENCODE) {
      if (p.square) {
        Tops<T> tops;
#pragma unroll
        for (int i = 0; i < 4; ++i) tops.add(raw[i]);
        unsigned top = max16(tops.all());
        top = max(top, (unsigned)__shfl_xor((int)top, 16));
        top = max(top, (unsigned)__shfl_xor((int)top, 32));
        __syncthreads();  // the last piece's readers are done
        if ((threadIdx.x & 63) == 0) all_top[wave] = top;
        __syncthreads();
        top = all_top[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = max(top, all_top[i]);
        s = scale_of(top);
      } else if (p.codes_t || p.scales_t) {
        Tops<T> tops;
#pragma unroll
        for (int i = 0; i < 4; ++i) tops.add(raw[i]);
#pragma unroll
        for (int j = 0; j < WORDS; ++j) {
          tops.w[j] = Tops<T>::larger(tops.w[j], (unsigned)__shfl_xor((int)tops.w[j], 16));
          tops.w[j] = Tops<T>::larger(tops.w[j], (unsigned)__shfl_xor((int)tops.w[j], 32));
        }
        // the last piece's readers of col_top and col_scale have passed the barriers below
        if ((threadIdx.x & 48) == 0)
#pragma unroll
          for (int j = 0; j < WORDS; ++j) col_top[wave][tc * WORDS + j] = tops.w[j];
        __syncthreads();
        if (threadIdx.x < 16 * WORDS) {
          unsigned top = col_top[0][threadIdx.x];
#pragma unroll
          for (int i = 1; i < 8; ++i) top = Tops<T>::larger(top, col_top[i][threadIdx.x]);
#pragma unroll
          for (int j = 0; j < 8 / WORDS; ++j)
            col_scale[threadIdx.x * (8 / WORDS) + j] = (uint8_t)scale_of(Tops<T>::column(&top, j));
        }
        __syncthreads();
      }
    }
    float v[4][8];  // row, column
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i].widen(v[i]);
    if (p.codes || p.scales || p.values) {
      const int64_t scales = (e * scale_rows + (p.square ? rb : r0)) * p.blocks + cb;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int si = s;
        if constexpr (ENCODE) {
          if (r0 + i < p.rows) si = p.scales_in[p.square ? scales : scales + (int64_t)i * p.blocks];
        } else if (!p.square) {
          Tops<T> tops;
          tops.add(raw[i]);
          si = scale_of(max16(tops.all()));
        }
        const u32x2 w = codes8<ENCODE>(v[i], si);
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
      if constexpr (ENCODE) __syncthreads();  // the last piece's readers of `turned`; else they have passed the barriers above
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        int sj = s;
        if constexpr (ENCODE) {
          if (c0 + j < p.K) sj = p.scales_in[p.square ? scales : scales + j * row_tiles];
        } else if (!p.square) {
          sj = col_scale[tc * 8 + j];
        }
        turned[tc * 8 + j][tr] = codes_for<ENCODE>(v[0][j], v[1][j], v[2][j], v[3][j], sj);
        if (p.scales_t && tr == 0 && c0 + j < p.K && (!p.square || (tc == 0 && j == 0)))
          p.scales_t[p.square ? scales : scales + j * row_tiles] = (uint8_t)sj;
      }
      __syncthreads();
      if (p.codes_t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = i * 64 + (threadIdx.x >> 3), at = (threadIdx.x & 7) * 4;
          const mx4::u32x4 line = {turned[c][at], turned[c][at + 1], turned[c][at + 2], turned[c][at + 3]};
          if (cb * 128 + c < p.K) *(mx4::u32x4*)(p.codes_t + ((e * p.K + cb * 128 + c) * row_tiles + rb) * 128 + at * 4) = line;
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
