// SPDX-License-Identifier: BSD-3-Clause
// Microscaled 4-bit floats: blocks of 32 consecutive elements of a row share a
// power-of-two scale, an element is one of 0, .5, 1, 1.5, 2, 3, 4, 6 with a
// sign (1 sign, 2 exponent, 1 mantissa bit).
//   scale   2^(s - 127), s = max(0, 127 + floor(log2 max|x|) - 2): the largest
//           element lands in [4, 8) and what exceeds 6 becomes 6; s = 255 marks
//           a block that holds an infinity or a NaN, all of it stands for NaN
//   code    sign, then x / scale to the nearest of the eight, ties to the even
//           code; the even element of a byte in its low half
// A row of K elements has ceil(K / 32) blocks, the last one filled up with
// zeros: codes [rows][16 blocks] bytes, scales [rows][blocks] bytes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xtc_hip {
namespace mx4 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// 8 consecutive elements as floats, of which the first n exist
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

// s of a block whose largest magnitude has the bits `top`
__device__ __forceinline__ int scale_of(unsigned top) {
  const int e = (int)(top >> 23);
  return e == 255 ? 255 : max(e - 2, 0);
}

// 1 / scale: 2^(127 - s); 0 for s = 255, whose blocks have codes of 0
__device__ __forceinline__ float inverse_scale(int s) {
  return s < 254 ? __uint_as_float((unsigned)(254 - s) << 23) : s == 254 ? 0x1p-127f : 0.f;
}

// 2^(s - 127), NaN for s = 255
__device__ __forceinline__ float scale_value(int s) {
  return s == 255 ? __uint_as_float(0x7fc00000u) : s ? __uint_as_float((unsigned)s << 23) : 0x1p-127f;
}

// code of x / scale
__device__ __forceinline__ unsigned encode(float x, float inv) {
  const float y = fabsf(x) * inv;
  const unsigned mag = (unsigned)(y > .25f) + (unsigned)(y >= .75f) + (unsigned)(y > 1.25f) + (unsigned)(y >= 1.75f) +
                       (unsigned)(y > 2.5f) + (unsigned)(y >= 3.5f) + (unsigned)(y > 5.f);
  return mag | (__float_as_uint(x) >> 31 << 3);
}

// the value of a code
__device__ __forceinline__ float decode(unsigned c) {
  const unsigned m = c & 7u;
  const float v = m < 4 ? 0.5f * m : m < 6 ? m - 2.f : 2.f * m - 8.f;
  return c & 8u ? -v : v;
}

template <typename U>
__device__ __forceinline__ void store8(U* p, const float (&v)[8], int n) {
  U out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = (U)v[i];
  if (n >= 8) {
    __builtin_memcpy(p, out, sizeof(out));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = out[i];
  }
}

}  // namespace mx4

struct Mx4QuantArgs {
  const void* x;       // [rows][ldx]; null: codes and scales_in are read
  const uint8_t* scales_in;  // codes are made for these scales, or null
  uint8_t* codes;      // each of the three results may be null
  uint8_t* scales;
  void* values;        // [rows][ldv]
  const uint8_t* codes_in;
  int64_t rows;
  int K, blocks, ldx, ldv;
};

// A lane takes a quarter of a block (8 elements), four lanes a block.
// T: elements of x and of the values.
template <typename T>
__global__ void __launch_bounds__(256) mx4_quantize(Mx4QuantArgs p) {
  using namespace mx4;
  const int quarters = 4 * p.blocks;
  const int q = blockIdx.x * 256 + threadIdx.x;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const int k = 8 * q;
    const int n = q < quarters ? p.K - k : 0;  // may be negative past K
    float v[8];
    load8(v, (const T*)p.x + row * p.ldx + k, n);
    int s;
    if (p.scales_in) {
      s = q < quarters ? p.scales_in[row * p.blocks + (q >> 2)] : 0;
    } else {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
      top = max(top, (unsigned)__shfl_xor((int)top, 1));
      top = max(top, (unsigned)__shfl_xor((int)top, 2));
      s = scale_of(top);
    }
    const float inv = inverse_scale(s);
    unsigned word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= encode(v[i], inv) << (4 * i);
    if (s == 255) word = 0;
    if (q >= quarters) continue;
    if (p.codes) *(unsigned*)(p.codes + row * (16 * (int64_t)p.blocks) + 4 * q) = word;
    if (p.scales && (q & 3) == 0) p.scales[row * p.blocks + (q >> 2)] = (uint8_t)s;
    if (p.values) {
      const float scale = scale_value(s);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = decode(word >> (4 * i)) * scale;
      store8((T*)p.values + row * p.ldv + k, v, n);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantize(Mx4QuantArgs p) {
  using namespace mx4;
  const int q = blockIdx.x * 256 + threadIdx.x;
  if (q >= 4 * p.blocks) return;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const unsigned word = *(const unsigned*)(p.codes_in + row * (16 * (int64_t)p.blocks) + 4 * q);
    const float scale = scale_value(p.scales_in[row * p.blocks + (q >> 2)]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = decode(word >> (4 * i)) * scale;
    store8((T*)p.values + row * p.ldv + 8 * q, v, p.K - 8 * q);
  }
}

}  // namespace xtc_hip
