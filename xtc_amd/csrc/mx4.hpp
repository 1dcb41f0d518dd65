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

// s of a block whose largest magnitude has the bits `top`
__device__ __forceinline__ int scale_of(unsigned top) {
  const int e = (int)(top >> 23);
  return e == 255 ? 255 : max(e - 2, 0);
}

// 2^(s - 127), NaN for s = 255
__device__ __forceinline__ float scale_value(int s) {
  return s == 255 ? __uint_as_float(0x7fc00000u) : s ? __uint_as_float((unsigned)s << 23) : 0x1p-127f;
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

namespace mx4 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The larger of this lane's and the lanes' of its quad, by cross-lane moves
// that stay in the vector unit.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // lanes 2 3 0 1
}

// A quarter block, as loaded: its largest magnitude as fp32 bits (only the
// exponent counts) and its codes for a scale, by the conversion instructions
// (which divide by the scale's exponent and round to nearest even, saturating).
struct QuarterBf16 {
  u32x4 v;
  // NaN to zero, keeping its sign
  __device__ __forceinline__ void drop_nan() {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned lo = (v[i] & 0x7fffu) > 0x7f80u ? 0x8000u : 0xffffu;
      const unsigned hi = (v[i] >> 16 & 0x7fffu) > 0x7f80u ? 0x80000000u : 0xffff0000u;
      v[i] &= lo | hi;
    }
  }
  __device__ __forceinline__ unsigned top() const {
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7fff7fffu));
    return (unsigned)max(m[0], m[1]) << 16;
  }
  // (unsigned)v[i]: a bit cast of a vector's element itself would take the first one
  __device__ __forceinline__ unsigned codes(float scale) const {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, (unsigned)v[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, (unsigned)v[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, (unsigned)v[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, (unsigned)v[3]), scale, 3);
  }
};
struct QuarterF32 {
  f32x4 v[2];
  __device__ __forceinline__ void drop_nan() {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = v[i / 4][i % 4];
      v[i / 4][i % 4] = x != x ? __uint_as_float(__float_as_uint(x) & 0x80000000u) : x;
    }
  }
  __device__ __forceinline__ unsigned top() const {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i / 4][i % 4]) & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ unsigned codes(float scale) const {
    unsigned w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0][0], v[0][1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0][2], v[0][3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[1][0], v[1][1], scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[1][2], v[1][3], scale, 3);
  }
};
template <typename T> struct Quarter;
template <> struct Quarter<float> { typedef QuarterF32 type; };
template <> struct Quarter<__bf16> { typedef QuarterBf16 type; };

// the first n of the 8 elements at p, zeros for the others
template <typename T>
__device__ __forceinline__ typename Quarter<T>::type load_quarter(const T* p, int n) {
  T raw[8];
  if (n >= 8) {
    __builtin_memcpy(raw, p, sizeof(raw));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = i < n ? p[i] : (T)0.f;
  }
  typename Quarter<T>::type q;
  __builtin_memcpy(&q, raw, sizeof(q));
  return q;
}

// the 8 values of a dword of codes
__device__ __forceinline__ void values8(float (&v)[8], unsigned word, int s) {
  const float scale = scale_value(s);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 1),
              c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 3);
  v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = s == 255 ? scale : v[i];
}

}  // namespace mx4

// Quantisation of dense rows of whole blocks (`quarters` of 8 elements in all):
// a lane takes QUARTERS of them, a workgroup's width apart, all loads first.  Four
// lanes share a block.  Bound by memory: 8192 x 8192 bf16 reads 134 MB and writes
// 36 (codes, scales) in 29 us or 170 MB (and values) in 51-55, 5.5-6 TB/s.
template <typename T, int QUARTERS>
__global__ void __launch_bounds__(256) mx4_quantize_dense(Mx4QuantArgs p, int64_t quarters) {
  using namespace mx4;
  const int64_t q0 = (int64_t)blockIdx.x * (256 * QUARTERS) + threadIdx.x;
  typename Quarter<T>::type x[QUARTERS];
#pragma unroll
  for (int i = 0; i < QUARTERS; ++i)
    if (q0 + i * 256 < quarters) __builtin_memcpy(&x[i], __builtin_assume_aligned((const T*)p.x + (q0 + i * 256) * 8, 16), sizeof(x[i]));
#pragma unroll
  for (int i = 0; i < QUARTERS; ++i) {
    const int64_t q = q0 + i * 256;
    if (q >= quarters) break;  // whole blocks: never inside a quad
    const int s = scale_of(quad_max(x[i].top()));
    const unsigned word = s == 255 ? 0u : x[i].codes(scale_value(s));
    if (p.codes) *(unsigned*)(p.codes + 4 * q) = word;
    if (p.scales && (threadIdx.x & 3) == 0) p.scales[q >> 2] = (uint8_t)s;
    if (p.values) {
      float v[8];
      values8(v, word, s);
      T out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = (T)v[e];
      __builtin_memcpy(__builtin_assume_aligned((T*)p.values + q * 8, 16), out, sizeof(out));
    }
  }
}

// The same for rows of any length, stride and alignment, and codes for given
// scales.  A lane takes a quarter of a block of each of its rows.  Bound by memory
// and unaligned rows: 8192 x 8100 bf16 41 us, with values 67; 8192 x 8100 fp32 55.
template <typename T>
__global__ void __launch_bounds__(256) mx4_quantize(Mx4QuantArgs p) {
  using namespace mx4;
  const int quarters = 4 * p.blocks;
  const int q = blockIdx.x * 256 + threadIdx.x;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const int n = q < quarters ? p.K - 8 * q : 0;  // may be negative past K
    typename Quarter<T>::type x = load_quarter((const T*)p.x + row * p.ldx + (int64_t)8 * q, n);
    int s;
    if (p.scales_in) {
      x.drop_nan();
      s = q < quarters ? p.scales_in[row * p.blocks + (q >> 2)] : 0;
    } else {
      s = scale_of(quad_max(x.top()));
    }
    const unsigned word = s == 255 ? 0u : x.codes(scale_value(s));
    if (q >= quarters) continue;
    if (p.codes) *(unsigned*)(p.codes + row * (16 * (int64_t)p.blocks) + 4 * q) = word;
    if (p.scales && (q & 3) == 0) p.scales[row * p.blocks + (q >> 2)] = (uint8_t)s;
    if (p.values) {
      float v[8];
      values8(v, word, s);
      store8((T*)p.values + row * p.ldv + (int64_t)8 * q, v, n);
    }
  }
}

// The values of codes and scales.  Bound by memory: 8192 x 8192 to bf16 41 us (4.2
// TB/s), to fp32 87.
template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantize(Mx4QuantArgs p) {
  using namespace mx4;
  const int q = blockIdx.x * 256 + threadIdx.x;
  if (q >= 4 * p.blocks) return;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const unsigned word = *(const unsigned*)(p.codes_in + row * (16 * (int64_t)p.blocks) + 4 * q);
    float v[8];
    values8(v, word, p.scales_in[row * p.blocks + (q >> 2)]);
    store8((T*)p.values + row * p.ldv + (int64_t)8 * q, v, p.K - 8 * q);
  }
}

}  // namespace xtc_hip
