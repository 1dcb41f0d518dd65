// SPDX-License-Identifier: BSD-3-Clause
// Accesses to memory that a call touches once: the caches are told not to keep it, which
// leaves them to what is read again.  Any alignment to two bytes.
//
// Measured (us, ordinary 16-byte loads and these, inputs that change from pass to pass):
// layer norm of 32768 x 4096 in bf16 99, 97 and in fp32 234, 204, its gradients for 16384 x
// 4096 88, 87 and 173, 152, 8-bit codes and values of 8192 x 8192 71, 69; longer rows go
// either way (fp32 gradients of 16384 x 8192 404, 415 and of 8192 x 16384 479, 442, bf16
// norm of 8192 x 16384 118, 124).  Stores past the caches are for fp32 gradients of rows
// past 4096 elements that the 256 MB of the last cache do not hold beside what was read
// (8192 x 16384 480, 442, 16384 x 8192 424, 415, but 16384 x 4096 152, 152); the norm itself
// loses by them (fp32 204, 209), and smaller results stay ordinary, as whoever reads them
// next finds them there.  Matrices of products of few rows gain nothing (expert layer of one
// token 19.4, 20.9; 16 rows by 8192 x 8192 in 8 bits 22.9, 23.2).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xtc_hip {
namespace stream {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr int64_t LARGE = (int64_t)128 << 20;  // bytes of a result that is not kept

template <typename V>
__device__ __forceinline__ void load(V& to, const void* p) {
  static_assert(sizeof(V) % 16 == 0, "whole vectors");
  u32x4 w[sizeof(V) / 16];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 16); ++i) w[i] = __builtin_nontemporal_load((const u32x4u*)p + i);
  __builtin_memcpy(&to, w, sizeof(V));
}

// PAST the caches, or an ordinary store of whole vectors: a copy of bf16 numbers by
// __builtin_memcpy becomes stores of 12 bytes and of 2 (layer norm of 32768 x 4096 112 us, 97)
template <bool PAST, typename V>
__device__ __forceinline__ void store(void* p, const V& from) {
  static_assert(sizeof(V) % 16 == 0, "whole vectors");
  u32x4u w[sizeof(V) / 16];
  __builtin_memcpy(w, &from, sizeof(V));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 16); ++i) {
    if constexpr (PAST) __builtin_nontemporal_store(w[i], (u32x4u*)p + i);
    else ((u32x4u*)p)[i] = w[i];
  }
}

}  // namespace stream
}  // namespace xtc_hip
