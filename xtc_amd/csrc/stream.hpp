// SPDX-License-Identifier: BSD-3-Clause
// Accesses to memory that a call touches once: the caches are told not to keep it, which
// leaves them to what is read again.  Any alignment to two bytes.
//
// Measured (us, ordinary loads and these): layer norm of 32768 x 4096 bf16 114, 93, its
// gradients for 16384 x 4096 124, 92, 8-bit codes of 8192 x 8192 77, 69.  Stores of results
// that the 256 MB of the last cache do not hold beside what was read gain as well (layer
// norm 129, 114); smaller results stay ordinary, as whoever reads them next finds them
// there.  Matrices of products of few rows gain nothing (expert layer of one token 19.4,
// 20.9; 16 rows by 8192 x 8192 in 8 bits 22.9, 23.2).
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

template <typename V>
__device__ __forceinline__ void store(void* p, const V& from) {
  static_assert(sizeof(V) % 16 == 0, "whole vectors");
  u32x4u w[sizeof(V) / 16];
  __builtin_memcpy(w, &from, sizeof(V));
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 16); ++i) __builtin_nontemporal_store(w[i], (u32x4u*)p + i);
}

}  // namespace stream
}  // namespace xtc_hip
