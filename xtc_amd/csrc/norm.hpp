// SPDX-License-Identifier: BSD-3-Clause
// Layer norm over the K elements of a row, and its gradients:
//   m = sum x / K,  r = 1 / sqrt(sum (x - m)^2 / K + eps),  xh = (x - m) r
//   y = xh w + b
//   g = dy w,  dx = r (g - sum g / K - xh sum (g xh) / K)
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// All sums are fp32; results are rounded once.
//
// A row stays in the registers of the THREADS threads that share it, VECS runs
// of 8 elements each, so that x (and dy) are read once: bound by memory.  The
// variance is summed from the differences to the mean, never as a difference of
// two sums.  The backward pass needs two rounds of sums a row, two sums each:
// (x, g), then with the mean known ((x - m)^2, g (x - m)).  It works out the
// statistics again, which costs no memory, where keeping them would.
//
// Gradients of the parameters: a workgroup keeps the sums of its rows in
// registers, column by column, and writes them as one part; a second kernel adds
// the parts up in order, so that results do not depend on timing.
//
// Bound by memory: 32768 x 4096 bf16 97 us (5.5 TB/s, a copy reaches 5.2; fp32 204, 5.3),
// the gradients of 16384 x 4096 87 (4.6 TB/s, and 5 us of them the second kernel; fp32 152,
// 5.3).  Rows are read past the caches (stream.hpp).  A row's loads run during the sums of
// the one before, a row of the gradients from 2049 to 4096 elements has 512 threads, one run
// each, as two runs leave registers for two workgroups of four waves a CU, and of the
// forward pass, which has them, two runs of 256 (an earlier form of both kernels, without
// and with each: 149, 129 and 145, 125; 152, 125; 171, 129; two rows ahead 125).
//
// Slower: rows whose 1024 threads leave 128 registers a lane, of which the gradients spill
// some inside the loop (fp32 16384 x 8192 415 us, 3.9 TB/s; 8192 x 16384 442, bf16 256);
// and rows of fewer than 512 elements, whose 64 threads have eight each (2^20 x 64 bf16 346
// us, 0.8 TB/s, gradients 956; 2^18 x 512 98, 5.5 TB/s).
//
// Rows past 16384 elements go through memory (L2) once for each sum: the kernels
// named *_long.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "stream.hpp"

namespace xtc_hip {

struct NormArgs {
  const void* x;   // [rows][ldx]
  const void* dy;  // [rows][ldy]
  const void* w;   // [K]; w, b null: 1, 0
  const void* b;
  void* y;         // forward: [rows][ldy]; backward: dx [rows][ldx], or null
  float* parts;    // backward: [2][gridDim.x][K], or null
  float* stats;    // *_long: [rows][2], mean and 1 / deviation
  int64_t rows;
  int K, ldx, ldy;
  float eps;
};

namespace norm {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// 8 elements as stored
template <typename T>
struct Raw8 {
  T v[8];
};
// the first n of the 8 elements at p, zeros for the others.  ONCE: nobody reads them again
template <bool ONCE, typename T>
__device__ __forceinline__ void load8(Raw8<T>& r, const T* p, int n) {
  if (n >= 8) {
    if constexpr (ONCE) stream::load(r, p);
    else __builtin_memcpy(&r, p, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
  }
}
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, int n) {
  Raw8<T> r;
  load8<false>(r, p, n);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)r.v[i];
}

// v - mean, zeros past the first n
__device__ __forceinline__ void centre(float (&v)[8], float mean, int n) {
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] -= mean;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? v[i] - mean : 0.f;
  }
}

template <bool PAST = false, typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
  T out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = (T)v[i];
  if (n >= 8) {
    stream::store<PAST>(p, out);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = out[i];
  }
}

// Sums of a and b over the THREADS threads of a row, to all of them.  `at` is LDS of
// 2 (THREADS / 64) floats that no one reads any more: callers alternate between two,
// whose barriers part the readers of one from its next writers.
template <int THREADS>
__device__ __forceinline__ void row_sums(float& a, float& b, float* at) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) a += __shfl_xor(a, d), b += __shfl_xor(b, d);
  if constexpr (THREADS > 64) {
    constexpr int WAVES = THREADS / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) at[2 * wave] = a, at[2 * wave + 1] = b;
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) a += at[2 * i], b += at[2 * i + 1];
  }
}

}  // namespace norm

// y of the rows blockIdx.x, blockIdx.x + gridDim.x, .. (of ROWS at once).
template <typename T, typename P, int THREADS, int VECS>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) layer_norm(NormArgs p) {
  using namespace norm;
  constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1;
  __shared__ float lds[2][2 * (THREADS / 64)];
  const int t = threadIdx.x % THREADS;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  Raw8<T> raw[VECS];
  auto load = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int k = (i * THREADS + t) * 8;
      load8<true>(raw[i], (const T*)p.x + row * p.ldx + k, p.K - k);
    }
  };
  int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
  if (row < p.rows) load(row);
  float w[VECS][8], b[VECS][8];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int k = (i * THREADS + t) * 8;
    if (p.w) load8(w[i], (const P*)p.w + k, p.K - k);
    if (p.b) load8(b[i], (const P*)p.b + k, p.K - k);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[i][j] = p.w ? w[i][j] : 1.f, b[i][j] = p.b ? b[i][j] : 0.f;
  }
  // uniform over the threads of a row: with THREADS > 64 over the workgroup
  for (; row < p.rows; row += step) {
    float v[VECS][8];
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (float)raw[i].v[j], sum += v[i][j];
    if (row + step < p.rows) load(row + step);
    row_sums<THREADS>(sum, none, lds[0]);
    const float mean = sum / (float)p.K;
    float var = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      centre(v[i], mean, p.K - (i * THREADS + t) * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) var += v[i][j] * v[i][j];
    }
    row_sums<THREADS>(var, none, lds[1]);
    const float r = 1.0f / sqrtf(var / (float)p.K + p.eps);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int k = (i * THREADS + t) * 8;
      float out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = v[i][j] * r * w[i][j] + b[i][j];
      store8((T*)p.y + row * p.ldy + k, out, p.K - k);
    }
  }
}

// dx of the rows blockIdx.x, blockIdx.x + gridDim.x, .. (of ROWS at once), and this
// workgroup's part of dw and db.  PAST: dx is stored past the caches (a choice at run time
// between the two kinds of stores becomes one ordinary store).
template <bool PAST, typename T, typename P, int THREADS, int VECS>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) layer_norm_grad(NormArgs p) {
  using namespace norm;
  constexpr int ROWS = THREADS < 256 ? 256 / THREADS : 1;
  constexpr int WIDE = VECS * THREADS * 8;
  __shared__ float lds[2][2 * (THREADS / 64)];
  __shared__ float joined[ROWS > 1 ? 2 * ROWS * WIDE : 1];
  const int t = threadIdx.x % THREADS, sub = threadIdx.x / THREADS;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  float w[VECS][8], dw[VECS][8], db[VECS][8];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int k = (i * THREADS + t) * 8;
    if (p.w) load8(w[i], (const P*)p.w + k, p.K - k);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = db[i][j] = 0.f, w[i][j] = p.w ? w[i][j] : 1.f;
  }
  const float inv = 1.0f / (float)p.K;
  Raw8<T> raw_x[VECS], raw_dy[VECS];
  auto load = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int k = (i * THREADS + t) * 8;
      load8<true>(raw_x[i], (const T*)p.x + row * p.ldx + k, p.K - k);
      load8<true>(raw_dy[i], (const T*)p.dy + row * p.ldy + k, p.K - k);
    }
  };
  // the next row's loads are on their way during the sums of this one, where registers last
  constexpr bool AHEAD = THREADS * VECS <= 1024;
  int64_t row = (int64_t)blockIdx.x * ROWS + sub;
  if (AHEAD && row < p.rows) load(row);
  // uniform over the threads of a row: with THREADS > 64 over the workgroup
  for (; row < p.rows; row += step) {
    float x[VECS][8], dy[VECS][8], gr[VECS][8];
    float sum_x = 0.f, sum_g = 0.f;
    if (!AHEAD) load(row);
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[i][j] = (float)raw_x[i].v[j], dy[i][j] = (float)raw_dy[i].v[j];
        gr[i][j] = dy[i][j] * w[i][j];
        sum_x += x[i][j], sum_g += gr[i][j];
      }
    if (AHEAD && row + step < p.rows) load(row + step);
    row_sums<THREADS>(sum_x, sum_g, lds[0]);
    const float mean = sum_x / (float)p.K;
    float var = 0.f, cov = 0.f;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      centre(x[i], mean, p.K - (i * THREADS + t) * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) var += x[i][j] * x[i][j], cov += gr[i][j] * x[i][j];
    }
    row_sums<THREADS>(var, cov, lds[1]);
    const float r = 1.0f / sqrtf(var / (float)p.K + p.eps);
    const float c1 = r * (sum_g * inv), c2 = cov * r * inv;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      float out[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xh = x[i][j] * r;
        out[j] = r * (gr[i][j] - xh * c2) - c1;
        dw[i][j] += dy[i][j] * xh, db[i][j] += dy[i][j];
      }
      const int k = (i * THREADS + t) * 8;
      if (p.y) store8<PAST>((T*)p.y + row * p.ldx + k, out, p.K - k);
    }
  }
  if (!p.parts) return;
  if constexpr (ROWS > 1) {
    // the rows that ran side by side, in order
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = (i * THREADS + t) * 8 + j;
        joined[(2 * sub) * WIDE + k] = dw[i][j];
        joined[(2 * sub + 1) * WIDE + k] = db[i][j];
      }
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += 256) {
      float a = joined[k], c = joined[WIDE + k];
#pragma unroll
      for (int s = 1; s < ROWS; ++s) a += joined[2 * s * WIDE + k], c += joined[(2 * s + 1) * WIDE + k];
      p.parts[(size_t)blockIdx.x * p.K + k] = a;
      p.parts[((size_t)gridDim.x + blockIdx.x) * p.K + k] = c;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int k = (i * THREADS + t) * 8;
      store8(p.parts + (size_t)blockIdx.x * p.K + k, dw[i], p.K - k);
      store8(p.parts + ((size_t)gridDim.x + blockIdx.x) * p.K + k, db[i], p.K - k);
    }
  }
}

// dw and db (blockIdx.y 0 and 1; either may be null) from `parts` parts: 64 columns
// a workgroup, its 16 waves take every 16th part, eight at once, and their sums are added
// in order.  It waits for its loads: with four waves 512 parts of 4096 took 6.6 us.
static __global__ void __launch_bounds__(1024) layer_norm_grad_sum(const float* from, float* dw, float* db, int parts, int K) {
  constexpr int N = 16, EACH = 8;
  __shared__ float lds[N][64];
  float* const to = blockIdx.y ? db : dw;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int k = blockIdx.x * 64 + lane;
  if (!to) return;
  const float* const at = from + (size_t)blockIdx.y * parts * K + min(k, K - 1);
  float sum = 0.f;
  for (int i = wave; i < parts; i += N * EACH) {
    float v[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) v[j] = at[(size_t)min(i + N * j, parts - 1) * K];
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += i + N * j < parts ? v[j] : 0.f;
  }
  lds[wave][lane] = sum;
  __syncthreads();
  if (wave || k >= K) return;
  for (int w = 1; w < N; ++w) sum += lds[w][lane];
  to[k] = sum;
}

// ---- rows past the registers: a workgroup a row, which it walks once for each sum

template <typename T, typename P, bool GRAD>
__global__ void __launch_bounds__(1024) layer_norm_long(NormArgs p) {
  using namespace norm;
  __shared__ float lds[2][2 * 16];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* const x = (const T*)p.x + row * p.ldx;
    const T* const dy = (const T*)p.dy + row * p.ldy;
    float sum_x = 0.f, sum_g = 0.f;
    for (int64_t k = 8 * threadIdx.x; k < p.K; k += 8192) {
      const int n = p.K - (int)k;
      float v[8], d[8], w[8];
      load8(v, x + k, n);
      if (GRAD) load8(d, dy + k, n);
      if (GRAD && p.w) load8(w, (const P*)p.w + k, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum_x += v[j];
        if (GRAD) sum_g += d[j] * (p.w ? w[j] : 1.f);
      }
    }
    row_sums<1024>(sum_x, sum_g, lds[0]);
    const float mean = sum_x / (float)p.K;
    float var = 0.f, cov = 0.f;
    for (int64_t k = 8 * threadIdx.x; k < p.K; k += 8192) {
      const int n = p.K - (int)k;
      float v[8], d[8], w[8];
      load8(v, x + k, n);
      if (GRAD) load8(d, dy + k, n);
      if (GRAD && p.w) load8(w, (const P*)p.w + k, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = j < n ? v[j] - mean : 0.f;
        var += c * c;
        if (GRAD) cov += d[j] * (p.w ? w[j] : 1.f) * c;
      }
    }
    row_sums<1024>(var, cov, lds[1]);
    const float r = 1.0f / sqrtf(var / (float)p.K + p.eps), c1 = sum_g / (float)p.K, c2 = cov * r / (float)p.K;
    if (GRAD && p.stats && threadIdx.x == 0) p.stats[2 * row] = mean, p.stats[2 * row + 1] = r;
    if (!p.y) continue;
    for (int64_t k = 8 * threadIdx.x; k < p.K; k += 8192) {
      const int n = p.K - (int)k;
      float v[8], d[8], w[8], b[8], out[8];
      load8(v, x + k, n);
      if (GRAD) load8(d, dy + k, n);
      if (p.w) load8(w, (const P*)p.w + k, n);
      if (!GRAD && p.b) load8(b, (const P*)p.b + k, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float xh = (v[j] - mean) * r, wj = p.w ? w[j] : 1.f;
        out[j] = GRAD ? r * (d[j] * wj - c1 - xh * c2) : xh * wj + (p.b ? b[j] : 0.f);
      }
      store8((T*)p.y + row * (GRAD ? p.ldx : p.ldy) + k, out, n);
    }
  }
}

// dw and db of long rows from their statistics: 2048 columns (blockIdx.y), the rows of
// part blockIdx.x.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_grad_columns(NormArgs p) {
  using namespace norm;
  const int64_t k = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
  if (k >= p.K) return;
  const int n = (int)(p.K - k);
  float dw[8] = {}, db[8] = {};
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.stats[2 * row], r = p.stats[2 * row + 1];
    float v[8], d[8];
    load8(v, (const T*)p.x + row * p.ldx + k, n);
    load8(d, (const T*)p.dy + row * p.ldy + k, n);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[j] += d[j] * ((v[j] - mean) * r), db[j] += d[j];
  }
  store8(p.parts + (size_t)blockIdx.x * p.K + k, dw, n);
  store8(p.parts + ((size_t)gridDim.x + blockIdx.x) * p.K + k, db, n);
}

}  // namespace xtc_hip
