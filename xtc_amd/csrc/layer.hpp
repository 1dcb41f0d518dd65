// SPDX-License-Identifier: BSD-3-Clause
// A whole layer of experts for a few tokens (T <= 64):
//   l = x R^T; of the top_k largest l of a token (ties: the lowest expert)
//   y = sum over its experts e of p_e D_e act(U_e x),  p = softmax(l)
// with the p divided by their sum or not.  act is relu, or silu of U's first H rows
// times its last H rows.  Matrices are stored [out][in], in the type of x, or of bf16 x
// as 8-bit floats in blocks of 128 x 128 (fp8.hpp) or 4-bit ones in blocks of 32
// (mx4.hpp), whose values are bf16 numbers: activations keep their precision.
//
// The cost is reading the chosen experts' matrices once.  Two launches:
//   layer_up    a workgroup takes one expert and a slice of its rows; it works out the
//               choice for all tokens by itself (so no launch has to pass it on),
//               gathers the tokens that chose its expert, and writes p_e act(U_e x) to
//               the place (token, rank of e in its choice) of the workspace
//   layer_down  the same for D_e; the last workgroup of a slice to arrive adds up the
//               experts of every token in the order of their ranks (splitk.hpp's
//               protocol: results do not depend on who is last)
// Where router and tokens are long (more than layer_up's workgroups should each read
// again from L2), layer_logits works the logits out first, in parts of k.
//
// A workgroup is eight waves that share out k in turn.  k may be summed in any order as
// long as matrix and token agree, so a lane takes 32 neighbouring elements of its row
// (16 of fp32): 64, 32 or 16 bytes, four v_mfma_f32_16x16x32_bf16 (or sixteen
// v_mfma_f32_16x16x4_f32).  The matrix is the first MFMA operand: a lane ends with four
// neighbouring rows of one token.  The waves' sums are added up in LDS, in order.
//
// The down product's operand is kept in two bf16 numbers (value and rest, 16 bits in
// all), multiplied one after the other: rounding it to one would cost as much
// precision as rounding the result does, where the MFMAs wait for memory anyway.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fp8.hpp"
#include "gemm_bf16_lds.hpp"
#include "splitk.hpp"

namespace xtc_hip {

struct LayerArgs {
  const void* x;       // [T][ldx]
  const void* router;  // [E][K]
  const void *up, *down;
  const uint8_t *up_scales, *down_scales;
  // workspace
  void* mid;           // [T top_k] rows: 2 planes of Hp bf16, or Hp fp32
  float* parts;        // [T top_k][K]
  float* logits;       // [logit_parts][T][E], or null: layer_up works them out
  int* choice;         // [T][top_k]
  unsigned* counters;  // [slices of layer_down]
  void* y;             // [T][ldy]
  int T, E, K, H, Hp, top_k, ldx, ldy;
  int normalize, swiglu;
  int logit_parts;
  int by_slot;         // workgroups per (token, rank) rather than per expert
  int slices;          // of the launch's rows
};

namespace layer {

using big::bf16x8;
using big::f32x4;
using big::u32x4;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

enum Format { F32 = 0, BF16 = 1, FP8 = 2, MX4 = 3 };

constexpr int WAVES = 8;
constexpr int LOGITS = 4096;  // of a round of the choice, in LDS

// ---- runs of a row: UNIT elements a lane

// Elements [k, k + 8) of a row of n elements, zeros past it
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* row, int k, int n) {
  constexpr int V = 16 / sizeof(T);
  u32x4 v = {0, 0, 0, 0};
  if (k + V <= n) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < n) {
    T raw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = k + i < n ? row[k + i] : (T)0.f;
    __builtin_memcpy(&v, raw, 16);
  }
  return v;
}

// A run of a matrix row as stored
template <int F> struct Raw;
template <> struct Raw<F32> { u32x4 v[4]; };
template <> struct Raw<BF16> { u32x4 v[4]; };
template <> struct Raw<FP8> { u32x4 v[2]; int s; };
template <> struct Raw<MX4> { u32x4 v[1]; int s; };

// One matrix row: its runs, `unit` elements each
template <int F> struct Row;
template <> struct Row<F32> {
  static constexpr int UNIT = 16;
  const float* p;
  int n;
  __device__ __forceinline__ Row(const void* w, const uint8_t*, int64_t e, int rows, int r, int depth) : p((const float*)w + (e * rows + r) * depth), n(depth) {}
  __device__ __forceinline__ void load(Raw<F32>& q, int u) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = load16(p, u * 16 + 4 * i, n);
  }
};
template <> struct Row<BF16> {
  static constexpr int UNIT = 32;
  const __bf16* p;
  int n;
  __device__ __forceinline__ Row(const void* w, const uint8_t*, int64_t e, int rows, int r, int depth) : p((const __bf16*)w + (e * rows + r) * depth), n(depth) {}
  __device__ __forceinline__ void load(Raw<BF16>& q, int u) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) q.v[i] = load16(p, u * 32 + 8 * i, n);
  }
};
template <> struct Row<FP8> {
  static constexpr int UNIT = 32;
  const uint8_t *p, *s;
  int units;
  __device__ __forceinline__ Row(const void* w, const uint8_t* scales, int64_t e, int rows, int r, int depth) {
    const int blocks = (depth + 127) / 128;
    p = (const uint8_t*)w + (e * rows + r) * blocks * 128;
    s = scales + (e * ((rows + 127) / 128) + r / 128) * blocks;
    units = 4 * blocks;
  }
  __device__ __forceinline__ void load(Raw<FP8>& q, int u) const {
    if (u < units) {
      q.v[0] = *(const u32x4*)(p + 32 * (int64_t)u), q.v[1] = *(const u32x4*)(p + 32 * (int64_t)u + 16);
      q.s = s[u >> 2];
    } else {
      q.v[0] = q.v[1] = u32x4{0, 0, 0, 0}, q.s = 127;
    }
  }
};
template <> struct Row<MX4> {
  static constexpr int UNIT = 32;
  const uint8_t *p, *s;
  int units;
  __device__ __forceinline__ Row(const void* w, const uint8_t* scales, int64_t e, int rows, int r, int depth) {
    units = (depth + 31) / 32;
    p = (const uint8_t*)w + (e * rows + r) * units * 16;
    s = scales + (e * rows + r) * units;
  }
  __device__ __forceinline__ void load(Raw<MX4>& q, int u) const {
    if (u < units) q.v[0] = *(const u32x4*)(p + 16 * (int64_t)u), q.s = s[u];
    else q.v[0] = u32x4{0, 0, 0, 0}, q.s = 127;
  }
};

__device__ __forceinline__ unsigned bits(bf16x2 v) { return __builtin_bit_cast(unsigned, v); }

// Elements 8 i .. 8 i + 7 of a run as bf16 numbers: exact, as scales are powers of two
__device__ __forceinline__ bf16x8 fragment(const Raw<BF16>& q, int i) { return __builtin_bit_cast(bf16x8, q.v[i]); }
__device__ __forceinline__ bf16x8 fragment(const Raw<FP8>& q, int i) {
  const bf16x8 v = fp8::values_bf16(q.v[i >> 1][2 * (i & 1)], q.v[i >> 1][2 * (i & 1) + 1], mx4::scale_value(q.s));
  return q.s == 255 ? __builtin_bit_cast(bf16x8, u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}) : v;
}
__device__ __forceinline__ bf16x8 fragment(const Raw<MX4>& q, int i) {
  const float scale = mx4::scale_value(q.s);
  const unsigned w = q.v[0][i];
  u32x4 v = {bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
             bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)), bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
  if (q.s == 255) v = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  return __builtin_bit_cast(bf16x8, v);
}

// acc += run of matrix rows times run of tokens
template <int F>
__device__ __forceinline__ f32x4 multiply(const Raw<F>& w, const u32x4 (&x)[4], f32x4 c) {
  if constexpr (F == F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.v[i][j]), __uint_as_float(x[i][j]), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fragment(w, i), __builtin_bit_cast(bf16x8, x[i]), c, 0, 0, 0);
  }
  return c;
}

// ---- the choice

// An order of the numbers in which the two zeros are one and NaN comes before all
__device__ __forceinline__ unsigned key(float v) {
  const unsigned u = __float_as_uint(v + 0.f);
  return v != v ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}

struct Choice {
  int e[64 * 16];       // [T][top_k]
  float p[64 * 16];
};

// The experts of every token and their weights, from the logits; eight lanes a token.
// `logits` is LDS of LOGITS floats.
template <typename GetRound>
__device__ __forceinline__ void choose(const LayerArgs& p, Choice& c, float* logits, GetRound&& fill) {
  const int round = min(LOGITS / p.E, 64);  // tokens at once
  const int sub = threadIdx.x & 7;
  for (int t0 = 0; t0 < p.T; t0 += round) {
    const int tokens = min(round, p.T - t0);
    __syncthreads();
    fill(t0, tokens);
    __syncthreads();
    const int t = threadIdx.x >> 3;
    if (t >= tokens) continue;
    const float* const l = logits + t * p.E;
    float top = 0.f, total = 0.f, picked = 0.f;
    uint32_t taken = 0;  // of the experts sub, sub + 8, ..: at most 32
    for (int j = 0; j < p.top_k; ++j) {
      unsigned best = 0;
      int at = 0x7fffffff;
      for (int i = sub, b = 0; i < p.E; i += 8, ++b) {
        const unsigned k = key(l[i]);
        if (!(taken >> b & 1) && (k > best || at == 0x7fffffff)) best = k, at = i;
      }
#pragma unroll
      for (int d = 1; d < 8; d *= 2) {
        const unsigned ob = (unsigned)__shfl_xor((int)best, d);
        const int oa = __shfl_xor(at, d);
        if (oa != 0x7fffffff && (at == 0x7fffffff || ob > best || (ob == best && oa < at))) best = ob, at = oa;
      }
      if ((at & 7) == sub) taken |= 1u << (at >> 3);
      const float v = l[at];
      if (j == 0) top = v;
      const float share = expf(v - top);
      picked += share;
      if (sub == 0) c.e[(t0 + t) * p.top_k + j] = at, c.p[(t0 + t) * p.top_k + j] = share;
    }
    for (int i = sub; i < p.E; i += 8) total += expf(l[i] - top);  // NaN where one is
#pragma unroll
    for (int d = 1; d < 8; d *= 2) total += __shfl_xor(total, d);
    const float by = 1.f / (p.normalize && total == total ? picked : total);
    if (sub == 0)
      for (int j = 0; j < p.top_k; ++j) c.p[(t0 + t) * p.top_k + j] *= by;
  }
  __syncthreads();
}

// The expert of workgroup column `a` and the places (token top_k + rank) that chose it,
// into `places`; how many, 0 where another workgroup has this expert.
__device__ __forceinline__ int gather(const LayerArgs& p, const int* chosen, int a, int* places, int& e) {
  const int slots = p.T * p.top_k, lane = threadIdx.x & 63;
  e = p.by_slot ? chosen[a] : a;
  int n = 0;
  for (int s0 = 0; s0 < slots; s0 += 64) {
    const int s = s0 + lane;
    const bool hit = s < slots && chosen[s] == e;
    const uint64_t hits = __ballot(hit);
    if (hit && threadIdx.x < 64) places[n + __popcll(hits & (((uint64_t)1 << lane) - 1))] = s;
    if (p.by_slot && s0 <= a && hits) {
      const int first = s0 + __builtin_ctzll(hits);
      if (first < a && n == 0) return 0;  // an earlier place has it
    }
    n += __popcll(hits);
  }
  __syncthreads();
  return n;
}

// acc[j][i]: 16 matrix rows j times 16 tokens i, this wave's share of the depth.
// `token(i, k)` gives the token run's 16 bytes at element k.
template <int F, int TM, int TN, int PLANES, typename LoadX>
__device__ __forceinline__ void product(f32x4 (&acc)[TN][TM], const Row<F> (&rows)[TN], int depth, int tiles, LoadX&& load_x) {
  constexpr int UNIT = Row<F>::UNIT;
  const int wave = threadIdx.x >> 6, g = (threadIdx.x & 63) >> 4;
  const int units = (depth + UNIT - 1) / UNIT;
  Raw<F> w[2][TN];
  auto load_w = [&](int buf, int u) {
#pragma unroll
    for (int j = 0; j < TN; ++j) rows[j].load(w[buf][j], u);
  };
  const int u0 = 4 * wave + g, step = 4 * WAVES;
  const int steps = (units - 4 * wave + step - 1) / step;  // of this wave
  if (steps > 0) load_w(0, u0);
  for (int s = 0; s < steps; s += 2) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (s + q >= steps) break;
      const int u = u0 + (s + q) * step;
      u32x4 x[PLANES][TM][4];
#pragma unroll
      for (int i = 0; i < TM; ++i)
        if (i < tiles)
#pragma unroll
          for (int h = 0; h < PLANES; ++h) load_x(x[h][i], i, h, u * UNIT);
      if (s + q + 1 < steps) load_w(1 - q, u + step);
#pragma unroll
      for (int i = 0; i < TM; ++i)
        if (i < tiles)
#pragma unroll
          for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int h = 0; h < PLANES; ++h) acc[j][i] = multiply<F>(w[q][j], x[h][i], acc[j][i]);
    }
  }
}

template <int TM, int TN>
struct Sums {
  float v[WAVES][TN * 16][16 * TM + 1];
};

template <int TM, int TN>
__device__ __forceinline__ void put(Sums<TM, TN>& sums, const f32x4 (&acc)[TN][TM]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums.v[wave][16 * j + 4 * (lane >> 4) + r][16 * i + (lane & 15)] = acc[j][i][r];
}
template <int TM, int TN>
__device__ __forceinline__ float total(const Sums<TM, TN>& sums, int row, int token) {
  float v = sums.v[0][row][token];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v += sums.v[w][row][token];
  return v;
}

template <int F> struct Type { typedef __bf16 type; };
template <> struct Type<F32> { typedef float type; };

}  // namespace layer

// logits[part][t][e] of 16 tokens and 16 experts, part of k: blockIdx.x, .y, .z
template <typename T>
__global__ void __launch_bounds__(512) layer_logits(LayerArgs p) {
  using namespace layer;
  constexpr int F = sizeof(T) == 4 ? F32 : BF16, UNIT = Row<F>::UNIT;
  __shared__ Sums<1, 1> sums;
  const int l16 = threadIdx.x & 15;
  const int t0 = blockIdx.x * 16, e0 = blockIdx.y * 16;
  // whole runs of a part
  const int units = (p.K + UNIT - 1) / UNIT;
  const int from = (int)((int64_t)units * blockIdx.z / gridDim.z) * UNIT;
  const int depth = min((int)((int64_t)units * (blockIdx.z + 1) / gridDim.z) * UNIT, p.K) - from;
  const T* const x = (const T*)p.x + (int64_t)min(t0 + l16, p.T - 1) * p.ldx + from;
  Row<F> rows[1] = {Row<F>(p.router, nullptr, 0, p.E, min(e0 + l16, p.E - 1), p.K)};
  rows[0].p += from, rows[0].n = depth;
  f32x4 acc[1][1] = {};
  product<F, 1, 1, 1>(acc, rows, depth, 1, [&](u32x4 (&v)[4], int, int, int k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = load16(x, k + (UNIT / 4) * i, depth);
  });
  put(sums, acc);
  __syncthreads();
  const int e = threadIdx.x & 15, t = threadIdx.x >> 4;
  if (t < 16 && t0 + t < p.T && e0 + e < p.E) p.logits[((int64_t)blockIdx.z * p.T + t0 + t) * p.E + e0 + e] = total(sums, e, t);
}

// p act(U x) of one expert's tokens, rows [slice, slice + ROWS) of H
template <int F, int TM, int TN, bool SWIGLU>
__global__ void __launch_bounds__(512) layer_up(LayerArgs p) {
  using namespace layer;
  typedef typename Type<F>::type T;
  constexpr int UNIT = Row<F>::UNIT, ROWS = SWIGLU ? 8 * TN : 16 * TN;
  __shared__ union {
    Sums<TM, TN> sums;
    Sums<1, 1> logit_sums;
  } lds;
  __shared__ float logits[LOGITS];
  __shared__ Choice choice;
  __shared__ int places[64];
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int slice = blockIdx.x % p.slices, a = blockIdx.x / p.slices;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < (p.K + 15) / 16; i += 512) p.counters[i] = 0;

  choose(p, choice, logits, [&](int t0, int tokens) {
    if (p.logits) {
      for (int i = threadIdx.x; i < tokens * p.E; i += 512) {
        float v = 0.f;
        for (int s = 0; s < p.logit_parts; ++s) v += p.logits[((int64_t)s * p.T + t0) * p.E + i];
        logits[i] = v;
      }
      return;
    }
    // T E <= LOGITS: one round; 16 experts and 16 tokens after the other
    constexpr int FR = sizeof(T) == 4 ? F32 : BF16, UR = Row<FR>::UNIT;
    const int et = (p.E + 15) / 16, pairs = et * ((p.T + 15) / 16);
    for (int q = 0; q < pairs; ++q) {
      const int ce = q % et * 16, ct = q / et * 16;
      const T* const x = (const T*)p.x + (int64_t)min(ct + l16, p.T - 1) * p.ldx;
      const Row<FR> rows[1] = {Row<FR>(p.router, nullptr, 0, p.E, min(ce + l16, p.E - 1), p.K)};
      f32x4 acc[1][1] = {};
      product<FR, 1, 1, 1>(acc, rows, p.K, 1, [&](u32x4 (&v)[4], int, int, int k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = load16(x, k + (UR / 4) * i, p.K);
      });
      __syncthreads();
      put(lds.logit_sums, acc);
      __syncthreads();
      const int e = ce + (threadIdx.x & 15), t = ct + (threadIdx.x >> 4);
      if (threadIdx.x < 256 && e < p.E && t < p.T) logits[t * p.E + e] = total(lds.logit_sums, threadIdx.x & 15, threadIdx.x >> 4);
    }
  });

  int e;
  const int n = gather(p, choice.e, a, places, e);
  if (n == 0) return;
  if (slice == 0 && (int)threadIdx.x < n) p.choice[places[threadIdx.x]] = e;

  const int n0 = slice * ROWS;
  for (int at = 0; at < n; at += 16 * TM) {
    const int tokens = min(n - at, 16 * TM), tiles = (tokens + 15) / 16;
    const T* x[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = (const T*)p.x + (int64_t)(places[min(at + 16 * i + l16, n - 1)] / p.top_k) * p.ldx;
    f32x4 acc[TN][TM] = {};
    // rows past the last one repeat it and are not kept
    auto row = [&](int j) {
      const int half = SWIGLU ? j / (TN / 2) : 0, r = n0 + 16 * (SWIGLU ? j % (TN / 2) : j) + l16;
      return Row<F>(p.up, p.up_scales, e, SWIGLU ? 2 * p.H : p.H, half * p.H + min(r, p.H - 1), p.K);
    };
    auto run = [&](const Row<F> (&rows)[TN]) {
      product<F, TM, TN, 1>(acc, rows, p.K, tiles, [&](u32x4 (&v)[4], int i, int, int k) {
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = load16(x[i], k + (UNIT / 4) * c, p.K);
      });
    };
    if constexpr (TN == 2) run({row(0), row(1)});
    else run({row(0), row(1), row(2), row(3)});
    __syncthreads();  // the last sums have been read
    put(lds.sums, acc);
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * ROWS; i += 512) {
      const int r = i % ROWS, t = i / ROWS;
      if (n0 + r >= p.Hp) continue;
      float h = 0.f;
      if (n0 + r < p.H) {
        h = total(lds.sums, r, t);
        if (SWIGLU) h = h / (1.f + expf(-h)) * total(lds.sums, r + 8 * TN, t);
        else h = h < 0.f ? 0.f : h;
        h *= choice.p[places[at + t]];
      }
      const int64_t to = (int64_t)places[at + t] * p.Hp;
      if constexpr (F == F32) {
        ((float*)p.mid)[to + n0 + r] = h;
      } else {
        const __bf16 hi = (__bf16)h;
        ((__bf16*)p.mid)[2 * to + n0 + r] = hi;
        ((__bf16*)p.mid)[2 * to + p.Hp + n0 + r] = (__bf16)(__builtin_isinf((float)hi) ? 0.f : h - (float)hi);
      }
    }
  }
}

// D of one expert's tokens, rows [slice, slice + 16 TN) of K, and the sum over a token's
// experts by the last workgroup of a slice
template <int F, int TM, int TN>
__global__ void __launch_bounds__(512) layer_down(LayerArgs p) {
  using namespace layer;
  typedef typename Type<F>::type T;
  constexpr int UNIT = Row<F>::UNIT, ROWS = 16 * TN, PLANES = F == F32 ? 1 : 2;
  __shared__ Sums<TM, TN> sums;
  __shared__ int chosen[64 * 16];
  __shared__ int places[64];
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int slice = blockIdx.x % p.slices, a = blockIdx.x / p.slices;
  const int slots = p.T * p.top_k, n0 = slice * ROWS, rows_here = min(ROWS, p.K - n0);
  for (int i = threadIdx.x; i < slots; i += 512) chosen[i] = p.choice[i];
  __syncthreads();
  int e;
  const int n = gather(p, chosen, a, places, e);
  for (int at = 0; at < n; at += 16 * TM) {
    const int tokens = min(n - at, 16 * TM), tiles = (tokens + 15) / 16;
    const T* x[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = (const T*)p.mid + (int64_t)places[min(at + 16 * i + l16, n - 1)] * (PLANES * p.Hp);
    f32x4 acc[TN][TM] = {};
    auto row = [&](int j) { return Row<F>(p.down, p.down_scales, e, p.K, min(n0 + 16 * j + l16, p.K - 1), p.H); };
    auto run = [&](const Row<F> (&rows)[TN]) {
      product<F, TM, TN, PLANES>(acc, rows, p.H, tiles, [&](u32x4 (&v)[4], int i, int h, int k) {
        // rows are Hp long, zeros past H
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = k < p.Hp ? *(const u32x4*)(x[i] + h * p.Hp + k + (UNIT / 4) * c) : u32x4{0, 0, 0, 0};
      });
    };
    if constexpr (TN == 2) run({row(0), row(1)});
    else run({row(0), row(1), row(2), row(3)});
    __syncthreads();
    put(sums, acc);
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * ROWS; i += 512) {
      const int r = i % ROWS, t = i / ROWS;
      if (r < rows_here) splitk_store(p.parts + (int64_t)places[at + t] * p.K + n0 + r, total(sums, r, t));
    }
  }
  if (!splitk_arrive(p.counters + slice, (int)gridDim.x / p.slices)) return;
  for (int i = threadIdx.x; i < p.T * ROWS; i += 512) {
    const int r = i % ROWS, t = i / ROWS;
    if (r >= rows_here) continue;
    ((T*)p.y)[(int64_t)t * p.ldy + n0 + r] = (T)splitk_sum1(p.parts + (int64_t)t * p.top_k * p.K + n0 + r, (size_t)p.K, p.top_k);
  }
}

// The two launches.
struct LayerGrid {
  bool wide;  // slices of four tiles of rows, or of two
  bool two;   // tiles of tokens at once, or one
  int up_slices, down_slices, columns;
};
// Each of a translation unit of its own: layer_f32.hip, layer_bf16.hip, ..
template <int F>
void layer_launch(const LayerArgs& a, const LayerGrid& g, hipStream_t s);

template <int F, int TM, int TN>
void layer_launch_tiles(const LayerArgs& a, const LayerGrid& g, hipStream_t s) {
  LayerArgs u = a, d = a;
  u.slices = g.up_slices, d.slices = g.down_slices;
  const dim3 up((unsigned)(g.up_slices * g.columns)), down((unsigned)(g.down_slices * g.columns));
  if (a.swiglu) hipLaunchKernelGGL((layer_up<F, TM, TN, true>), up, dim3(512), 0, s, u);
  else hipLaunchKernelGGL((layer_up<F, TM, TN, false>), up, dim3(512), 0, s, u);
  hipLaunchKernelGGL((layer_down<F, TM, TN>), down, dim3(512), 0, s, d);
}
#define XTC_HIP_LAYER_LAUNCH(F)                                                              \
  template <>                                                                                \
  void layer_launch<F>(const LayerArgs& a, const LayerGrid& g, hipStream_t s) {              \
    if (g.wide) g.two ? layer_launch_tiles<F, 2, 4>(a, g, s) : layer_launch_tiles<F, 1, 4>(a, g, s); \
    else g.two ? layer_launch_tiles<F, 2, 2>(a, g, s) : layer_launch_tiles<F, 1, 2>(a, g, s);      \
  }
template <> void layer_launch<layer::F32>(const LayerArgs&, const LayerGrid&, hipStream_t);
template <> void layer_launch<layer::BF16>(const LayerArgs&, const LayerGrid&, hipStream_t);
template <> void layer_launch<layer::FP8>(const LayerArgs&, const LayerGrid&, hipStream_t);
template <> void layer_launch<layer::MX4>(const LayerArgs&, const LayerGrid&, hipStream_t);

}  // namespace xtc_hip
