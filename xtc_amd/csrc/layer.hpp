// SPDX-License-Identifier: BSD-3-Clause
// A whole layer of experts for a few tokens (T <= 64):
//   l = x R^T; of the top_k largest l of a token (ties: the lowest expert)
//   y = sum over its experts e of p_e D_e act(U_e x),  p = softmax(l)
// with the p divided by their sum or not.  act is relu, or silu of U's first H rows
// times its last H rows.  Matrices are stored [out][in], in the type of x, or of bf16 x
// as 8-bit floats in blocks of 128 x 128 (fp8.hpp) or 4-bit ones in blocks of 32
// (mx4.hpp), whose values are bf16 numbers (8-bit scale bytes from 3 to 246, 4-bit ones up
// to 252): activations keep their precision.
//
// The cost is reading the chosen experts' matrices once.  Two launches:
//   layer_up    every workgroup works out the choice for all tokens by itself (so no
//               launch has to pass it on), then walks over pieces of work, each some
//               rows of one chosen expert: it gathers the tokens that chose it and
//               writes p_e act(U_e x) to the place (token, rank of e in its choice) of
//               the workspace
//   layer_down  the same for D_e; the last workgroup that brings a slice of rows adds up
//               the experts of every token in the order of their ranks (splitk.hpp's
//               protocol: results do not depend on who is last)
// Where router and tokens are long (more than every workgroup of layer_up should read
// again from L2), layer_logits works the logits out first, in parts of k.
//
// A workgroup is four waves, and as many workgroups as the CUs hold walk over the pieces.
// The four share out k in turn and add their sums up in LDS, in order (DEPTH 4); for packed
// matrices of many rows two do (DEPTH 2), which halves the tokens' trips through LDS.  k may
// be summed in any order as long as matrix and token agree, so the four lanes of a row read
// 64 neighbouring bytes of it with an instruction, and a step takes 256.  The matrix is the first MFMA operand: a lane ends with four neighbouring rows
// of one token.  A tile of 16 rows of U holds 8 of its first half and the 8 of the second
// that these are multiplied with, 32 lanes away.
//
// Bound by the matrices where there are many (16 tokens, 4 of 64 experts of 2048/1024 in
// 8 bits: 40 us and 20, 4 TB/s, 24 with fp32 activations), and by latency else: a token at 2
// of 8 experts of 1024/2048 in bf16 10 us and 7 (8), of which starting, logits and choice
// are 6; 64 tokens at 2 of 16 of 4096/2048 in 4 bits 28 and 31 (53).
//
// The activations p_e act(U_e x) between the two products: fp32, or as the caller has it
// rounded to bf16 where x is bf16, which is what the second product's instructions take.
// An fp32 number is the sum of three bf16 ones, its bits in turn, and layer_down
// multiplies each matrix fragment by all three (PLANES 3).  The 16 rows of tokens in LDS
// then hold five tokens, or 32 rows of half the length ten.  Whole calls, us, rounded and
// in fp32: few tokens an expert 18.5, 19.6 (a token at 2 of 8 of 1024/2048 in bf16) and
// 72.6, 74.9 (16 at 4 of 64 of 2048/1024 in 8 bits), eight 64, 82 (64 at 2 of 16 of
// 4096/2048 in 4 bits: three times the MFMAs and LDS reads, stretches of half the length),
// 32 61, 103 (64 at 2 of 4 of 2048/2048 in 8 bits: four passes over a matrix instead of
// two).  With the planes read from L2 into registers instead of LDS: 19.8, 85.7, 86.9.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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
  void* mid;           // [T top_k][planes][Hp] of x's type
  float* parts;        // [T top_k][K]
  float* logits;       // [logit_parts][T][E], or null: layer_up works them out
  int* choice;         // [T][top_k]
  unsigned* counters;  // [slices of layer_down]
  void* y;             // [T][ldy]
  int T, E, K, H, Hp, top_k, ldx, ldy;
  int normalize, swiglu;
  int planes;          // bf16 numbers that add up to an activation: 1 or 3
  int logit_parts;
  int slices;          // of the launch's rows
};

namespace layer {

using big::bf16x8;
using big::f32x4;
using big::u32x4;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

enum Format { F32 = 0, BF16 = 1, FP8 = 2, MX4 = 3 };

constexpr int WAVES = 4, THREADS = 64 * WAVES;

// This thread's wave, known to be the same for all of its lanes
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

constexpr int LOGITS = 4096;         // of a round of the choice, in LDS
constexpr int ROUND = THREADS / 8;   // tokens of a round, at most

// ---- runs of a row: UNIT elements a lane

// 16 bytes from element k of a row of n elements, zeros past it
template <typename T>
__device__ __forceinline__ u32x4 load16(const T* row, int k, int n) {
  constexpr int V = 16 / sizeof(T);
  u32x4 v = {0, 0, 0, 0};
  if (k + V <= n) __builtin_memcpy(&v, row + k, 16);
  if (n % V != 0 && k < n && k + V > n) {
    unsigned __int128 w = 0;
    if (n >= V) {
      // the row's last 16 bytes, without those before k
      __builtin_memcpy(&w, row + (n - V), 16);
      w >>= 8 * (int)sizeof(T) * (k + V - n);
    } else {
#pragma unroll 1
      for (int i = n - 1; i >= k; --i) {
        uint32_t x = 0;
        __builtin_memcpy(&x, row + i, sizeof(T));
        w = w << (8 * sizeof(T)) | x;
      }
    }
    __builtin_memcpy(&v, &w, 16);
  }
  return v;
}

// Lane g's 16 bytes of the four places of the step at element k
template <typename T>
__device__ __forceinline__ void load_step(u32x4 (&v)[4], const T* row, int k, int g, int n) {
  constexpr int V = 16 / sizeof(T);
  k = __builtin_amdgcn_readfirstlane(k);  // a step is a whole wave's
  if (k + 16 * V <= n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) __builtin_memcpy(&v[i], row + k + V * (4 * i + g), 16);
  } else {
    asm volatile("" : "+s"(k));  // a pointer for every place would take the loop's registers
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = load16(row, k + V * (4 * i + g), n);
  }
}

// A step of a matrix row is 256 bytes, of which lane g of the row's four holds bytes 64 i +
// 16 g: an instruction reads 64 neighbouring bytes of every row
template <int F>
struct Raw {
  u32x4 v[4];
  u32x4 s;  // scales: of 8-bit elements s[0] for i < 2 and s[1], of 4-bit ones byte g of s[i]
};

// One matrix row: its steps, STEP elements each.  Elements at step s, place i: s STEP + i
// STEP / 4 + g STEP / 16 ..
template <int F> struct Row;
template <typename T>
struct DenseRow {
  static constexpr int STEP = 256 / sizeof(T);
  const T* p;
  int n;
  __device__ __forceinline__ DenseRow(const void* w, const uint8_t*, int64_t e, int rows, int r, int depth) : p((const T*)w + (e * rows + r) * depth), n(depth) {}
  template <int F>
  __device__ __forceinline__ void load(Raw<F>& q, int s, int g) const { load_step(q.v, p, s * STEP, g, n); }
};
template <> struct Row<F32> : DenseRow<float> { using DenseRow::DenseRow; };
template <> struct Row<BF16> : DenseRow<__bf16> { using DenseRow::DenseRow; };
template <> struct Row<FP8> {
  static constexpr int STEP = 256;
  const uint8_t *p, *s;
  int blocks;
  __device__ __forceinline__ Row(const void* w, const uint8_t* scales, int64_t e, int rows, int r, int depth) {
    blocks = (depth + 127) / 128;
    p = (const uint8_t*)w + (e * rows + r) * blocks * 128;
    s = scales + (e * ((rows + 127) / 128) + r / 128) * blocks;
  }
  __device__ __forceinline__ void load(Raw<FP8>& q, int st, int g) const {
    st = __builtin_amdgcn_readfirstlane(st);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (2 * st + h < blocks) {
        q.v[2 * h] = *(const u32x4*)(p + 256 * st + 128 * h + 16 * g), q.v[2 * h + 1] = *(const u32x4*)(p + 256 * st + 128 * h + 64 + 16 * g);
        q.s[h] = s[2 * st + h];
      } else {
        q.v[2 * h] = q.v[2 * h + 1] = u32x4{0, 0, 0, 0}, q.s[h] = 127;
      }
  }
};
template <> struct Row<MX4> {
  static constexpr int STEP = 512;
  const uint8_t *p, *s;
  int blocks;
  __device__ __forceinline__ Row(const void* w, const uint8_t* scales, int64_t e, int rows, int r, int depth) {
    blocks = (depth + 31) / 32;
    p = (const uint8_t*)w + (e * rows + r) * blocks * 16;
    s = scales + (e * rows + r) * blocks;
  }
  __device__ __forceinline__ void load(Raw<MX4>& q, int st, int g) const {
    st = __builtin_amdgcn_readfirstlane(st);
    if (16 * st + 16 <= blocks) {
#pragma unroll
      for (int i = 0; i < 4; ++i) q.v[i] = *(const u32x4*)(p + 256 * st + 64 * i + 16 * g);
      __builtin_memcpy(&q.s, s + 16 * st, 16);
    } else {
      asm volatile("" : "+s"(st));  // a pointer for every place would take the loop's registers
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int block = 16 * st + 4 * i + g;
        q.v[i] = block < blocks ? *(const u32x4*)(p + 16 * block) : u32x4{0, 0, 0, 0};
        q.s[i] = (block < blocks ? (unsigned)s[block] : 127u) << (8 * g);
      }
    }
  }
};

__device__ __forceinline__ unsigned bits(bf16x2 v) { return __builtin_bit_cast(unsigned, v); }

// 8 elements, the c-th of place i, as bf16 numbers
__device__ __forceinline__ bf16x8 fragment(const Raw<BF16>& q, int i, int) { return __builtin_bit_cast(bf16x8, q.v[i]); }
__device__ __forceinline__ bf16x8 fragment(const Raw<FP8>& q, int i, int c) {
  return fp8::values_bf16(q.v[i][2 * c], q.v[i][2 * c + 1], fp8::scale_of_byte(q.s[i >> 1]));
}
__device__ __forceinline__ bf16x8 fragment(const Raw<MX4>& q, int i, int c) {
  const float scale = fp8::scale_of_byte(q.s[i] >> (threadIdx.x >> 1 & 24));  // the bits above the byte fall on the sign, or out
  const unsigned w = q.v[i][c];
  return __builtin_bit_cast(bf16x8, u32x4{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                                          bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                                          bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                                          bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))});
}

// acc += 16 bytes of tokens times the same elements (the c-th of place i) of matrix rows
template <int F>
__device__ __forceinline__ f32x4 multiply(const Raw<F>& w, int i, int c, u32x4 x, f32x4 acc) {
  if constexpr (F == F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.v[i][j]), __uint_as_float(x[j]), acc, 0, 0, 0);
    return acc;
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(fragment(w, i, c), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
  }
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

// The largest of the eight lanes of a token, to all of them, by moves within the vector unit
template <typename T>
__device__ __forceinline__ T among8(T v, int how) {
  const int u = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(T, how == 0   ? __builtin_amdgcn_mov_dpp(u, 0xb1, 0xf, 0xf, true)     // lanes 1 0 3 2
                               : how == 1 ? __builtin_amdgcn_mov_dpp(u, 0x4e, 0xf, 0xf, true)     // lanes 2 3 0 1
                                          : __builtin_amdgcn_mov_dpp(u, 0x141, 0xf, 0xf, true));  // lanes 7 .. 0
}

// A token's choice by its eight lanes: lane sub looks after the experts sub, sub + 8, ..
__device__ __forceinline__ void choose_token(const LayerArgs& p, const float* l, int* ids, float* shares) {
  const int sub = threadIdx.x & 7;
  uint32_t taken = 0;  // of this lane's experts
  float top = 0.f, total = 0.f, picked = 0.f, mine[2] = {0.f, 0.f};  // of ranks sub and sub + 8
  int id[2] = {0, 0};
  for (int j = 0; j < p.top_k; ++j) {
    unsigned best = 0;
    int at = 0x7fffffff;
    float value = 0.f;
#pragma unroll 4
    for (int i = 0; i < (p.E + 7) / 8; ++i) {
      const int e = min(sub + 8 * i, p.E - 1);
      const float v = l[e];
      const bool better = sub + 8 * i < p.E && !(taken >> i & 1) && (at == 0x7fffffff || key(v) > best);
      best = better ? key(v) : best, at = better ? e : at, value = better ? v : value;
    }
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      const unsigned ob = among8(best, d);
      const int oa = among8(at, d);
      const float ov = among8(value, d);
      const bool better = oa != 0x7fffffff && (at == 0x7fffffff || ob > best || (ob == best && oa < at));
      best = better ? ob : best, at = better ? oa : at, value = better ? ov : value;
    }
    if ((at & 7) == sub) taken |= 1u << (at >> 3);
    if (j == 0) top = value;
    const float share = expf(value - top);
    picked += share;
    if ((j & 7) == sub) mine[j >> 3] = share, id[j >> 3] = at;
  }
#pragma unroll 4
  for (int i = sub; i < p.E; i += 8) total += expf(l[i] - top);  // NaN where one is
#pragma unroll
  for (int d = 0; d < 3; ++d) total += among8(total, d);
  const float by = 1.f / (p.normalize && total == total ? picked : total);
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (sub + 8 * h < p.top_k) ids[sub + 8 * h] = id[h], shares[sub + 8 * h] = mine[h] * by;
}

// The experts of every token and their weights, from the logits.  `logits` is LDS of
// LOGITS floats that fill(t0, tokens) writes.
template <typename GetRound>
__device__ __forceinline__ void choose(const LayerArgs& p, Choice& c, float* logits, GetRound&& fill) {
  const int round = min(LOGITS / p.E, ROUND);  // tokens at once
  for (int t0 = 0; t0 < p.T; t0 += round) {
    const int tokens = min(round, p.T - t0), t = threadIdx.x >> 3;
    __syncthreads();
    fill(t0, tokens);
    __syncthreads();
    if (t >= tokens) continue;
    const float* const l = logits + t * p.E;
    int* const ids = c.e + (t0 + t) * p.top_k;
    float* const shares = c.p + (t0 + t) * p.top_k;
    choose_token(p, l, ids, shares);
  }
  __syncthreads();
}

// The experts that any token chose, ascending, into `active`; how many.
__device__ __forceinline__ int list_active(const LayerArgs& p, const int* chosen, int* active) {
  __shared__ unsigned bits[256 / 32];
  const int slots = p.T * p.top_k, lane = threadIdx.x & 63;
  if (threadIdx.x < 256 / 32) bits[threadIdx.x] = 0;
  __syncthreads();
  for (int s = threadIdx.x; s < slots; s += THREADS) atomicOr(&bits[chosen[s] >> 5], 1u << (chosen[s] & 31));
  __syncthreads();
  int n = 0;
  for (int e0 = 0; e0 < p.E; e0 += 64) {
    const int e = e0 + lane;
    const bool hit = e < p.E && (bits[e >> 5] >> (e & 31) & 1);
    const uint64_t hits = __ballot(hit);
    if (hit && threadIdx.x < 64) active[n + __popcll(hits & (((uint64_t)1 << lane) - 1))] = e;
    n += __popcll(hits);
  }
  __syncthreads();
  return n;
}

// The places (token top_k + rank) that chose expert e, into the wave's own `places`; how
// many.
__device__ __forceinline__ int gather(const LayerArgs& p, const int* chosen, int e, int* places) {
  const int slots = p.T * p.top_k, lane = threadIdx.x & 63;
  int n = 0;
  for (int s0 = 0; s0 < slots; s0 += 64) {
    const int s = s0 + lane;
    const bool hit = s < slots && chosen[s] == e;
    const uint64_t hits = __ballot(hit);
    if (hit) places[n + __popcll(hits & (((uint64_t)1 << lane) - 1))] = s;
    n += __popcll(hits);
  }
  // a wave's LDS accesses keep their order; the compiler has to as well
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
  return n;
}

template <int F> struct Type { typedef __bf16 type; };
template <> struct Type<F32> { typedef float type; };

// A piece's tokens in LDS: a stretch of LEN elements of each, 16 rows or, in as much room,
// 32 of half the length.  Rows lie 16 bytes past a multiple of 256, which parts the 16 rows
// but not the four lanes of each: a ds_read_b128 serves lanes 0-3, 12-15 and 20-27 at once,
// and of these lanes 20-27 meet the banks of lanes 12-15 (25 % of the LDS cycles with bf16
// matrices, 38 to 48 % with packed ones)
template <int F, int ROWS>
struct Tokens {
  static constexpr int LEN = (F == F32 ? 512 : F == MX4 ? 2048 : 1024) * 16 / ROWS;
  typename Type<F>::type v[ROWS][LEN + 16 / sizeof(typename Type<F>::type)];
};

// acc[j]: 16 matrix rows j times `count` tokens, at most 16 and ROWS / PLANES, part `part` of
// DEPTH of the depth, in stretches of Tokens::LEN.  `token(t)` is token t, the first of
// PLANES rows of `depth` elements that add up to it, `wide` apart.  k is taken in the same
// order whatever ROWS and `count`.
// Two tiles of tokens at once were tried: a branch round the MFMAs of the second leaves
// out the wait states that the first one's sums need when it is taken.
template <int F, int TN, int DEPTH, int PLANES, int ROWS, typename GetToken>
__device__ __forceinline__ void product(f32x4 (&acc)[TN], Row<F> (&rows)[TN], Tokens<F, ROWS>& x, int depth, int wide, int count, int part, GetToken&& token) {
  typedef typename Type<F>::type T;
  constexpr int STEP = Row<F>::STEP, V = 16 / sizeof(T), LEN = Tokens<F, ROWS>::LEN, RING = 2;
  const int lane = threadIdx.x & 63, l16 = PLANES == 1 ? lane & 15 : min(lane & 15, count - 1), g = lane >> 4;
  constexpr int EACH = LEN / STEP / DEPTH;  // steps of a wave on a stretch
  static_assert(EACH * STEP * DEPTH == LEN, "every wave has as many steps on a stretch");
  const int all = (depth + STEP - 1) / STEP;
  const int steps = (all - part + DEPTH - 1) / DEPTH, most = (all + DEPTH - 1) / DEPTH;  // of this wave, of any
  Raw<F> w[RING][TN];
  auto load = [&](int buf, int s) {
#pragma unroll
    for (int j = 0; j < TN; ++j) rows[j].load(w[buf][j], part + s * DEPTH, g);
  };
#pragma unroll
  for (int s = 0; s < RING - 1; ++s)
    if (s < steps) load(s, s);
  for (int s = 0; s < most; s += RING) {
#pragma unroll
    for (int q = 0; q < RING; ++q) {
      if (s + q >= most) break;
      if ((s + q) % EACH == 0) {
        const int from = (s + q) * DEPTH * STEP, here = min(depth - from, LEN);
        // 16-byte vectors, with zeros and without; rows of planes have zeros up to `wide`
        const int row = (here + STEP - 1) / STEP * (STEP / V), whole = (PLANES == 1 ? here : here + V - 1) / V;
        __syncthreads();  // the last tokens, or sums, have been read
        // a wave takes AT_ONCE rows at a time, all of their loads first: as many as its registers
        // leave room for (eight vectors for 4 bits 82 us of the call above, four 87; for 8 bits
        // more than two spill)
        constexpr int VECS = (LEN / V + 63) / 64, AT_ONCE = PLANES == 1 ? 1 : (F == MX4 ? 8 : F == FP8 ? 2 : 4) / VECS;
        for (int t0 = wave_of(); t0 < count * PLANES; t0 += WAVES * AT_ONCE) {
          u32x4 v[AT_ONCE][VECS];
#pragma unroll
          for (int r = 0; r < AT_ONCE; ++r) {
            const int t = min(t0 + WAVES * r, count * PLANES - 1);
            const T* const src = PLANES == 1 ? token(t) + from : token(t % count) + (int64_t)(t / count) * wide + from;
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
              v[r][i] = u32x4{0, 0, 0, 0};
              if (lane + 64 * i < whole) __builtin_memcpy(&v[r][i], src + (lane + 64 * i) * V, 16);
            }
          }
#pragma unroll
          for (int r = 0; r < AT_ONCE; ++r) {
            const int t = t0 + WAVES * r;
            if (t >= count * PLANES) break;
#pragma unroll
            for (int i = 0; i < VECS; ++i)
              if (lane + 64 * i < row) __builtin_memcpy(__builtin_assume_aligned(&x.v[t][(lane + 64 * i) * V], 16), &v[r][i], 16);
            // what is left of the row, after the zeros
            if (PLANES == 1 && lane < here % V) x.v[t][whole * V + lane] = token(t)[from + whole * V + lane];
          }
        }
        __syncthreads();
      }
      if (s + q >= steps) break;
      if (s + q + RING - 1 < steps) load((q + RING - 1) % RING, s + q + RING - 1);
      const int k = (part + (s + q) % EACH * DEPTH) * STEP + g * (STEP / 16);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
#pragma unroll
        for (int c = 0; c < STEP / 16 / V; ++c) {
#pragma unroll
          for (int i = PLANES - 1; i >= 0; --i) {
            const u32x4 v = *(const u32x4*)&x.v[i * count + l16][k + h * (STEP / 4) + V * c];
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[j] = multiply<F>(w[q][j], h, c, v, acc[j]);
          }
        }
        // a place's conversions follow those before it: all at once they fill the registers
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // the sums are read behind branches: their wait states are spelled out
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15");
  __builtin_amdgcn_sched_barrier(0);
}

// The three bf16 numbers, as their bits, that add up to v: its leading eight bits, the next
// and the last.  Cut off, not rounded, so that the first is finite where v is.
__device__ __forceinline__ void split3(float v, unsigned short (&out)[3]) {
  const unsigned first = __float_as_uint(v) & 0xffff0000u;
  const float rest = (first & 0x7f800000u) == 0x7f800000u ? 0.f : v - __uint_as_float(first);
  const unsigned second = __float_as_uint(rest) & 0xffff0000u;
  out[0] = (unsigned short)(first >> 16), out[1] = (unsigned short)(second >> 16);
  out[2] = (unsigned short)(__float_as_uint(rest - __uint_as_float(second)) >> 16);
}

// The sums of the DEPTH waves that share a piece's depth: f(v, q) with tile q of them, in
// one wave each.
template <int TN>
struct Sums {
  f32x4 v[WAVES][TN][64];
};
template <int DEPTH, int TN, typename Keep>
__device__ __forceinline__ void summed(Sums<TN>& sums, const f32x4 (&acc)[TN], Keep&& f) {
  const int lane = threadIdx.x & 63, wave = wave_of(), member = wave % DEPTH;
  __syncthreads();  // the tokens, or the last sums, have been read
#pragma unroll
  for (int j = 0; j < TN; ++j) sums.v[wave][j][lane] = acc[j];
  __syncthreads();
#pragma unroll
  for (int q0 = 0; q0 < TN; q0 += DEPTH) {
    const int q = q0 + member;
    if (q >= TN) break;
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < DEPTH; ++w) v += sums.v[wave - member + w][q][lane];
    f(v, q);
  }
}

}  // namespace layer

// Sixteen tokens' logits of sixteen experts: element r of lane (g, l16) is expert 4 g + r
// of token l16.  `from` .. `from` + `depth` of K.
template <typename T>
__device__ __forceinline__ layer::f32x4 logit_tile(layer::Sums<1>& sums, const LayerArgs& p, int t0, int e0, int from, int depth) {
  using namespace layer;
  constexpr int F = sizeof(T) == 4 ? F32 : BF16;
  const int l16 = threadIdx.x & 15;
  const int wave = wave_of(), g = threadIdx.x >> 4 & 3;
  const T* const x = (const T*)p.x + (int64_t)min(t0 + l16, p.T - 1) * p.ldx + from;
  const T* const w = (const T*)p.router + (int64_t)min(e0 + l16, p.E - 1) * p.K + from;
  constexpr int STEP = Row<F>::STEP;
  f32x4 acc[1] = {};
  for (int k = wave * STEP; k < depth; k += WAVES * STEP) {
    Raw<F> a;
    u32x4 b[4];
    load_step(a.v, w, k, g, depth), load_step(b, x, k, g, depth);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[0] = multiply<F>(a, i, 0, b[i], acc[0]);
  }
  layer::f32x4 got = {};
  summed<WAVES>(sums, acc, [&](layer::f32x4 v, int) { got = v; });
  return got;
}

// logits[part][t][e]: blockIdx.x 16 tokens, .y 16 experts, .z a part of k
template <typename T>
__global__ void __launch_bounds__(layer::THREADS) layer_logits(LayerArgs p) {
  using namespace layer;
  constexpr int STEP = 256 / sizeof(T);
  __shared__ Sums<1> sums;
  const int t0 = blockIdx.x * 16, e0 = blockIdx.y * 16;
  // whole steps of a part
  const int steps = (p.K + STEP - 1) / STEP;
  const int from = (int)((int64_t)steps * blockIdx.z / gridDim.z) * STEP;
  const int depth = min((int)((int64_t)steps * (blockIdx.z + 1) / gridDim.z) * STEP, p.K) - from;
  const f32x4 v = logit_tile<T>(sums, p, t0, e0, from, depth);
  const int t = t0 + (threadIdx.x & 15), e = e0 + (threadIdx.x >> 4) * 4;
  if (threadIdx.x < 64 && t < p.T)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (e + r < p.E) p.logits[((int64_t)blockIdx.z * p.T + t) * p.E + e + r] = v[r];
}

// p act(U x): pieces of TN tiles of rows for every DEPTH waves
template <int F, int TN, bool SWIGLU, int DEPTH>
__global__ void __launch_bounds__(layer::THREADS, F == layer::MX4 ? 2 : 3) layer_up(LayerArgs p) {
  using namespace layer;
  typedef typename Type<F>::type T;
  constexpr int TILE = SWIGLU ? 8 : 16, ROWS = TILE * TN * (WAVES / DEPTH);
  __shared__ __attribute__((aligned(16))) union {
    Tokens<F, 16> tokens;
    Sums<TN> sums;
    Sums<1> logit_sums;
    float logits[LOGITS];
  } lds;
  __shared__ Choice choice;
  __shared__ int active[256], places_of[WAVES][64];
  const int lane = threadIdx.x & 63, wave = wave_of(), l16 = lane & 15, g = lane >> 4;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < (p.K + 15) / 16; i += THREADS) p.counters[i] = 0;

  choose(p, choice, lds.logits, [&](int t0, int tokens) {
    if (p.logits) {
      for (int i = threadIdx.x; i < tokens * p.E; i += THREADS) {
        float v = 0.f;
        for (int s = 0; s < p.logit_parts; ++s) v += p.logits[((int64_t)s * p.T + t0) * p.E + i];
        lds.logits[i] = v;
      }
      return;
    }
    // T <= ROUND and T E <= LOGITS: one round.  A tile's sums stay in registers until all are done
    constexpr int MOST = 4;  // tiles that the caller allows
    f32x4 mine[MOST];
    const int et = (p.E + 15) / 16, tiles = et * ((p.T + 15) / 16);
#pragma unroll 1
    for (int q = 0; q < tiles; ++q) {
      const f32x4 v = logit_tile<T>(lds.logit_sums, p, q / et * 16, q % et * 16, 0, p.K);
#pragma unroll
      for (int i = 0; i < MOST; ++i)
        if (i == q) mine[i] = v;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      const int t = q / et * 16 + l16, e = q % et * 16 + 4 * g;
      if (q < tiles && wave == 0 && t < p.T)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (e + r < p.E) lds.logits[t * p.E + e + r] = mine[q][r];
    }
  });
  const int experts = list_active(p, choice.e, active);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.T * p.top_k; i += THREADS) p.choice[i] = choice.e[i];

  int* const places = places_of[wave];
  for (int piece = blockIdx.x; piece < experts * p.slices; piece += gridDim.x) {
    const int e = active[piece / p.slices], slice = piece % p.slices;
    const int n = gather(p, choice.e, e, places);
    const int n0 = slice * ROWS + wave / DEPTH * (TILE * TN);  // first row of the wave's first tile
    // h of four rows from `row` of the token at `place`
    auto keep = [&](f32x4 v, int row, int place, bool there) {
      f32x4 h;
      if constexpr (SWIGLU) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float u = __shfl_xor(v[r], 32);
          h[r] = v[r] / (1.f + expf(-v[r])) * u;
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) h[r] = v[r] < 0.f ? 0.f : v[r];
      }
      if (!there || row >= p.Hp || (SWIGLU && g >= 2)) return;
      const float share = choice.p[place];
#pragma unroll
      for (int r = 0; r < 4; ++r) h[r] = row + r < p.H ? h[r] * share : 0.f;
      // Hp is a multiple of 32: four rows at once
      if constexpr (F == F32) {
        *(f32x4*)((float*)p.mid + (int64_t)place * p.Hp + row) = h;
      } else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
        __bf16* const to = (__bf16*)p.mid + (int64_t)place * p.planes * p.Hp + row;
        if (p.planes == 1) {
          *(bf16x4*)to = __builtin_convertvector(h, bf16x4);
        } else {
          unsigned short parts[4][3];
#pragma unroll
          for (int r = 0; r < 4; ++r) split3(h[r], parts[r]);
#pragma unroll
          for (int i = 0; i < 3; ++i) *(u16x4*)(to + (int64_t)i * p.Hp) = u16x4{parts[0][i], parts[1][i], parts[2][i], parts[3][i]};
        }
      }
    };
    for (int at = 0; at < n; at += 16) {
      f32x4 acc[TN] = {};
      // rows past the last one repeat it and are not kept
      auto row = [&](int j) {
        const int r = n0 + TILE * j + (SWIGLU ? l16 & 7 : l16);
        return Row<F>(p.up, p.up_scales, e, SWIGLU ? 2 * p.H : p.H, (SWIGLU && l16 >= 8 ? p.H : 0) + min(r, p.H - 1), p.K);
      };
      Row<F> rows[2] = {row(0), row(1)};
      static_assert(TN == 2, "two tiles of rows a wave");
      product<F, TN, DEPTH, 1, 16>(acc, rows, lds.tokens, p.K, p.K, min(n - at, 16), wave % DEPTH,
                                [&](int t) { return (const T*)p.x + (int64_t)(places[at + t] / p.top_k) * p.ldx; });
      summed<DEPTH>(lds.sums, acc, [&](f32x4 v, int q) {
        const int t = at + l16;
        keep(v, n0 + TILE * q + 4 * (SWIGLU ? g & 1 : g), places[min(t, n - 1)], t < n);
      });
    }
  }
}

// D of the same, and the sum over a token's experts by the last workgroup of a slice
template <int F, int TN, int DEPTH, int PLANES>
__global__ void __launch_bounds__(layer::THREADS, F == layer::MX4 ? 2 : 3) layer_down(LayerArgs p) {
  using namespace layer;
  typedef typename Type<F>::type T;
  constexpr int ROWS = 16 * TN * (WAVES / DEPTH);
  // with three planes 16 rows are five tokens; ten have 32 where a step of every wave is half a
  // stretch
  constexpr bool WIDE = PLANES > 1 && 2 * DEPTH * Row<F>::STEP <= Tokens<F, 16>::LEN;
  __shared__ __attribute__((aligned(16))) union {
    Tokens<F, 16> tokens;
    Tokens<F, WIDE ? 32 : 16> more;
    Sums<TN> sums;
  } lds;
  __shared__ int chosen[64 * 16], active[256], places_of[WAVES][64];
  const int lane = threadIdx.x & 63, wave = wave_of(), l16 = lane & 15, g = lane >> 4;
  for (int i = threadIdx.x; i < p.T * p.top_k; i += THREADS) chosen[i] = p.choice[i];
  __syncthreads();
  const int experts = list_active(p, chosen, active);
  int* const places = places_of[wave];
  const bool whole = (p.K & 3) == 0;
  for (int piece = blockIdx.x; piece < experts * p.slices; piece += gridDim.x) {
    const int e = active[piece / p.slices], slice = piece % p.slices;
    const int n = gather(p, chosen, e, places);
    const int n0 = slice * ROWS + wave / DEPTH * (16 * TN);
    auto keep = [&](f32x4 v, int row, int place, bool there) {
      if (!there || row >= p.K) return;
      float* const to = p.parts + (int64_t)place * p.K + row;
      if (whole) {
        splitk_store4(to, v);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (row + r < p.K) splitk_store(to + r, v[r]);
      }
    };
    for (int at = 0, here; at < n; at += here) {
      here = min(n - at, WIDE ? 32 / PLANES : 16 / PLANES);
      f32x4 acc[TN] = {};
      auto row = [&](int j) { return Row<F>(p.down, p.down_scales, e, p.K, min(n0 + 16 * j + l16, p.K - 1), p.H); };
      auto token = [&](int t) { return (const T*)p.mid + (int64_t)places[at + t] * PLANES * p.Hp; };
      auto sum = [&](Row<F>(&rows)[TN]) {
        if constexpr (WIDE)
          if (here > 16 / PLANES) return product<F, TN, DEPTH, PLANES, 32>(acc, rows, lds.more, p.H, p.Hp, here, wave % DEPTH, token);
        product<F, TN, DEPTH, PLANES, 16>(acc, rows, lds.tokens, p.H, p.Hp, here, wave % DEPTH, token);
      };
      static_assert(TN == 1 || TN == 2, "one or two tiles of rows a wave");
      if constexpr (TN == 1) {
        Row<F> rows[1] = {row(0)};
        sum(rows);
      } else {
        Row<F> rows[2] = {row(0), row(1)};
        sum(rows);
      }
      summed<DEPTH>(lds.sums, acc, [&](f32x4 v, int q) {
        const int t = at + l16;
        keep(v, n0 + 16 * q + 4 * g, places[min(t, n - 1)], l16 < here);
      });
    }
    if (!splitk_arrive(p.counters + slice, experts)) continue;
    const int first = slice * ROWS, rows_here = min(ROWS, p.K - first);
    for (int i = threadIdx.x; i < p.T * ROWS; i += THREADS) {
      const int r = i % ROWS, t = i / ROWS;
      if (r >= rows_here) continue;
      ((T*)p.y)[(int64_t)t * p.ldy + first + r] = (T)splitk_sum1(p.parts + (int64_t)t * p.top_k * p.K + first + r, (size_t)p.K, p.top_k);
    }
  }
}

// The two launches.
struct LayerGrid {
  bool shared;  // four waves share the depth, or two
  bool narrow;  // pieces of layer_down have 16 rows, not 32
  int up_slices, down_slices;
  unsigned up, down;  // workgroups
};
// Each of a translation unit of its own: layer_f32.hip, layer_bf16.hip, ..
template <int F>
void layer_launch(const LayerArgs& a, const LayerGrid& g, hipStream_t s);

template <int F, int DEPTH, int PLANES>
void layer_launch_down(const LayerArgs& a, const LayerGrid& g, hipStream_t s) {
  if constexpr (DEPTH == layer::WAVES)
    if (g.narrow) {
      hipLaunchKernelGGL((layer_down<F, 1, DEPTH, PLANES>), dim3(g.down), dim3(layer::THREADS), 0, s, a);
      return;
    }
  hipLaunchKernelGGL((layer_down<F, 2, DEPTH, PLANES>), dim3(g.down), dim3(layer::THREADS), 0, s, a);
}
template <int F, int DEPTH>
void layer_launch_tiles(const LayerArgs& a, const LayerGrid& g, hipStream_t s) {
  LayerArgs u = a, d = a;
  u.slices = g.up_slices, d.slices = g.down_slices;
  if (a.swiglu) hipLaunchKernelGGL((layer_up<F, 2, true, DEPTH>), dim3(g.up), dim3(layer::THREADS), 0, s, u);
  else hipLaunchKernelGGL((layer_up<F, 2, false, DEPTH>), dim3(g.up), dim3(layer::THREADS), 0, s, u);
  if constexpr (F != layer::F32)
    if (a.planes == 3) return layer_launch_down<F, DEPTH, 3>(d, g, s);
  layer_launch_down<F, DEPTH, 1>(d, g, s);
}
#define XTC_HIP_LAYER_LAUNCH(F)                                                  \
  template <>                                                                    \
  void layer_launch<F>(const LayerArgs& a, const LayerGrid& g, hipStream_t s) {  \
    if constexpr (F == layer::FP8 || F == layer::MX4)                            \
      if (!g.shared) return layer_launch_tiles<F, 2>(a, g, s);                   \
    layer_launch_tiles<F, layer::WAVES>(a, g, s);                                \
  }
template <> void layer_launch<layer::F32>(const LayerArgs&, const LayerGrid&, hipStream_t);
template <> void layer_launch<layer::BF16>(const LayerArgs&, const LayerGrid&, hipStream_t);
template <> void layer_launch<layer::FP8>(const LayerArgs&, const LayerGrid&, hipStream_t);
template <> void layer_launch<layer::MX4>(const LayerArgs&, const LayerGrid&, hipStream_t);

}  // namespace xtc_hip
