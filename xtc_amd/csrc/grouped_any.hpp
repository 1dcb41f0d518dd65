// SPDX-License-Identifier: BSD-3-Clause
// Products by group for operands of any size, stride and alignment:
//   y[r, :] = x[r, :] w[e]            for the rows r of group e      (GRAD = false)
//   dw[e]   = sum_r x[r, :]^T dy[r, :] over the rows r of group e    (GRAD = true)
// Both are sums C[i, j] = sum_k A[i, k] B[k, j]: i the rows and k the depth of w,
// or i the depth of w and k the rows.
//
// grouped_any: a workgroup of 2 x 2 waves computes a 64 x 64 tile of C, k in slabs
// of 32 through two LDS buffers, the next three in registers meanwhile.  An operand
// is loaded 8 elements a lane along its contiguous axis (unaligned vectors, which
// global memory takes at element alignment; element by element where the operand
// ends inside) and kept in LDS as it came: bf16 in the layouts of grouped_dma.hpp,
// fp32 in padded rows.  bf16 runs on v_mfma_f32_16x16x32_bf16, fp32 on
// v_mfma_f32_16x16x4_f32 (exact products, a lane's 8 k of a slab in any order as
// long as A and B agree).  Sums are fp32; a bf16 result is rounded once, at the
// store.  4096 rows over 8 experts of 1001 x 999: bf16 68 us, the gradient of w 50, where
// memory and MFMAs need 7 and 10; fp32 112, where the MFMAs need 53.  The time goes into
// loads by way of registers, in pieces of 8 elements, into tiles so small that x is read N / 64
// times and a group's matrix once for every 64 of its rows, with a barrier every slab;
// LDS-DMA from copies in whole vectors has not been tried.
//
// grouped_small takes the calls whose 64 x 64 tiles do not fill the card, and few
// rows a group (then it streams the matrices): a workgroup computes a tile of 16
// or 32 rows with 8 waves that share out the depth in turn,
// load their fragments straight into registers, two or three steps ahead, and add their sums
// up in LDS, in order.  No barrier but that one: the loads of a whole call are in
// flight together.  Bound by the latency of one walk: 777 fp32 rows over 5 experts of
// 509 x 301 9.3 us (22 in slabs), 2 bf16 rows at 8 of 1024 x 1024 3.8, a launch.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "grouped_dma.hpp"
#include "groups.hpp"

namespace xtc_hip {

struct GroupedArgs {
  const void* x;     // [T][ldx]
  const void* w;     // [E] matrices, stride_w elements apart; GRAD: dy [T][ldw]
  const int* sizes;  // [E]
  void* y;           // [T][ldy]; GRAD: [E] matrices [K][ldy], stride_y apart
  int64_t stride_w, stride_y;
  int E, T, N, K;
  int ldx, ldw, ldy;
  int tiles_n, tiles_k;
};

namespace gany {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr int BM = 64, BN = 64, BK = 32, NT = 256;

// the elements at p, of which the first n exist, zeros for the others
template <typename T, int LEN>
__device__ __forceinline__ void load_some(T (&v)[LEN], const T* p, int n) {
  if (n >= LEN) {
    __builtin_memcpy(v, p, LEN * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < LEN; ++i) v[i] = i < n ? p[i] : (T)0.f;
  }
}

// a lane's share of a slab: KC: 8 k of one row, else 8 rows at one k
template <typename T, bool KC>
__device__ __forceinline__ void load(T (&v)[8], const T* p, int64_t ld, int rows, int depth) {
  const int tid = threadIdx.x;
  if constexpr (KC) {
    const int r = tid >> 2, k = (tid & 3) * 8;
    load_some(v, p + (int64_t)r * ld + k, r < rows ? depth - k : 0);
  } else {
    const int k = tid >> 3, r = (tid & 7) * 8;
    load_some(v, p + (int64_t)k * ld + r, k < depth ? rows - r : 0);
  }
}

// An operand's slab in LDS and a lane's fragment of 16 of its rows from 16 f on.
template <typename T, bool KC> struct Slab;
template <bool KC> struct Slab<__bf16, KC> {
  static constexpr int BYTES = 64 * BK * 2;
  static __device__ __forceinline__ void store(unsigned char* st, const __bf16 (&v)[8]) {
    const int tid = threadIdx.x;
    int at;
    if constexpr (KC) at = (tid >> 2) * 64 + 16 * ((tid & 3) ^ gdma::swz_row<false>(tid >> 2));
    else at = (tid >> 3) * 128 + 32 * ((tid & 7) / 2 ^ gdma::swz_col<64>(tid >> 3)) + 16 * (tid & 1);
    __builtin_memcpy(__builtin_assume_aligned(st + at, 16), v, 16);
  }
  typedef gdma::u32x4 Fragment;
  static __device__ __forceinline__ Fragment read(const unsigned char* st, int f, int l16, int g) {
    return gdma::fragment<KC, 64>(st, 0, f, l16, g);
  }
};
template <bool KC> struct Slab<float, KC> {
  static constexpr int STRIDE = KC ? BK + 4 : 64 + 4, BYTES = (KC ? 64 : BK) * STRIDE * 4;
  static __device__ __forceinline__ void store(unsigned char* st, const float (&v)[8]) {
    const int tid = threadIdx.x;
    float* const p = (float*)st + (KC ? (tid >> 2) * STRIDE + (tid & 3) * 8 : (tid >> 3) * STRIDE + (tid & 7) * 8);
    __builtin_memcpy(__builtin_assume_aligned(p, 16), v, 32);
  }
  struct Fragment { f32x4 v[2]; };
  static __device__ __forceinline__ Fragment read(const unsigned char* st, int f, int l16, int g) {
    const float* const p = (const float*)st;
    Fragment r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (KC) {
        r.v[h] = *(const f32x4*)(p + (16 * f + l16) * STRIDE + 16 * h + 4 * g);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) r.v[h][q] = p[(16 * h + 4 * g + q) * STRIDE + 16 * f + l16];
      }
    }
    return r;
  }
};

__device__ __forceinline__ void mma(f32x4& c, gdma::u32x4 b, gdma::u32x4 a) { c = gdma::mfma(b, a, c); }
template <typename B, typename A>
__device__ __forceinline__ void mma(f32x4& c, const B& b, const A& a) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(b.v[h][q], a.v[h][q], c, 0, 0, 0);
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

// grouped_small: what a lane feeds to the 16 x 16 products of one step
constexpr int SWAVES = 8;
template <typename T> struct Small;
template <> struct Small<float> {
  static constexpr int STEP = 16, PER = 4;  // k of a step, of a lane in it
  static __device__ __forceinline__ void mma(f32x4& c, const float (&b)[4], const float (&a)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) c = __builtin_amdgcn_mfma_f32_16x16x4f32(b[q], a[q], c, 0, 0, 0);
  }
};
template <> struct Small<__bf16> {
  static constexpr int STEP = 32, PER = 8;
  static __device__ __forceinline__ void mma(f32x4& c, const __bf16 (&b)[8], const __bf16 (&a)[8]) {
    bf16x8 bv, av;
    __builtin_memcpy(&bv, b, 16);
    __builtin_memcpy(&av, a, 16);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bv, av, c, 0, 0, 0);
  }
};

// An operand's part of a step: W fragments of 16 lines (rows or columns) each.
// KC: k contiguous, a lane takes PER k of lines l16, 16 + l16, ...; otherwise its W
// neighbouring lines at PER k, loaded together: W l16 .. W l16 + W - 1, or the last
// W of the tile where it ends among or before them.  What lanes hold twice comes
// out the same twice; lines past a tile of less than W are zeros.
template <typename T, bool KC, int W>
struct SmallOperand {
  static constexpr int PER = Small<T>::PER;
  const T* at[KC ? W : 1];
  int64_t ld, next;  // between k rows; to the wave's next step
  int edge;          // lines of the tile

  __device__ __forceinline__ int line(int w, int l16) const {
    return KC ? 16 * w + l16 : min(W * l16, max(edge - W, 0)) + w;
  }
  // lines past the edge repeat the last one (KC)
  __device__ __forceinline__ void set(const T* p, int64_t stride, int l16, int k, int lines, int step) {
    ld = stride;
    next = KC ? step : step * stride;
    edge = lines;
    if constexpr (KC) {
#pragma unroll
      for (int w = 0; w < W; ++w) at[w] = p + min(line(w, l16), edge - 1) * stride + k;
    } else {
      at[0] = p + k * stride + line(0, l16);
    }
  }
  // a step as loaded: fragments, or W lines at each of PER k (turned over only when
  // they are used, so that the loads stay in flight)
  static constexpr int ROWS = KC ? W : PER, COLS = KC ? PER : W;
  typedef T Raw[ROWS][COLS];
  static __device__ __forceinline__ void fragment(T (&f)[PER], const Raw& v, int w) {
#pragma unroll
    for (int i = 0; i < PER; ++i) f[i] = KC ? v[w][i] : v[i][w];
  }
  // the step, `left` k from the lane's first one to the end; then on to the next
  __device__ __forceinline__ void load(Raw& v, int left) {
    if constexpr (KC) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
        load_some(v[w], at[w], left);
        at[w] += next;
      }
    } else {
      if (left >= PER && edge >= W) {
#pragma unroll
        for (int i = 0; i < PER; ++i) __builtin_memcpy(v[i], at[0] + i * ld, sizeof(v[i]));
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) load_some(v[i], at[0] + i * ld, i < left ? edge : 0);
      }
      at[0] += next;
    }
  }
};

}  // namespace gany

// 16 TM x 16 TN tiles.
template <typename T, typename U, bool WT, bool GRAD, int TM, int TN>
__global__ void __launch_bounds__(64 * gany::SWAVES) grouped_small(GroupedArgs p) {
  using namespace gany;
  typedef Small<T> S;
  typedef SmallOperand<T, !GRAD, TM> OpA;
  typedef SmallOperand<T, WT && !GRAD, TN> OpB;
  constexpr int SM = 16 * TM, SN = 16 * TN;
  __shared__ float sums[SWAVES][SM][SN + 4];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const T *a = (const T*)p.x, *b = (const T*)p.w;
  U* c = (U*)p.y;
  int rows, depth, n0;
  if constexpr (GRAD) {
    const int e = blockIdx.x / (p.tiles_k * p.tiles_n), t = blockIdx.x % (p.tiles_k * p.tiles_n);
    const int k0 = t / p.tiles_n * SM;
    n0 = t % p.tiles_n * SN;
    const RowGroup gr = find_group(p.sizes, p.E, p.T, e);
    a += (int64_t)gr.begin * p.ldx + k0;
    b += (int64_t)gr.begin * p.ldw + n0;
    c += e * p.stride_y + (int64_t)k0 * p.ldy + n0;
    rows = min(p.K - k0, SM);
    depth = gr.end - gr.begin;
  } else {
    n0 = blockIdx.x % p.tiles_n * SN;
    const RowGroup gr = find_tile<SM>(p.sizes, p.E, p.T, blockIdx.x / p.tiles_n);
    if (gr.e < 0) return;
    a += (int64_t)gr.begin * p.ldx;
    b += (gr.e < p.E ? gr.e : 0) * p.stride_w + (int64_t)n0 * (WT ? p.ldw : 1);
    c += (int64_t)gr.begin * p.ldy + n0;
    rows = min(gr.end - gr.begin, SM);
    depth = gr.e < p.E ? p.K : 0;  // rows of no group: zeros
  }
  const int cols = min(p.N - n0, SN);

  constexpr int STRIDE = SWAVES * S::STEP, RING = TM == 1 ? 4 : 3;
  const int k0 = wave * S::STEP, kl = k0 + g * S::PER;
  OpA oa;
  OpB ob;
  oa.set(a, p.ldx, l16, kl, rows, STRIDE);
  ob.set(b, p.ldw, l16, kl, cols, STRIDE);
  f32x4 acc[TM][TN] = {};
  typename OpA::Raw av[RING];
  typename OpB::Raw bv[RING];
  int left = depth - kl;  // k from the lane's next element on
  auto load = [&](int buf) {
    ob.load(bv[buf], left);
    oa.load(av[buf], left);
    left -= STRIDE;
  };
  const int steps = (depth - k0 + STRIDE - 1) / STRIDE;  // of this wave
#pragma unroll
  for (int s = 0; s < RING - 1; ++s)
    if (s < steps) load(s);
  for (int s = 0; s < steps; s += RING) {
#pragma unroll
    for (int q = 0; q < RING; ++q) {
      if (s + q >= steps) break;
      if (s + q + RING - 1 < steps) load((q + RING - 1) % RING);
      T fa[TM][S::PER], fb[TN][S::PER];
#pragma unroll
      for (int i = 0; i < TM; ++i) OpA::fragment(fa[i], av[q], i);
#pragma unroll
      for (int j = 0; j < TN; ++j) OpB::fragment(fb[j], bv[q], j);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) S::mma(acc[i][j], fb[j], fa[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][oa.line(i, l16)][ob.line(j, 4 * g + r)] = acc[i][j][r];
  __syncthreads();
  for (int t = threadIdx.x; t < SM * SN; t += 64 * SWAVES) {
    const int m = t / SN, n = t % SN;
    if (m >= rows || n >= cols) continue;
    float v = sums[0][m][n];
#pragma unroll
    for (int w = 1; w < SWAVES; ++w) v += sums[w][m][n];
    c[(int64_t)m * p.ldy + n] = (U)v;
  }
}

// T: operands, U: result; WT: w stored transposed ([N][K]; GRAD: unused)
template <typename T, typename U, bool WT, bool GRAD>
__global__ void __launch_bounds__(256) grouped_any(GroupedArgs p) {
  using namespace gany;
  constexpr bool A_KC = !GRAD, B_KC = WT && !GRAD;
  typedef Slab<T, A_KC> SlabA;
  typedef Slab<T, B_KC> SlabB;
  __shared__ __attribute__((aligned(16))) unsigned char lds_a[2][SlabA::BYTES], lds_b[2][SlabB::BYTES];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l16 = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
  const T* const x = (const T*)p.x;
  const T* const w = (const T*)p.w;

  const T *a, *b;
  U* c;
  int rows, cols, depth;  // of the tile and its sums
  int64_t a_step, b_step;  // a slab further along k
  int n0;
  if constexpr (GRAD) {
    const int e = blockIdx.x / (p.tiles_k * p.tiles_n), t = blockIdx.x % (p.tiles_k * p.tiles_n);
    const int k0 = t / p.tiles_n * BM;
    n0 = t % p.tiles_n * BN;
    const RowGroup gr = find_group(p.sizes, p.E, p.T, e);
    a = x + (int64_t)gr.begin * p.ldx + k0;
    b = w + (int64_t)gr.begin * p.ldw + n0;
    c = (U*)p.y + e * p.stride_y + (int64_t)k0 * p.ldy + n0;
    rows = p.K - k0;
    depth = gr.end - gr.begin;
    a_step = (int64_t)BK * p.ldx;
    b_step = (int64_t)BK * p.ldw;
  } else {
    const int mt = blockIdx.x / p.tiles_n;
    n0 = blockIdx.x % p.tiles_n * BN;
    const RowGroup gr = find_tile<BM>(p.sizes, p.E, p.T, mt);
    if (gr.e < 0) return;
    a = x + (int64_t)gr.begin * p.ldx;
    b = w + (gr.e < p.E ? gr.e : 0) * p.stride_w + (int64_t)n0 * (WT ? p.ldw : 1);
    c = (U*)p.y + (int64_t)gr.begin * p.ldy + n0;
    rows = gr.end - gr.begin;
    depth = gr.e < p.E ? p.K : 0;  // rows of no group: zeros
    a_step = BK;
    b_step = WT ? (int64_t)BK : (int64_t)BK * p.ldw;
  }
  rows = min(rows, BM);
  cols = min(p.N - n0, BN);

  f32x4 acc[2][2] = {};
  const int steps = (depth + BK - 1) / BK;
  // slabs s + 1 .. s + RING in registers during step s
  constexpr int RING = 3;
  T av[RING][8], bv[RING][8];
  auto load_next = [&](int buf) {
    load<T, A_KC>(av[buf], a, p.ldx, rows, depth);
    load<T, B_KC>(bv[buf], b, p.ldw, cols, depth);
    a += a_step;
    b += b_step;
    depth -= BK;
  };
#pragma unroll
  for (int q = 0; q < RING; ++q)
    if (q < steps) load_next(q);
  if (steps > 0) {
    SlabA::store(lds_a[0], av[0]);
    SlabB::store(lds_b[0], bv[0]);
    if (RING < steps) load_next(0);
  }
  for (int s0 = 0; s0 < steps; s0 += RING) {
#pragma unroll
    for (int q = 0; q < RING; ++q) {
      const int s = s0 + q;
      if (s >= steps) break;
      __syncthreads();
      typename SlabA::Fragment fa[2];
      typename SlabB::Fragment fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) fa[i] = SlabA::read(lds_a[s & 1], wm * 2 + i, l16, g);
#pragma unroll
      for (int j = 0; j < 2; ++j) fb[j] = SlabB::read(lds_b[s & 1], wn * 2 + j, l16, g);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) mma(acc[i][j], fb[j], fa[i]);
      if (s + 1 < steps) {
        constexpr int NEXT_OF[RING] = {1, 2, 0};
        const int next = NEXT_OF[q];
        SlabA::store(lds_a[(s + 1) & 1], av[next]);
        SlabB::store(lds_b[(s + 1) & 1], bv[next]);
        if (s + 1 + RING < steps) load_next(next);
      }
    }
  }
  // a lane holds C[i][j .. j+3]: B is the first MFMA operand
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = wm * 32 + i * 16 + l16;
    if (m >= rows) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = wn * 32 + j * 16 + 4 * g;
      put(c + (int64_t)m * p.ldy + n, acc[i][j], cols - n);
    }
  }
}

}  // namespace xtc_hip
