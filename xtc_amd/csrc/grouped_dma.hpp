// SPDX-License-Identifier: BSD-3-Clause
// Products by group of bf16 or microscaled 4-bit operands in whole 16-byte
// vectors, staged through LDS by DMA:
//   C[i, j] = sum_k A[i, k] B[k, j]
// for the rows i of a group and its matrix B, or (GRAD) over the rows k of a
// group: see grouped_any.hpp and mx4_any.hpp, which take what this kernel does
// not.
//
// Tile and slab.  A workgroup of WGM x WGN waves computes (16 WGM TM) x
// (16 WGN TN) outputs, k in slabs of a row: 64 bytes or 32 bf16, one
// v_mfma_f32_16x16x32_bf16 deep, or 128 bytes or 256 4-bit elements, four
// v_mfma_scale_f32_32x32x64_f8f6f4 deep (registers only: 6.5 PFLOP/s, the
// 16x16x128 form 5.6: the scales take issue slots), read and multiplied in two
// halves.  A lane feeds either with 16 bytes of a row.  B is the first MFMA operand:
// a lane ends with four neighbouring columns of one row.  4-bit slabs are whole
// cache lines, because half lines are what bounds the DMA from L2: 17 TB/s in 64
// bytes a row, 26 in 128 (8192^3 349 us and 320, in 64 x 64 tiles 741 and 600).
//
// Operands come in two forms.
//   ROW  k contiguous: staged [rows][slab], its 16-byte chunk c of row r at
//        c ^ ((r >> 1) & 3), 4-bit c ^ ((r >> 1) & 7), read by ds_read_b128.
//   COL  k strided (bf16): staged [32 k][16-bit columns], its 32-byte chunk c of
//        row k at c ^ swz(k), read transposed by ds_read_b64_tr_b16.
// 4-bit operands bring 8 scale bytes a row and slab.  They are staged for two
// slabs at a time, [rows][16], with the pair's first (8 bytes of each row a slab
// would touch as many cache lines as the codes), and a lane reads its row's 16 at
// once and keeps the 8 of its k (byte reads for every step cost 8192^3 80 us).
//
// What bounds it: bf16, the board's power (32768 rows over 16 experts of 4096 x 4096
// 912-957 us by card, 1.15-1.2 PFLOP/s, as a large library product); gradients, writing
// fp32 tiles of shallow sums after their products (16384 rows over 16 of 2048 x 2048
// 172-209 us by card, 268 MB); 4-bit, LDS: two slabs of 64 KB, so that the DMA is one slab
// ahead (8192^3 300-320 us, 3.4-3.7 PFLOP/s).  Of 256 registers that two waves a SIMD leave
// each, the 256 x 256 tiles take 190 (bf16, transposed) to 218 (gradients), 128 of them sums.
//
// Edges cost nothing in the loop: every DMA goes through a buffer descriptor
// that ends where the tile's rows end, and what lies past it arrives in LDS as
// zeros.  Only a slab cut by K within ROW rows needs a lane to give up its chunk
// (an offset past the descriptor's end) and, 4-bit, scales of 1.  Rows and columns
// past the tile's edge hold zeros or neighbours and are not stored.
//
// Schedules.  PP ("ping-pong", 2 x 4 waves, one workgroup a CU): two groups of
// four waves, one of each on every SIMD, run half a step apart, so that one
// computes while the other reads LDS; the barriers and waits are those of
// gemm_bf16_pingpong.hpp.  Otherwise the plain loop: wait for the slab, barrier,
// start the DMA of the slab STAGES - 1 ahead, read, compute; several workgroups
// share a CU and fill each other's gaps.
//
// Few tiles of many rows (GRAD) are split over the rows, each group in as many
// parts as it has slabs, at most `splits`: fp32 partial planes that a second kernel
// adds up in order, all CUs at it (the last workgroup of each tile alone took 60 us
// of 83 for 32768 rows over 2 matrices of 256 x 512).
//
// Raster.  Tiles run in bands of (at most 8) tile rows, down the band first;
// 4 columns of a band go to one XCD (workgroups reach the XCDs in turn), whose
// 32 CUs then share 8 panels of A and 4 of B in its L2.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "gemm_bf16_pingpong.hpp"
#include "groups.hpp"

namespace xtc_hip {

struct DmaArgs {
  const uint8_t* a;   // ROW: [M] rows; GRAD: x, [M] rows of K columns
  const uint8_t* b;   // matrices of E groups, stride_b bytes apart; GRAD: dy
  const uint8_t* sa;  // scales of 4-bit operands, a byte a chunk
  const uint8_t* sb;
  const int* sizes;   // null: one group of all rows
  void* c;
  int64_t stride_b, stride_sb;  // bytes
  int64_t stride_c;             // elements (GRAD)
  int E, M, N;        // groups, rows in all, columns of C
  int K;              // GRAD: rows of C; otherwise 16-byte chunks of a row of A
  int lda, ldb;       // bytes
  int ldc;            // elements
  int tiles_m, tiles_n;  // tiles_m: of all groups (at most), GRAD: of one C
  int band;           // tile rows of a band
  int splits;         // GRAD: parts of a group's rows, at most
  float* partial;     // GRAD, splits > 1: [splits][E][K][N]
  int out16;          // C is bf16
};

namespace gdma {

using big::bf16x8;
using big::f32x4;
using big::i16x4;
using big::lds_i16x4;
using big::lds_u32x4;
using big::u32x4;
using big::waitcnt_vm;
using pingpong::phase_barrier;
using pingpong::waitcnt_lgkm0;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr unsigned PAST = 0x80000000u;  // an offset past every descriptor's end (they are shorter)

// Issued from asm, as in lds_dma.hpp: 16 bytes a lane from `off` (4-byte aligned)
// into buffer `r` go to LDS at `lds` + `ADD` + 16 lane; dwords past the
// descriptor's end arrive as zeros.  The wait states cover M0 and, in the FIRST
// one of a run, a descriptor written right before.
template <bool FIRST, int ADD>
__device__ __forceinline__ void dma16(u32x4 r, unsigned off, unsigned lds) {
  if constexpr (FIRST)
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 4\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r), "s"(lds),
                 "n"(ADD)
                 : "memory", "m0", "scc");
  else
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r), "s"(lds),
                 "n"(ADD)
                 : "memory", "m0", "scc");
}
__device__ __forceinline__ u32x4 descriptor(uint64_t at, unsigned bytes) {
  return u32x4{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, bytes, 0x00020000u};
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  typedef __attribute__((address_space(3))) void lds_void_t;
  return (unsigned)(uintptr_t)(lds_void_t*)p;
}

// The bytes of an operand that its next slab may touch, a slab after the other
// from slab `slab`, then from the start; none once all `left` slabs are done, so
// that the loops start a DMA with every step and wait for constant counts.  All
// of it is wave-uniform.
template <bool ROW, int SLAB>
struct Walk {
  uint64_t start, at;  // tile's corner in slab 0, in the next slab
  uint64_t step;       // bytes from a slab to the next
  int slab, slabs, left;
  int ld;              // COL: bytes of a k row
  unsigned width;      // ROW: bytes from the corner to the end; COL: of the last k row
  int depth;           // COL: k rows in all

  __device__ __forceinline__ u32x4 next() {
    unsigned bytes;
    if constexpr (ROW) bytes = width - (unsigned)(SLAB * slab);
    else bytes = (unsigned)((min(depth - 32 * slab, 32) - 1) * ld) + width;
    const u32x4 r = descriptor(at, left > 0 ? bytes : 0u);
    --left;
    ++slab;
    at += step;
    if (slab == slabs) slab = 0, at = start;
    return r;
  }
};

// A ds_read_b128 serves lanes 0-3, 12-15, 20-27 (and 4-11, 16-19, 28-31) at once: the
// chunk that 16-row (32-row) fragments find without bank conflicts
template <bool MX>
__device__ __forceinline__ int swz_row(int r) {
  return MX ? (r >> 1) & 7 : (r >> 1) & 3;
}
template <int COLS>
__device__ __forceinline__ int swz_col(int k) {
  return COLS >= 128 ? ((k & 3) | ((k >> 1) & 4)) : (k & 3);
}

// Where lane `lane` finds its 16 bytes of KB `kb` of an operand's stage: bytes
// from the operand's tile corner.
template <bool MX, bool ROW, int LEN>
__device__ __forceinline__ unsigned source(int kb, int lane, int ld) {
  if constexpr (ROW) {
    constexpr int CHUNKS = MX ? 8 : 4;
    const int r = kb * (64 / CHUNKS) + lane / CHUNKS;
    return (unsigned)r * (unsigned)ld + (unsigned)(((lane % CHUNKS) ^ swz_row<MX>(r)) * 16);
  } else {
    constexpr int SLOTS = LEN / 8, PER = 64 / SLOTS;  // 16-byte slots of a k row, k rows of a KB
    const int k = kb * PER + lane / SLOTS, slot = lane % SLOTS;
    return (unsigned)k * (unsigned)ld + (unsigned)(((slot >> 1) ^ swz_col<LEN>(k)) * 32 + (slot & 1) * 16);
  }
}

// Fragment `f` (16 rows or columns from f0) of an operand's stage.
template <bool ROW, int LEN>
__device__ __forceinline__ u32x4 fragment(const unsigned char* st, int f0, int f, int l16, int g) {
  if constexpr (ROW) {
    const int r = (f0 + f) * 16 + l16;
    return *(const lds_u32x4*)(st + r * 64 + 16 * (g ^ swz_row<false>(l16)));
  } else {
    const int k = 8 * g + (l16 >> 2);
    const unsigned char* p = st + k * (2 * LEN) + 32 * ((f0 + f) ^ swz_col<LEN>(k)) + 8 * (l16 & 3);
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p);
    const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 8 * LEN));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

__device__ __forceinline__ f32x4 mfma(u32x4 b, u32x4 a, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
// 4-bit; the scales are byte `BYTE` of sa and sb
template <int BYTE>
__device__ __forceinline__ f32x16 mfma(u32x4 b, unsigned sb, u32x4 a, unsigned sa, f32x16 c) {
  const i32x8 bv = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(bv, av, c, 4, 4, BYTE, (int)sb, BYTE, (int)sa);
}

// columns n .. n+3 (those below `cols`) of a row
__device__ __forceinline__ void store4(void* c, int out16, int64_t at, f32x4 v, int n, int cols, bool whole) {
  if (out16) {
    __bf16* p = (__bf16*)c + at + n;
    const bf16x4 h = __builtin_convertvector(v, bf16x4);
    if (whole && n + 4 <= cols) *(bf16x4*)p = h;
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < cols) p[i] = h[i];
  } else {
    float* p = (float*)c + at + n;
    if (whole && n + 4 <= cols) *(f32x4*)p = v;
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < cols) p[i] = v[i];
  }
}

// Into how many parts the rows of a group of `slabs` slabs go.
__device__ __forceinline__ int gradient_parts(int slabs, int splits) { return max(min(splits, slabs), 1); }

// f(0) .. f(N - 1), the argument a compile-time constant
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each_stage(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    each_stage<N, I + 1>(f);
  }
}

}  // namespace gdma

template <bool MX, bool GRAD, bool B_ROW, int WGM, int WGN, int TM, int TN, int STAGES, bool PP>
__global__ void __launch_bounds__(WGM* WGN * 64) grouped_dma(DmaArgs p) {
  using namespace gdma;
  constexpr bool A_ROW = !GRAD;
  constexpr int WAVES = WGM * WGN, BM = WGM * TM * 16, BN = WGN * TN * 16;
  constexpr int SLAB = MX ? 128 : 64, CHUNKS = SLAB / 16, HALVES = SLAB / 64;  // bytes, 16-byte chunks, steps of a row
  constexpr int A_KB = BM * SLAB / 1024, B_KB = BN * SLAB / 1024, PER = (A_KB + B_KB) / WAVES;  // DMA kilobytes
  constexpr int S_ALL = MX ? (BM + BN) / 64 : 0;        // scale DMA of two slabs: 64 rows each
  constexpr int S_PER = (S_ALL + WAVES - 1) / WAVES;    // a wave's with every second slab
  constexpr int A_AT = 0, B_AT = BM * SLAB, STAGE = B_AT + BN * SLAB;
  constexpr int S_STAGE = S_ALL * 1024, S_STAGES = 2;
  constexpr int D = STAGES - 1;
  static_assert(PER * WAVES == A_KB + B_KB && A_KB % PER == 0, "a slab splits evenly over the waves, one operand each");
  static_assert(!MX || (B_ROW && !GRAD), "4-bit operands have k along their rows");
  static_assert(!PP || (WGM == 2 && WGN == 4), "two groups of four waves");
  static_assert(STAGES * STAGE + S_STAGES * S_STAGE <= 160 * 1024 && D * PER + S_PER < 64, "LDS and wait counts");
  static_assert(STAGES % 2 == 0 && STAGES <= 4, "a slab's place in its pair follows from its stage; scales are read in time");

  __shared__ __attribute__((aligned(1024))) unsigned char lds[STAGES * STAGE + S_STAGES * S_STAGE];
  unsigned char* const lds_s = lds + STAGES * STAGE;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const int l16 = lane & 15, g = lane >> 4;

  // ---- the workgroup's tile
  const int slot = blockIdx.x >> 3, run = 4 * p.band;  // run: tiles that follow one another on an XCD
  const int t = (slot / run * 8 + (blockIdx.x & 7)) * run + slot % run;
  const int per_matrix = (p.tiles_m + p.band - 1) / p.band * p.band * p.tiles_n;
  const int matrix = GRAD ? t / per_matrix : 0;  // part by part
  const int e_grad = GRAD ? matrix % p.E : 0;
  const int part = GRAD ? matrix / p.E : 0;
  const int tt = GRAD ? t - matrix * per_matrix : t;
  const int in_band = tt % (p.band * p.tiles_n);
  const int mt = tt / (p.band * p.tiles_n) * p.band + in_band % p.band, n0 = in_band / p.band * BN;
  if (mt >= p.tiles_m || (GRAD && part >= p.splits)) return;

  const uint8_t *a, *b;                        // tile corners
  const uint8_t *as = nullptr, *bs = nullptr;  // and those of the scales
  int64_t c_at;              // element of C at the tile's corner
  int rows, nk, chunks = 0;  // rows of C, slabs, 16-byte chunks of a ROW row
  int depth = 0;             // k rows of a COL operand
  int parts = 1;             // of the group's rows
  const int cols = p.N - n0;
  if constexpr (GRAD) {
    const RowGroup gr = find_group(p.sizes, p.E, p.M, e_grad);
    const int m0 = mt * BM;
    rows = p.K - m0;
    // this part's slabs of the group's
    const int slabs = (gr.end - gr.begin + 31) / 32;
    parts = gradient_parts(slabs, p.splits);
    if (part >= parts) return;
    const int first = (int)((int64_t)slabs * part / parts);
    nk = (int)((int64_t)slabs * (part + 1) / parts) - first;
    const int64_t row0 = gr.begin + 32 * (int64_t)first;
    depth = (int)min((int64_t)32 * nk, gr.end - row0);
    a = p.a + row0 * p.lda + 2 * (int64_t)m0;
    b = p.b + row0 * p.ldb + 2 * (int64_t)n0;
    c_at = (int64_t)e_grad * p.stride_c + (int64_t)m0 * p.ldc + n0;
  } else {
    RowGroup gr{0, mt * BM, p.M};
    if (p.sizes) gr = find_tile<BM>(p.sizes, p.E, p.M, mt);
    if (gr.e < 0) return;
    const int e = gr.e < p.E ? gr.e : 0;
    rows = min(gr.end - gr.begin, BM);
    chunks = gr.e < p.E ? p.K : 0;  // rows of no group: zeros
    depth = 8 * chunks;
    nk = (chunks + CHUNKS - 1) / CHUNKS;
    a = p.a + (int64_t)gr.begin * p.lda;
    b = p.b + e * p.stride_b + (B_ROW ? (int64_t)n0 * p.ldb : 2 * (int64_t)n0);
    if constexpr (MX) {
      as = p.sa + (int64_t)gr.begin * chunks;
      bs = p.sb + e * p.stride_sb + (int64_t)n0 * chunks;
    }
    c_at = (int64_t)gr.begin * p.ldc + n0;
  }

  // ---- this wave's share of a slab's DMA: PER kilobytes of one operand
  const bool is_a = wave * PER < A_KB;
  const int kb0 = is_a ? wave * PER : wave * PER - A_KB;  // in the operand's stage
  const int ld = is_a ? p.lda : p.ldb;
  const int lines = is_a ? min(rows, BM) : min(cols, BN);  // rows (ROW) or columns (COL) of the operand in the tile
  // Where the lane finds its 16 bytes of each KB: the pattern of 4-bit rows repeats
  // after two KB (16 rows)
  constexpr int OFFS = MX ? 2 : PER;
  unsigned off[OFFS];
#pragma unroll
  for (int i = 0; i < OFFS; ++i) off[i] = is_a ? source<MX, A_ROW, BM>(kb0 + i, lane, ld) : source<MX, B_ROW, BN>(kb0 + i, lane, ld);
  auto offset = [&](int i, int step) { return off[i % OFFS] + (unsigned)(i / OFFS) * (unsigned)step; };
  // the chunk of a ROW slab that it loads
  auto chunk = [&](int i) { return (lane % CHUNKS) ^ swz_row<MX>((kb0 + i % OFFS) * (64 / CHUNKS) + lane / CHUNKS); };
  // K stagger: tiles that share a panel start their walk at different slabs
  // (bf16 8192^3 850 -> 830 us; 4-bit slabs go in pairs, and gain nothing by it)
  const int kofs = !MX && nk > 0 ? ((mt + 2 * (n0 / BN)) & 15) % nk : 0;
  const bool row = is_a ? A_ROW : B_ROW;
  Walk<true, SLAB> by_row;
  Walk<false, SLAB> by_col;
  if (row) {
    by_row.start = (uint64_t)(is_a ? a : b);
    by_row.step = SLAB;
    by_row.width = (unsigned)(lines - 1) * (unsigned)ld + 16u * (unsigned)chunks;
    by_row.slab = kofs, by_row.slabs = by_row.left = nk;
    by_row.at = by_row.start + (uint64_t)kofs * SLAB;
  } else {
    by_col.start = (uint64_t)(is_a ? a : b);
    by_col.step = (uint64_t)32 * (uint64_t)ld;
    by_col.ld = ld, by_col.width = 2u * (unsigned)lines, by_col.depth = depth;
    by_col.slab = kofs, by_col.slabs = by_col.left = nk;
    by_col.at = by_col.start + (uint64_t)kofs * by_col.step;
  }
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds)), share = (unsigned)((is_a ? 0 : B_AT) + kb0 * 1024);

  // Scales of slabs 2 q and 2 q + 1, in the place of slabs 2 q - 4 and 2 q - 3, whose
  // scales everyone has read with the first: slab 2 q - STAGES is read.  Past the
  // last slab they are the next row's or zeros, and nobody reads them
  const int s_kb = min(wave * S_PER, S_ALL - S_PER);  // a wave without a share repeats the last one
  const bool s_is_a = s_kb < BM / 64;
  const uint64_t s_at = (uint64_t)(s_is_a ? as : bs);
  const unsigned s_bytes = (unsigned)(s_is_a ? min(rows, BM) : min(cols, BN)) * (unsigned)chunks;
  const unsigned s_off = (unsigned)((s_is_a ? s_kb : s_kb - BM / 64) * 64 + lane) * (unsigned)chunks;
  auto issue_scales = [&](int q) {
    static_assert(S_PER <= 1, "one DMA of scales a wave");
    dma16<true, 0>(descriptor(s_at + 16 * (uint64_t)q, (unsigned)max((int)s_bytes - 16 * q, 0)), s_off,
                   lds0 + STAGES * STAGE + q % S_STAGES * S_STAGE + s_kb * 1024);
  };

  auto issue = [&](int kt, const int stage) {
    const unsigned at = lds0 + share + stage * STAGE;
    int step = 16 * ld;  // opaque: the sums of a lane's offsets would fill the registers
    if constexpr (MX) asm volatile("" : "+s"(step));
    if (row) {
      const int left = chunks - CHUNKS * by_row.slab;
      const u32x4 r = by_row.next();
      if (left < CHUNKS) {
        each_stage<PER>([&](auto i) { dma16<i == 0, i * 1024>(r, chunk(i) < left ? offset(i, step) : PAST, at); });
      } else {
        each_stage<PER>([&](auto i) { dma16<i == 0, i * 1024>(r, offset(i, step), at); });
      }
    } else {
      const u32x4 r = by_col.next();
      each_stage<PER>([&](auto i) { dma16<i == 0, i * 1024>(r, offset(i, step), at); });
    }
    if (MX && kt % 2 == 0) issue_scales(kt / 2);
  };

  // DMA instructions of this wave's slabs kt+first .. kt+last, kt % STAGES == s
  auto dma_count = [](int s, int first, int last) constexpr {
    int n = 0;
    for (int i = first; i <= last; ++i) n += PER + (MX && (s + i) % 2 == 0 ? S_PER : 0);
    return n;
  };

  // 16 x 16 tiles of bf16, or 32 x 32 tiles of 4-bit products
  constexpr int IM = MX ? TM / 2 : TM, JN = MX ? TN / 2 : TN, STEPS = MX ? 2 : 1;
  typedef std::conditional_t<MX, f32x16, f32x4> Acc;
  Acc acc[IM][JN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < JN; ++j) acc[i][j] = Acc{};

  u32x4 fa[STEPS][IM], fb[STEPS][JN];
  unsigned ha[IM][2], hb[JN][2];  // scales of this lane's row and half of k, of a pair of slabs
  const int l32 = lane & 31, half = lane >> 5;
  // half `hf` (64 bytes a row) of slab kt
  auto read = [&](int kt, const int s, const int hf, const unsigned char* st) {
    if constexpr (MX) {
      // chunk 4 hf + 2 h + half of the lane's rows; kept from being worked out for
      // every stage ahead of the loop, which registers do not suffice for
      unsigned at = (unsigned)(l32 * SLAB + 16 * (half ^ swz_row<MX>(l32)));
      asm volatile("" : "+v"(at));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned char* const rows = st + (at ^ (unsigned)(16 * (4 * hf + 2 * h)));
#pragma unroll
        for (int i = 0; i < IM; ++i) fa[h][i] = *(const lds_u32x4*)(rows + A_AT + (wm * IM + i) * 32 * SLAB);
#pragma unroll
        for (int j = 0; j < JN; ++j) fb[h][j] = *(const lds_u32x4*)(rows + B_AT + (wn * JN + j) * 32 * SLAB);
      }
      if (s % 2 == 0 && hf == 0) {
        const unsigned char* ss = lds_s + kt / 2 % S_STAGES * S_STAGE + l32 * 16;
        const unsigned pick = half ? 0x07050301u : 0x06040200u;
        auto keep = [&](unsigned (&h)[2], int row) {
          const u32x4 v = *(const lds_u32x4*)(ss + row * 16);
          h[0] = __builtin_amdgcn_perm(v[1], v[0], pick);
          h[1] = __builtin_amdgcn_perm(v[3], v[2], pick);
        };
#pragma unroll
        for (int i = 0; i < IM; ++i) keep(ha[i], (wm * IM + i) * 32);
#pragma unroll
        for (int j = 0; j < JN; ++j) keep(hb[j], BM + (wn * JN + j) * 32);
      }
      // a last slab of four blocks: the others' codes are zeros, scaled by 1
      if (hf == 1 && kt == nk - 1 && (chunks & 4)) {
#pragma unroll
        for (int i = 0; i < IM; ++i) ha[i][s % 2] = (ha[i][s % 2] & 0xffffu) | 0x7f7f0000u;
#pragma unroll
        for (int j = 0; j < JN; ++j) hb[j][s % 2] = (hb[j][s % 2] & 0xffffu) | 0x7f7f0000u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < IM; ++i) fa[0][i] = fragment<A_ROW, BM>(st + A_AT, wm * TM, i, l16, g);
#pragma unroll
      for (int j = 0; j < JN; ++j) fb[0][j] = fragment<B_ROW, BN>(st + B_AT, wn * TN, j, l16, g);
    }
  };
  auto mma = [&](const int s, const int hf) {
#pragma unroll
    for (int h = 0; h < STEPS; ++h)
#pragma unroll
      for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < JN; ++j) {
          if constexpr (MX) {
            const unsigned sb = hb[j][s % 2], sa = ha[i][s % 2];
            const int byte = 2 * hf + h;
            acc[i][j] = byte == 0 ? mfma<0>(fb[h][j], sb, fa[h][i], sa, acc[i][j])
                        : byte == 1 ? mfma<1>(fb[h][j], sb, fa[h][i], sa, acc[i][j])
                        : byte == 2 ? mfma<2>(fb[h][j], sb, fa[h][i], sa, acc[i][j])
                                    : mfma<3>(fb[h][j], sb, fa[h][i], sa, acc[i][j]);
          } else {
            acc[i][j] = mfma(fb[h][j], fa[h][i], acc[i][j]);
          }
        }
  };

  // keeps the products of a compute phase within it
  auto settle = [&] {
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
      for (int j = 0; j < JN; ++j) asm volatile("" : "+v"(acc[i][j]));
  };

  if (nk > 0) {
    each_stage<D>([&](auto s) { issue(s, s); });
    if constexpr (PP) {
      const int group = wm;
      __builtin_amdgcn_s_waitcnt(waitcnt_vm(dma_count(0, 1, D - 1)));
      phase_barrier();
      if (group == 1) phase_barrier();
      auto step = [&](int kt, auto stage) {
        constexpr int s = decltype(stage)::value;
        each_stage<HALVES>([&](auto hf) {
          constexpr bool last = hf == HALVES - 1;
          // ---- memory phase
          if (hf == 0) issue(kt + D, (s + D) % STAGES);
          read(kt, s, hf, lds + s * STAGE);
          __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0());
          // this wave's DMA of slab kt+1 has landed: group 0 waits after computing
          if (last && group == 1) __builtin_amdgcn_s_waitcnt(waitcnt_vm(dma_count(s, 2, D)));
          phase_barrier();
          // ---- compute phase, ahead of the SIMD's other wave
          __builtin_amdgcn_s_setprio(1);
          mma(s, hf);
          if constexpr (MX) settle();
          __builtin_amdgcn_s_setprio(0);
          __builtin_amdgcn_sched_barrier(0);
          if (last && group == 0) __builtin_amdgcn_s_waitcnt(waitcnt_vm(dma_count(s, 2, D)));
          phase_barrier();
        });
      };
      for (int kt = 0; kt < nk; kt += STAGES) each_stage<STAGES>([&](auto s) { if (kt + s < nk) step(kt + s, s); });
      if (group == 0) phase_barrier();
    } else {
      auto step = [&](int kt, auto stage) {
        constexpr int s = decltype(stage)::value;
        // slab kt has landed; the ones after it may be in flight
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(dma_count(s, 1, D - 1)));
        // everyone has read slab kt-1, whose stage the DMA now fills
        __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0());
        phase_barrier();
        issue(kt + D, (s + D) % STAGES);
        each_stage<HALVES>([&](auto hf) {
          read(kt, s, hf, lds + s * STAGE);
          mma(s, hf);
        });
      };
      for (int kt = 0; kt < nk; kt += STAGES) each_stage<STAGES>([&](auto s) { if (kt + s < nk) step(kt + s, s); });
    }
    // no DMA may write LDS after the workgroup has left it
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
  }

  if constexpr (GRAD) {
    if (parts > 1) {
      // whole quads of columns: N is one of whole vectors
      float* const tile = p.partial + (((size_t)part * p.E + e_grad) * p.K + (p.K - rows)) * p.N + n0;
#pragma unroll
      for (int i = 0; i < IM; ++i) {
        const int m = (wm * IM + i) * 16 + l16;
#pragma unroll
        for (int j = 0; j < JN; ++j) {
          const int n = (wn * JN + j) * 16 + 4 * g;
          if (m < rows && n < cols) *(f32x4*)(tile + (size_t)m * p.N + n) = acc[i][j];
        }
      }
      return;
    }
  }

  // ---- a lane holds C[m][n .. n+3] of each 16 x 16, or n, n+8, n+16 and n+24 of
  // each 32 x 32
  const bool whole = (p.ldc & 3) == 0 && ((uintptr_t)p.c & (p.out16 ? 7 : 15)) == 0 && (!GRAD || (p.stride_c & 3) == 0);
#pragma unroll
  for (int i = 0; i < IM; ++i) {
    const int m = MX ? (wm * IM + i) * 32 + l32 : (wm * IM + i) * 16 + l16;
    if (m >= rows) continue;
    const int64_t at = c_at + (int64_t)m * p.ldc;
#pragma unroll
    for (int j = 0; j < JN; ++j) {
      if constexpr (MX) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          store4(p.c, p.out16, at, f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]},
                 (wn * JN + j) * 32 + 8 * q + 4 * half, cols, whole);
      } else {
        store4(p.c, p.out16, at, acc[i][j], (wn * JN + j) * 16 + 4 * g, cols, whole);
      }
    }
  }
}

// Adds up the parts of the groups that have more than one, in order: a thread
// four columns, `chunks` workgroups a matrix.
static __global__ void __launch_bounds__(256) grouped_grad_sum(DmaArgs p, int chunks) {
  using namespace gdma;
  const int e = blockIdx.x / chunks;
  const RowGroup gr = find_group(p.sizes, p.E, p.M, e);
  const int parts = gradient_parts((gr.end - gr.begin + 31) / 32, p.splits);
  if (parts == 1) return;
  const int64_t q = (int64_t)(blockIdx.x % chunks) * 256 + threadIdx.x;
  const int quads = p.N / 4, m = (int)(q / quads), n = (int)(q % quads) * 4;
  if (m >= p.K) return;
  const size_t plane = (size_t)p.E * p.K * p.N;
  const float* const at = p.partial + ((size_t)e * p.K + m) * p.N + n;
  f32x4 v = *(const f32x4*)at;
  for (int s0 = 1; s0 < parts; s0 += 8) {
    f32x4 t[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = *(const f32x4*)(at + min(s0 + j, parts - 1) * plane);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (s0 + j < parts) v += t[j];
  }
  const bool whole = (p.ldc & 3) == 0 && (p.stride_c & 3) == 0 && ((uintptr_t)p.c & (p.out16 ? 7 : 15)) == 0;
  store4(p.c, p.out16, e * p.stride_c + (int64_t)m * p.ldc, v, n, p.N, whole);
}

// What a tile's slab costs, from which the calls choose their tiles: microseconds
// where a CU has one workgroup and the others none, and where every CU is full.
struct DmaCost {
  int bm, bn, per_cu;
  double light, full;
};
// `tiles` of `slabs` on 256 CUs, without what every tile has in common.  A round of
// tiles ends with writing them out, a CU 24 bytes a nanosecond.  Small tiles even out
// over the CUs (a last round of few 128 x 128 ones still costs half a full one: 4096
// rows over 8 experts of 4096 x 2048, 1.1 rounds of them 128 us, one of 256 x 256
// tiles 116); a 256 x 256 one takes a CU for itself, so nothing hides its first loads
// (2 us) and a last round costs as much as a full one.
inline double dma_cost(const DmaCost& c, double tiles, double slabs, int out_bytes) {
  const double load = tiles / (256.0 * c.per_cu), out = c.per_cu * c.bm * c.bn * out_bytes / 24e3 + (c.per_cu == 1 ? 2 : 0);
  if (load <= 1) return slabs * (c.light + (c.full - c.light) * load) + out;
  return (slabs * c.full + out) * (load + (ceil(load) - load) / c.per_cu);
}
// Tiles of bm rows that a fair share of T rows to E groups makes.
inline double likely_tiles(double T, double E, int bm) {
  return E == 1 ? ceil(T / bm) : fmax(fmin(E, T), T / bm + 0.5 * fmin(E, T));
}

// Workgroups of `a` (its tiles and band set): bands and runs filled up.
inline int64_t dma_groups(const DmaArgs& a, int64_t matrices) {
  const int64_t per_matrix = ((int64_t)a.tiles_m + a.band - 1) / a.band * a.band * a.tiles_n;
  const int64_t whole = (int64_t)8 * 4 * a.band;
  return (matrices * per_matrix + whole - 1) / whole * whole;
}

}  // namespace xtc_hip
