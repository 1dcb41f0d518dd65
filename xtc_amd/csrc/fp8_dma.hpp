// SPDX-License-Identifier: BSD-3-Clause
// Products of 8-bit floats with a scale for every 128 elements (fp8.hpp), staged
// through LDS by DMA:
//   C[m, n] = sum_k A[m, k] B[n, k], both operands with k along their rows.
//
// Which instructions.  v_mfma_scale_f32_32x32x64_f8f6f4 takes the codes and scales as they
// are, at twice the rate of bf16 ones (registers only, random codes: 3.3-3.8 PFLOP/s
// against 1.9-2.0), but adds up eight products at a time with 16 bits below the
// largest (2^16 + 1 gives 2^16 within eight neighbours, 2^16 + 2^-7 across): sums are
// off by 1.5e-5 of themselves for normal data, and by up to 2^-12 of the sum of the
// products' magnitudes (each of the eight by less than 2^-15 of the largest).  A caller may
// choose them (FAST).  Otherwise v_mfma_f32_32x32x16_bf16 takes the codes' values in bf16,
// scaled on the way, with fp32 sums.  The 8-bit instructions without scales (16x16x32) add
// up likewise and are no faster than bf16 ones.  All tiles add k up in the same order, a
// slab after another: a row's result does not depend on the tile.
//
// Tile and slab.  A workgroup of WGM x WGN waves computes (32 WGM TM) x (32 WGN TN)
// outputs, k in slabs of 64 bytes of a row, half a block.  k may be summed in any order
// as long as A and B agree, and all of a row's slab has one scale: a lane takes 32
// bytes of its row at once (FAST) or two times 16.  B is the first operand: a lane
// ends with runs of four neighbouring columns of one row.
//
// Slabs are staged [rows][64 bytes], 16-byte chunk c of row r at c ^ ((r >> 3) & 3): a
// ds_read_b128 of 32-row fragments serves lanes 0-3, 12-15, 20-27 at once, which then
// find all banks.  DMA, walk and descriptors are those of grouped_dma.hpp: what lies
// past the tile's rows arrives as zeros, rows are whole blocks, so that no slab is cut.
//
// Scales.  SCALES blocks of k of the tile's rows are copied to LDS by ordinary loads
// (any alignment) before the slabs of those blocks are walked; a lane reads four
// blocks' bytes of its rows at once.  A walk ends after SCALES blocks (8192 elements)
// and the next begins.
//
// Schedules.  PLAIN: a barrier a slab, two or more workgroups a CU cover each other's
// waits.  AHEAD (256 x 256, FAST): four waves of 128 x 128, one a SIMD with all of its
// registers, read the next slab's fragments between this one's matrix instructions: two
// thirds of the LDS reads of eight waves of 128 x 64.  Its loop spills nothing; before the
// stores, unrolled over 16 tiles, 32 registers are put aside and read back (8 KB a wave, 34
// MB at 8192 x 8192).  PINGPONG, as in grouped_dma.hpp:
// eight waves, one of a SIMD's two computes while the other reads and converts.  At 8192 x
// 8192 x 8192 with 8-bit sums AHEAD takes 483 us (2.3 PFLOP/s), PINGPONG 511; for fp32
// sums conversions need the second wave.
//
// The tiles walk k in step.  With the walks staggered, which spreads the first loads over
// the memory channels, an XCD's L2 no longer holds what its tiles share: 600 us.
#pragma once
#include "fp8_scales.hpp"
#include "grouped_dma.hpp"

namespace xtc_hip {

struct Fp8Args {
  const uint8_t *a, *b;    // codes [M], [N] rows of 128 blocks bytes
  const uint8_t *sa, *sb;  // scales [M][blocks]; [N][blocks] or [ceil(N / 128)][blocks]
  void* c;
  int M, N, blocks, ldc;
  int b_shift;             // log2 of the rows of b that share a scale
  int tiles_m, tiles_n, band;
  int out16;               // C is bf16
};

namespace fp8 {

enum Schedule { PLAIN, PINGPONG, AHEAD };

__device__ __forceinline__ gdma::f32x16 mfma(const gdma::u32x4 (&b)[2], unsigned sb, const gdma::u32x4 (&a)[2], unsigned sa, gdma::f32x16 c) {
  using gdma::i32x8;
  const i32x8 bv = {(int)b[0][0], (int)b[0][1], (int)b[0][2], (int)b[0][3], (int)b[1][0], (int)b[1][1], (int)b[1][2], (int)b[1][3]};
  const i32x8 av = {(int)a[0][0], (int)a[0][1], (int)a[0][2], (int)a[0][3], (int)a[1][0], (int)a[1][1], (int)a[1][2], (int)a[1][3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(bv, av, c, 0, 0, 0, (int)sb, 0, (int)sa);
}

}  // namespace fp8

template <bool FAST, int WGM, int WGN, int TM, int TN, int STAGES, fp8::Schedule SCHEDULE>
__global__ void __launch_bounds__(WGM* WGN * 64) fp8_dma(Fp8Args p) {
  using namespace gdma;
  constexpr int WAVES = WGM * WGN, BM = WGM * TM * 32, BN = WGN * TN * 32;
  constexpr int SLAB = 64, HALVES = FAST ? 1 : 2;  // steps of a slab
  constexpr int A_KB = BM * SLAB / 1024, B_KB = BN * SLAB / 1024;  // DMA kilobytes
  constexpr int A_PER = A_KB / WAVES, B_PER = B_KB / WAVES, PER = A_PER + B_PER;
  constexpr int B_AT = BM * SLAB, STAGE = B_AT + BN * SLAB;
  constexpr bool PP = SCHEDULE == fp8::PINGPONG, RP = SCHEDULE == fp8::AHEAD;
  constexpr int D = RP ? STAGES : STAGES - 1;  // slabs on their way before the first is waited for
  static_assert(A_PER * WAVES == A_KB && B_PER * WAVES == B_KB, "a slab splits evenly over the waves");
  static_assert(!PP || (WGM == 2 && WGN == 4), "two groups of four waves");
  static_assert(STAGES == 4, "a slab's half of its block follows from its stage");
  static_assert(STAGES * STAGE + (BM + BN) * fp8::SCALES <= 160 * 1024 && D * PER < 64, "LDS and wait counts");

  __shared__ __attribute__((aligned(1024))) unsigned char lds[STAGES * STAGE + (BM + BN) * fp8::SCALES];
  unsigned char* const lds_s = lds + STAGES * STAGE;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const int l32 = lane & 31, half = lane >> 5;

  // ---- the workgroup's tile, bands and XCDs as in grouped_dma
  const int slot = blockIdx.x >> 3, run = 4 * p.band;
  const int t = (slot / run * 8 + (blockIdx.x & 7)) * run + slot % run;
  const int in_band = t % (p.band * p.tiles_n);
  const int mt = t / (p.band * p.tiles_n) * p.band + in_band % p.band, nt = in_band / p.band;
  if (mt >= p.tiles_m) return;
  const int m0 = mt * BM, n0 = nt * BN;
  const int rows = min(p.M - m0, BM), cols = min(p.N - n0, BN);
  const int ld = 128 * p.blocks;

  // ---- this wave's share of a slab's DMA: A_PER kilobytes of A, B_PER of B
  // a lane's 16 bytes of KB i: the pattern repeats after two KB (32 rows)
  const int a_kb = wave * A_PER, b_kb = wave * B_PER;
  unsigned a_off[2], b_off[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int ra = (a_kb + i) * 16 + lane / 4, rb = (b_kb + i) * 16 + lane / 4;
    a_off[i] = (unsigned)ra * (unsigned)ld + (unsigned)(((lane % 4) ^ fp8::swz(ra)) * 16);
    b_off[i] = (unsigned)rb * (unsigned)ld + (unsigned)(((lane % 4) ^ fp8::swz(rb)) * 16);
  }
  const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds));

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};

  for (int first = 0; first < p.blocks; first += fp8::SCALES) {
    const int blocks = min(p.blocks - first, fp8::SCALES), nk = 2 * blocks;
    auto walk_of = [&](const uint8_t* operand, int row, int lines) {
      Walk<true, SLAB> w;
      w.start = (uint64_t)(operand + (int64_t)row * ld) + (uint64_t)128 * first;
      w.step = SLAB;
      w.width = (unsigned)(lines - 1) * (unsigned)ld + 128u * (unsigned)blocks;
      w.slab = 0, w.slabs = w.left = nk;
      w.at = w.start;
      return w;
    };
    Walk<true, SLAB> walk_a = walk_of(p.a, m0, rows), walk_b = walk_of(p.b, n0, cols);
    auto issue = [&](const int stage) {
      const unsigned at = lds0 + stage * STAGE;
      int step = 32 * ld;  // opaque: the sums of a lane's offsets would fill the registers
      asm volatile("" : "+s"(step));
      const u32x4 ra = walk_a.next();
      each_stage<A_PER>([&](auto i) { dma16<i == 0, i * 1024>(ra, a_off[i % 2] + (unsigned)(i / 2) * (unsigned)step, at + a_kb * 1024); });
      const u32x4 rb = walk_b.next();
      each_stage<B_PER>([&](auto i) { dma16<i == 0, i * 1024>(rb, b_off[i % 2] + (unsigned)(i / 2) * (unsigned)step, at + B_AT + b_kb * 1024); });
    };

    if (first) __syncthreads();  // everyone is done with the last walk
    each_stage<D>([&](auto s) { issue(s); });
    // ---- the walk's scales: rows past the edge keep what was there, no one stores theirs
    for (int r = threadIdx.x; r < BM + BN; r += 64 * WAVES) {
      const bool of_a = r < BM;
      const int row = of_a ? r : r - BM;
      if (row >= (of_a ? rows : cols)) continue;
      const uint8_t* const from = (of_a ? p.sa + (int64_t)(m0 + row) * p.blocks : p.sb + (int64_t)((n0 + row) >> p.b_shift) * p.blocks) + first;
#pragma unroll
      for (int q = 0; q < fp8::SCALES / 16; ++q) {
        u32x4 v = {0, 0, 0, 0};
        if (16 * q + 16 <= blocks) {
          __builtin_memcpy(&v, from + 16 * q, 16);
        } else if (16 * q < blocks) {
          unsigned char* const at = lds_s + r * fp8::SCALES + 16 * (q ^ fp8::swz(r));
          for (int i = 0; i < blocks - 16 * q; ++i) at[i] = from[16 * q + i];
          continue;
        }
        *(u32x4*)(lds_s + r * fp8::SCALES + 16 * (q ^ fp8::swz(r))) = v;
      }
    }
    __syncthreads();

    u32x4 fa[TM][2], fb[TN][2];  // FAST: codes of 32 elements; otherwise 16 of them in bf16
    unsigned ha[TM], hb[TN];     // scales of this lane's rows, four blocks
    int at = 0;                  // slab of the walk
    auto scales = [&] {
#pragma unroll
      for (int i = 0; i < TM; ++i) ha[i] = *(const unsigned*)(lds_s + fp8::scales_at((wm * TM + i) * 32 + l32, at));
#pragma unroll
      for (int j = 0; j < TN; ++j) hb[j] = *(const unsigned*)(lds_s + fp8::scales_at(BM + (wn * TN + j) * 32 + l32, at));
    };
    auto convert = [](u32x4 (&to)[2], u32x4 v, unsigned h) {
      const float scale = fp8::scale_of_byte(h & 255);
#pragma unroll
      for (int c = 0; c < 2; ++c) to[c] = __builtin_bit_cast(u32x4, fp8::values_bf16(v[2 * c], v[2 * c + 1], scale));
    };
    auto read = [&](const int s, const int hf, const unsigned char* st) {
      if (s % 2 == 0 && hf == 0)
        if ((at & 7) == 0) scales();
      if constexpr (FAST) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char* const at_row = st + l32 * SLAB + 16 * ((2 * half + h) ^ fp8::swz(l32));
#pragma unroll
          for (int i = 0; i < TM; ++i) fa[i][h] = *(const lds_u32x4*)(at_row + (wm * TM + i) * 32 * SLAB);
#pragma unroll
          for (int j = 0; j < TN; ++j) fb[j][h] = *(const lds_u32x4*)(at_row + B_AT + (wn * TN + j) * 32 * SLAB);
        }
      } else {
        const unsigned char* const at_row = st + l32 * SLAB + 16 * ((2 * hf + half) ^ fp8::swz(l32));
        u32x4 ra[TM], rb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) ra[i] = *(const lds_u32x4*)(at_row + (wm * TM + i) * 32 * SLAB);
#pragma unroll
        for (int j = 0; j < TN; ++j) rb[j] = *(const lds_u32x4*)(at_row + B_AT + (wn * TN + j) * 32 * SLAB);
#pragma unroll
        for (int i = 0; i < TM; ++i) convert(fa[i], ra[i], ha[i]);
#pragma unroll
        for (int j = 0; j < TN; ++j) convert(fb[j], rb[j], hb[j]);
      }
    };
    auto mma = [&](const int s, const int hf) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if constexpr (FAST) {
            acc[i][j] = fp8::mfma(fb[j], hb[j], fa[i], ha[i], acc[i][j]);
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, fb[j][c]), __builtin_bit_cast(bf16x8, fa[i][c]), acc[i][j], 0, 0, 0);
          }
        }
      if (hf < HALVES - 1) return;
      ++at;
      if (s % 2 == 1) {  // the next block's bytes
#pragma unroll
        for (int i = 0; i < TM; ++i) ha[i] >>= 8;
#pragma unroll
        for (int j = 0; j < TN; ++j) hb[j] >>= 8;
      }
    };

    if constexpr (PP) {
      const int group = wm;
      __builtin_amdgcn_s_waitcnt(waitcnt_vm((D - 1) * PER));
      phase_barrier();
      if (group == 1) phase_barrier();
      auto step = [&](auto stage) {
        constexpr int s = decltype(stage)::value;
        each_stage<HALVES>([&](auto hf) {
          constexpr bool last = hf == HALVES - 1;
          // ---- memory phase
          if (hf == 0) issue((s + D) % STAGES);
          read(s, hf, lds + s * STAGE);
          __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0());
          // this wave's DMA of the next slab has landed: group 0 waits after computing
          if (last && group == 1) __builtin_amdgcn_s_waitcnt(waitcnt_vm((D - 1) * PER));
          phase_barrier();
          // ---- compute phase, ahead of the SIMD's other wave
          __builtin_amdgcn_s_setprio(1);
          mma(s, hf);
          __builtin_amdgcn_s_setprio(0);
          __builtin_amdgcn_sched_barrier(0);
          if (last && group == 0) __builtin_amdgcn_s_waitcnt(waitcnt_vm((D - 1) * PER));
          phase_barrier();
        });
      };
      for (int kt = 0; kt < nk; kt += STAGES) each_stage<STAGES>([&](auto s) { if (kt + s < nk) step(s); });
      if (group == 0) phase_barrier();
    } else if constexpr (RP) {
      static_assert(FAST, "the codes go into the matrix instructions as they are");
      u32x4 na[2][TM][2], nb[2][TN][2];  // this slab's fragments and the next one's
      auto fetch = [&](u32x4 (&ta)[TM][2], u32x4 (&tb)[TN][2], const unsigned char* st) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned char* const at_row = st + l32 * SLAB + 16 * ((2 * half + h) ^ fp8::swz(l32));
#pragma unroll
          for (int i = 0; i < TM; ++i) ta[i][h] = *(const lds_u32x4*)(at_row + (wm * TM + i) * 32 * SLAB);
#pragma unroll
          for (int j = 0; j < TN; ++j) tb[j][h] = *(const lds_u32x4*)(at_row + B_AT + (wn * TN + j) * 32 * SLAB);
        }
      };
      __builtin_amdgcn_s_waitcnt(waitcnt_vm((D - 1) * PER));
      phase_barrier();
      scales();
      fetch(na[0], nb[0], lds);
      auto step = [&](auto stage) {
        constexpr int s = decltype(stage)::value, cur = s % 2;
        // everyone has this slab in registers, its stage is free, and the next slab has landed
        __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0());
        __builtin_amdgcn_s_waitcnt(waitcnt_vm((D - 2) * PER));
        phase_barrier();
        issue(s);
        fetch(na[1 - cur], nb[1 - cur], lds + (s + 1) % STAGES * STAGE);
        constexpr int READS = 2 * (TM + TN), EACH = (READS + TM * TN - 1) / (TM * TN);  // of LDS
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = fp8::mfma(nb[cur][j], hb[j], na[cur][i], ha[i], acc[i][j]);
#pragma unroll
        for (int i = 0; i < TM * TN; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);       // a matrix instruction
          __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);  // reads of LDS
        }
        __builtin_amdgcn_sched_barrier(0);
        // the sums stay in this step: they would sink past the branch below and the next barrier
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) asm volatile("" : "+a"(acc[i][j]));
        ++at;
        if (s % 2 == 1) {
#pragma unroll
          for (int i = 0; i < TM; ++i) ha[i] >>= 8;
#pragma unroll
          for (int j = 0; j < TN; ++j) hb[j] >>= 8;
          if ((at & 7) == 0) scales();  // after the last slab too: scales_at stays in the row
        }
      };
      // an even number of slabs.  No branch inside: matrix instructions would sink past it
      int kt = 0;
      for (; kt + STAGES <= nk; kt += STAGES) each_stage<STAGES>(step);
      if (kt < nk) each_stage<2>(step);
    } else {
      auto step = [&](auto stage) {
        constexpr int s = decltype(stage)::value;
        // this slab has landed; the ones after it may be in flight
        __builtin_amdgcn_s_waitcnt(waitcnt_vm((D - 1) * PER));
        // everyone has read the last slab, whose stage the DMA now fills
        __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0());
        phase_barrier();
        issue((s + D) % STAGES);
        each_stage<HALVES>([&](auto hf) {
          read(s, hf, lds + s * STAGE);
          mma(s, hf);
        });
      };
      for (int kt = 0; kt < nk; kt += STAGES) each_stage<STAGES>([&](auto s) { if (kt + s < nk) step(s); });
    }
    // no DMA may write LDS after the workgroup has left it, or the walk
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
  }

  // the sums are read behind branches: their wait states are spelled out
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_nop 15\n\ts_nop 15");
  __builtin_amdgcn_sched_barrier(0);

  // ---- a lane holds C[m][n .. n+3] for n, n+8, n+16 and n+24 of each 32 x 32
  void* const c = p.c;
  const int ldc = p.ldc, out16 = p.out16;
  const bool whole = (ldc & 3) == 0 && ((uintptr_t)c & (out16 ? 7 : 15)) == 0;
  const bool wide = out16 && (ldc & 7) == 0 && ((uintptr_t)c & 15) == 0;
  auto pair16 = [](float lo, float hi) { return __builtin_bit_cast(unsigned, fp8::bf16x2{(__bf16)lo, (__bf16)hi}); };
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = (wm * TM + i) * 32 + l32;
    if (m >= rows) continue;
    const int64_t at = (int64_t)(m0 + m) * ldc + n0;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      if (wide && n0 + (wn * TN + j) * 32 + 32 <= p.N) {
        // the two halves of the wave swap runs: eight neighbouring columns a lane
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          u32x4 v;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const auto got = __builtin_amdgcn_permlane32_swap(pair16(acc[i][j][4 * q + 2 * w], acc[i][j][4 * q + 2 * w + 1]),
                                                              pair16(acc[i][j][4 * q + 4 + 2 * w], acc[i][j][4 * q + 5 + 2 * w]), false, false);
            v[w] = got[0], v[2 + w] = got[1];
          }
          *(u32x4*)((__bf16*)c + at + (wn * TN + j) * 32 + 8 * q + 8 * half) = v;
        }
        continue;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        store4(c, out16, at, f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]},
               (wn * TN + j) * 32 + 8 * q + 4 * half, cols, whole);
    }
  }
}

}  // namespace xtc_hip
