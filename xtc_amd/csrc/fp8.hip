// SPDX-License-Identifier: BSD-3-Clause
// Entry points of the 8-bit operators.
#include "xtc_hip.h"
#include "core.hpp"
#include "fp8.hpp"
#include "fp8_dma.hpp"
#include "fp8_rows.hpp"

using namespace xtc_hip;
using core::aligned16;
using core::fail;

namespace {

// Largest extent: tiles and blocks past it stay within 32 bits.
constexpr int kMost = 0x7fffffff - 1023;
constexpr int64_t kMostGroups = 1 << 22;  // of a launch that walks: its threads stay within 32 bits

int done(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

unsigned groups_of(int64_t items, int64_t each) {
  const int64_t groups = (items + each - 1) / each;
  return (unsigned)(groups < kMostGroups ? groups : kMostGroups);
}

int check(const xtc_hip_fp8_desc* d, const char* what) {
  if (!core::ready()) return fail("xtc_hip_init not called");
  if (!d) return fail("%s: null descriptor", what);
  if (d->dtype != XTC_HIP_F32 && d->dtype != XTC_HIP_BF16) return fail("%s: unsupported dtype %d", what, d->dtype);
  if (d->matrices < 0 || d->rows < 0 || d->K < 1)
    return fail("%s: invalid sizes matrices=%d rows=%lld K=%d", what, d->matrices, (long long)d->rows, d->K);
  if (d->block_rows != 1 && d->block_rows != 128) return fail("%s: blocks of %d rows (they have 1 or 128)", what, d->block_rows);
  if (d->transpose != 0 && d->transpose != 1) return fail("%s: transpose %d is neither 0 nor 1", what, d->transpose);
  if (d->ld && d->ld < d->K) return fail("%s: row stride %d is below the %d elements of a row", what, d->ld, d->K);
  // no operand has more bytes than 4 of each element and 128 of each block, whole rows
  // of blocks
  const int64_t row = 4 * (int64_t)(d->ld ? d->ld : d->K) + 128 * (((int64_t)d->K + 127) / 128);
  if (d->K > kMost || d->rows > (int64_t)kMost * 64 || (d->matrices && d->rows + 127 > INT64_MAX / row / d->matrices))
    return fail("%s: sizes matrices=%d rows=%lld K=%d are too many", what, d->matrices, (long long)d->rows, d->K);
  return 0;
}

Fp8QuantArgs args_of(const xtc_hip_fp8_desc& d) {
  Fp8QuantArgs a{};
  a.matrices = d.matrices, a.rows = d.rows, a.K = d.K, a.blocks = (d.K + 127) / 128;
  a.ldx = d.ld ? d.ld : d.K, a.ldv = d.K, a.square = d.block_rows == 128;
  return a;
}

constexpr int kRuns = 4;  // of 8 elements a lane

int quantize(const xtc_hip_fp8_desc& d, const Fp8QuantArgs& a, const char* what) {
  if (!aligned16(a.codes) || !aligned16(a.codes_t)) return fail("%s: codes must be 16-byte aligned", what);
  const hipStream_t s = core::pick_stream(d.stream);
  if (!a.square && !a.codes_t && !a.scales_t) {
    const int64_t runs = a.matrices * a.rows * a.blocks * 16;
    const dim3 grid(groups_of(runs, 256 * kRuns));
    const int dense = a.K % 128 == 0 && a.ldx == a.K;
    const auto kernel = d.dtype == XTC_HIP_F32 ? (a.scales_in ? fp8_quantize_rows<float, kRuns, true> : fp8_quantize_rows<float, kRuns, false>)
                                               : (a.scales_in ? fp8_quantize_rows<__bf16, kRuns, true> : fp8_quantize_rows<__bf16, kRuns, false>);
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, runs, dense);
    return done(what);
  }
  const dim3 grid(groups_of(a.matrices * ((a.rows + 127) / 128) * a.blocks, 1));
  const auto kernel = d.dtype == XTC_HIP_F32 ? (a.scales_in ? fp8_quantize_tiles<float, true> : fp8_quantize_tiles<float, false>)
                                             : (a.scales_in ? fp8_quantize_tiles<__bf16, true> : fp8_quantize_tiles<__bf16, false>);
  hipLaunchKernelGGL(kernel, grid, dim3(512), 0, s, a);
  return done(what);
}

// ---- products

struct DmaTile {
  DmaCost cost[2];  // fp32 sums, those of the 8-bit instructions
  void (*launch[2])(const Fp8Args&, unsigned, hipStream_t);
};
template <bool FAST, int WGM, int WGN, int TM, int TN, fp8::Schedule S>
void dma_launch(const Fp8Args& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((fp8_dma<FAST, WGM, WGN, TM, TN, 4, S>), dim3(groups), dim3(WGM * WGN * 64), 0, s, a);
}
// Microseconds a block, a CU with one workgroup and with all it takes, measured (us, the
// three tiles in this order; M x N x k):
//   8-bit instructions, to bf16:
//             4096 x 4096 x 2048  43, 48, 72    4096 x 2048 x 4096  68, 45, 76    2048 x 2048 x 2048  40, 17, 23
//             512 x 4096 x 4096  54, 26, 23    1024 x 1024 x 8192  98, 52, 33    8192 x 8192 x 4096  250, 322, 502
//   fp32 sums, to fp32:
//             4096 x 4096 x 2048  80, 81, 100   4096 x 2048 x 4096  111, 73, 97   2048 x 2048 x 2048  56, 29, 30
//             512 x 4096 x 4096  88, 40, 31    1024 x 1024 x 8192  167, 78, 44   8192 x 8192 x 4096  469, 497, 680
//   the other two kinds lose up to 5 % of a product by the choice, 13 % once (8-bit to fp32 at 2048^3):
//   fp32 sums, to bf16
//             4096 x 4096 x 2048  65, 73, 93    4096 x 2048 x 4096  106, 72, 94   2048 x 2048 x 2048  52, 25, 26
//             512 x 4096 x 4096  84, 39, 30    1024 x 1024 x 8192  163, 76, 43   8192 x 8192 x 4096  432, 486, 676
//   8-bit instructions, to fp32
//             4096 x 4096 x 2048  57, 60, 85    4096 x 2048 x 4096  78, 55, 84    2048 x 2048 x 2048  41, 21, 24
//             512 x 4096 x 4096  62, 33, 27    1024 x 1024 x 8192  102, 53, 33   8192 x 8192 x 4096  385, 374, 551
// fp32 sums are bound by the conversions, which take longer than the products: a
// schedule of fragments read ahead and 256 x 128 tiles made 4096 x 2048 x 4096 no faster (79).
const DmaTile kDmaTiles[] = {
    {{{256, 256, 1, 2.4, 3.3}, {256, 256, 1, 1.3, 1.8}}, {&dma_launch<false, 2, 4, 4, 2, fp8::PINGPONG>, &dma_launch<true, 2, 2, 4, 4, fp8::AHEAD>}},
    {{{128, 128, 2, 1.0, 1.85}, {128, 128, 2, 0.6, 1.2}}, {&dma_launch<false, 2, 2, 2, 2, fp8::PLAIN>, &dma_launch<true, 2, 2, 2, 2, fp8::PLAIN>}},
    {{{64, 64, 4, 0.55, 1.3}, {64, 64, 4, 0.4, 1.0}}, {&dma_launch<false, 2, 2, 1, 1, fp8::PLAIN>, &dma_launch<true, 2, 2, 1, 1, fp8::PLAIN>}},
};

struct RowsTile {
  int bm, bn;
  void (*run[2])(const Fp8Args&, unsigned, hipStream_t);  // to fp32, to bf16
};
template <typename U, int TM, int TN>
void rows_launch(const Fp8Args& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((fp8_rows<U, TM, TN>), dim3(groups), dim3(64 * fp8::RWAVES), 0, s, a);
}
const RowsTile kRows16 = {16, 32, {&rows_launch<float, 1, 2>, &rows_launch<__bf16, 1, 2>}};
const RowsTile kRows32 = {32, 32, {&rows_launch<float, 2, 2>, &rows_launch<__bf16, 2, 2>}};

int64_t tiles_of(int64_t size, int tile) { return (size + tile - 1) / tile; }

int check(const xtc_hip_fp8_matmul_desc* desc, const char* what) {
  if (!core::ready()) return fail("xtc_hip_init not called");
  if (!desc) return fail("%s: null descriptor", what);
  const xtc_hip_fp8_matmul_desc& d = *desc;
  if (d.out_dtype != XTC_HIP_F32 && d.out_dtype != XTC_HIP_BF16) return fail("%s: unsupported result dtype %d", what, d.out_dtype);
  if (d.M < 0 || d.N < 1 || d.blocks < 1) return fail("%s: invalid sizes M=%d N=%d blocks=%d", what, d.M, d.N, d.blocks);
  if (d.b_block_rows != 1 && d.b_block_rows != 128) return fail("%s: blocks of %d rows of b (they have 1 or 128)", what, d.b_block_rows);
  if (d.M > kMost || d.N > kMost || d.blocks >= 1 << 16)
    return fail("%s: sizes M=%d N=%d blocks=%d are too many", what, d.M, d.N, d.blocks);
  if (d.ldc && d.ldc < d.N) return fail("%s: row stride %d of c is below its %d columns", what, d.ldc, d.N);
  if (d.sums < XTC_HIP_SUMS_ANY || d.sums > XTC_HIP_SUMS_FP8) return fail("%s: unsupported sums %d", what, d.sums);
  return 0;
}

int product(const xtc_hip_fp8_matmul_desc& d, Fp8Args& a, const char* what) {
  const hipStream_t s = core::pick_stream(d.stream);
  const bool fast = d.sums == XTC_HIP_SUMS_FP8 || (d.sums == XTC_HIP_SUMS_ANY && a.out16);
  // Few tiles: the kernel that sums in fp32 (unless the caller has asked for the other sums),
  // with as many rows a tile as take the fewer rounds of the 256 CUs, and up to two rounds.
  // us, 16 rows a tile, 32, and the best tile of LDS-DMA with fp32 sums and 8-bit ones (M x N x k):
  //   one round   16 x 8192 x 8192  18, 21, 50, 41   32 x 8192 x 8192  33, 23, 50, 42   16 x 4096 x 1024  5.1, 4.8, 8.1, 6.9
  //   two         16 x 11008 x 8192  31, 35, 51, 42   16 x 14336 x 2048  11, 12, 15, 13   32 x 14336 x 8192  60, 43, 52, 45
  //               128 x 4096 x 4096  31, 22, 22, 18   64 x 8192 x 1024  12, 8.4, 8.5, 7.3
  //   four        16 x 28672 x 8192  63, 69, 64, 62   64 x 14336 x 8192  105, 81, 52, 46
  // In two rounds tiles of 32 rows lose to 8-bit sums.
  const auto rounds = [&](const RowsTile& t) { return (tiles_of(d.M, t.bm) * tiles_of(d.N, t.bn) + 255) / 256; };
  const RowsTile& few = rounds(kRows16) <= rounds(kRows32) ? kRows16 : kRows32;
  if (d.sums != XTC_HIP_SUMS_FP8 && rounds(few) <= (fast && few.bm == 32 ? 1 : 2)) {
    a.tiles_n = (int)tiles_of(d.N, few.bn);
    few.run[a.out16](a, (unsigned)(tiles_of(d.M, few.bm) * a.tiles_n), s);
    return done(what);
  }
  const DmaTile* best = nullptr;
  double least = 0;
  for (const DmaTile& t : kDmaTiles) {
    const DmaCost& c = t.cost[fast];
    const double cost = dma_cost(c, (double)tiles_of(d.M, c.bm) * tiles_of(d.N, c.bn), d.blocks, a.out16 ? 2 : 4);
    if (!best || cost < least) best = &t, least = cost;
  }
  a.tiles_m = (int)tiles_of(d.M, best->cost[0].bm), a.tiles_n = (int)tiles_of(d.N, best->cost[0].bn);
  a.band = a.tiles_m < 8 ? a.tiles_m : 8;
  const int64_t tiles = ((int64_t)a.tiles_m + a.band - 1) / a.band * a.band * a.tiles_n, whole = (int64_t)8 * 4 * a.band;
  const int64_t groups = (tiles + whole - 1) / whole * whole;
  if (groups >= (int64_t)1 << 22) return fail("%s: %lld workgroups are too many", what, (long long)groups);
  best->launch[fast](a, (unsigned)groups, s);
  return done(what);
}

}  // namespace

extern "C" {

int xtc_hip_fp8_desc_size(void) { return (int)sizeof(xtc_hip_fp8_desc); }
int xtc_hip_fp8_matmul_desc_size(void) { return (int)sizeof(xtc_hip_fp8_matmul_desc); }

int xtc_hip_fp8_quantize(const xtc_hip_fp8_desc* desc, const void* x, uint8_t* codes, uint8_t* scales, void* values) {
  const char* const what = "fp8_quantize";
  if (check(desc, what)) return 1;
  if (desc->transpose && values) return fail("%s: values of the transposed matrix come from fp8_dequantize", what);
  if (desc->rows == 0 || desc->matrices == 0) return 0;
  if (!x || (!codes && !scales && !values)) return fail("%s: null operand", what);
  Fp8QuantArgs a = args_of(*desc);
  a.x = x, a.values = values;
  if (desc->transpose) a.codes_t = codes, a.scales_t = scales;
  else a.codes = codes, a.scales = scales;
  return quantize(*desc, a, what);
}

int xtc_hip_fp8_quantize_both(const xtc_hip_fp8_desc* desc, const void* x, uint8_t* codes, uint8_t* scales, uint8_t* codes_t,
                              uint8_t* scales_t) {
  const char* const what = "fp8_quantize_both";
  if (check(desc, what)) return 1;
  if (desc->transpose) return fail("%s: the results are those of x and of its transpose; transpose must be 0", what);
  if (desc->rows == 0 || desc->matrices == 0) return 0;
  if (!x || !codes || !scales || !codes_t || !scales_t) return fail("%s: null operand", what);
  Fp8QuantArgs a = args_of(*desc);
  a.x = x, a.codes = codes, a.scales = scales, a.codes_t = codes_t, a.scales_t = scales_t;
  return quantize(*desc, a, what);
}

int xtc_hip_fp8_encode(const xtc_hip_fp8_desc* desc, const void* x, const uint8_t* scales, uint8_t* codes) {
  const char* const what = "fp8_encode";
  if (check(desc, what)) return 1;
  if (desc->rows == 0 || desc->matrices == 0) return 0;
  if (!x || !scales || !codes) return fail("%s: null operand", what);
  Fp8QuantArgs a = args_of(*desc);
  a.x = x, a.scales_in = scales;
  (desc->transpose ? a.codes_t : a.codes) = codes;
  return quantize(*desc, a, what);
}

int xtc_hip_fp8_dequantize(const xtc_hip_fp8_desc* desc, const uint8_t* codes, const uint8_t* scales, void* values) {
  const char* const what = "fp8_dequantize";
  if (check(desc, what)) return 1;
  if (desc->transpose) return fail("%s: transpose must be 0", what);
  if (desc->rows == 0 || desc->matrices == 0) return 0;
  if (!codes || !scales || !values) return fail("%s: null operand", what);
  if (!aligned16(codes)) return fail("%s: codes must be 16-byte aligned", what);
  Fp8QuantArgs a = args_of(*desc);
  a.codes_in = codes, a.scales_in = scales, a.values = values, a.ldv = a.ldx;
  const int64_t runs = a.matrices * a.rows * a.blocks * 16;
  const dim3 grid(groups_of(runs, 256));
  const hipStream_t s = core::pick_stream(desc->stream);
  if (desc->dtype == XTC_HIP_F32) hipLaunchKernelGGL(fp8_dequantize<float>, grid, dim3(256), 0, s, a, runs);
  else hipLaunchKernelGGL(fp8_dequantize<__bf16>, grid, dim3(256), 0, s, a, runs);
  return done(what);
}

int xtc_hip_fp8_matmul(const xtc_hip_fp8_matmul_desc* desc, const uint8_t* a_codes, const uint8_t* a_scales,
                       const uint8_t* b_codes, const uint8_t* b_scales, void* c) {
  const char* const what = "fp8_matmul";
  if (check(desc, what)) return 1;
  if (desc->M == 0) return 0;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !c) return fail("%s: null operand", what);
  if (!aligned16(a_codes) || !aligned16(b_codes)) return fail("%s: codes must be 16-byte aligned", what);
  Fp8Args a{};
  a.a = a_codes, a.sa = a_scales, a.b = b_codes, a.sb = b_scales, a.c = c;
  a.M = desc->M, a.N = desc->N, a.blocks = desc->blocks, a.ldc = desc->ldc ? desc->ldc : desc->N;
  a.b_shift = desc->b_block_rows == 128 ? 7 : 0, a.out16 = desc->out_dtype == XTC_HIP_BF16;
  return product(*desc, a, what);
}

}  // extern "C"
