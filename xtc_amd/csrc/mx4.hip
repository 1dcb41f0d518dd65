// SPDX-License-Identifier: BSD-3-Clause
// Entry points of the microscaled 4-bit operators.
#include "xtc_hip.h"
#include "core.hpp"
#include "grouped_dma.hpp"
#include "mx4_any.hpp"
#include "mx4_rows.hpp"

using namespace xtc_hip;
using core::aligned16;
using core::fail;

namespace {

// Largest extent: tiles and blocks past it stay within 32 bits.
constexpr int kMost = 0x7fffffff - 1023;

int done(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

int check(const xtc_hip_mx4_desc* d, const char* what) {
  if (!core::ready()) return fail("xtc_hip_init not called");
  if (!d) return fail("%s: null descriptor", what);
  if (d->dtype != XTC_HIP_F32 && d->dtype != XTC_HIP_BF16) return fail("%s: unsupported dtype %d", what, d->dtype);
  if (d->rows < 0 || d->K < 1 || d->K > kMost)
    return fail("%s: invalid sizes rows=%lld K=%d", what, (long long)d->rows, d->K);
  if (d->ld && d->ld < d->K) return fail("%s: row stride %d is below the %d elements of a row", what, d->ld, d->K);
  // no operand has more bytes a row than 4 of each element and 16 of each block
  const int64_t row = 4 * (int64_t)(d->ld ? d->ld : d->K) + 16 * (((int64_t)d->K + 31) / 32);
  if (d->rows > INT64_MAX / row) return fail("%s: sizes rows=%lld K=%d are too many", what, (long long)d->rows, d->K);
  return 0;
}

Mx4QuantArgs args_of(const xtc_hip_mx4_desc& d) {
  Mx4QuantArgs a{};
  a.rows = d.rows, a.K = d.K, a.blocks = (d.K + 31) / 32;
  a.ldx = d.ld ? d.ld : d.K, a.ldv = d.K;
  return a;
}

constexpr int kQuarters = 4;  // of a block a lane, dense rows

dim3 grid_of(const Mx4QuantArgs& a) {
  return dim3((unsigned)((4 * (int64_t)a.blocks + 255) / 256), (unsigned)(a.rows < 65535 ? a.rows : 65535));
}

int quantize(const xtc_hip_mx4_desc& d, const Mx4QuantArgs& a, const char* what) {
  if (!aligned16(a.codes)) return fail("%s: codes must be 16-byte aligned", what);
  if (a.K % 32 == 0 && a.ldx == a.K && !a.scales_in && aligned16(a.x) && aligned16(a.values)) {
    const int64_t quarters = a.rows * (a.K / 8), groups = (quarters + 256 * kQuarters - 1) / (256 * kQuarters);
    if (groups < (int64_t)1 << 31) {
      const dim3 grid((unsigned)groups);
      if (d.dtype == XTC_HIP_F32)
        hipLaunchKernelGGL((mx4_quantize_dense<float, kQuarters>), grid, dim3(256), 0, core::pick_stream(d.stream), a, quarters);
      else
        hipLaunchKernelGGL((mx4_quantize_dense<__bf16, kQuarters>), grid, dim3(256), 0, core::pick_stream(d.stream), a, quarters);
      return done(what);
    }
  }
  if (d.dtype == XTC_HIP_F32)
    hipLaunchKernelGGL(mx4_quantize<float>, grid_of(a), dim3(256), 0, core::pick_stream(d.stream), a);
  else
    hipLaunchKernelGGL(mx4_quantize<__bf16>, grid_of(a), dim3(256), 0, core::pick_stream(d.stream), a);
  return done(what);
}

// ---- products of whole slabs (4 blocks)

struct DmaTile {
  DmaCost cost;
  void (*launch)(const DmaArgs&, unsigned, hipStream_t);
};
template <int WGM, int WGN, int TM, int TN, int STAGES, bool PP>
void dma_launch(const DmaArgs& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((grouped_dma<true, false, true, WGM, WGN, TM, TN, STAGES, PP>), dim3(groups), dim3(WGM * WGN * 64), 0, s, a);
}
// Costs as measured: 1 x 8192 x 8192 (light), 4096 x 8192 x 8192 and 8192^3 (full).
const DmaTile kDmaTiles[] = {
    {{256, 256, 1, 1.25, 2.00}, &dma_launch<2, 4, 8, 4, 2, true>},
    {{128, 128, 2, 0.73, 1.45}, &dma_launch<2, 2, 4, 4, 2, false>},
    {{64, 64, 2, 0.24, 0.62}, &dma_launch<2, 2, 2, 2, 4, false>},
};

const DmaTile& dma_tile(int64_t rows, int64_t groups, int N, int blocks, int out_bytes) {
  const DmaTile* best = nullptr;
  double least = 0;
  for (const DmaTile& t : kDmaTiles) {
    const double tiles = likely_tiles(rows, groups, t.cost.bm) * ((N + t.cost.bn - 1) / t.cost.bn);
    const double cost = dma_cost(t.cost, tiles, (blocks + 4) / 8, out_bytes);
    if (!best || cost < least) best = &t, least = cost;
  }
  return *best;
}

// ---- few rows

struct RowsTile {
  int bm, bn;
  void (*run[2])(const Mx4Args&, unsigned, hipStream_t);  // to fp32, to bf16
};
template <typename U, int TM, int TN, bool QUANTIZE>
void rows_launch(const Mx4Args& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((mx4_rows<U, TM, TN, QUANTIZE>), dim3(groups), dim3(64 * mx4::RWAVES), 0, s, a);
}
const RowsTile kRows16 = {16, 32, {&rows_launch<float, 1, 2, false>, &rows_launch<__bf16, 1, 2, false>}};
const RowsTile kRows32 = {32, 32, {&rows_launch<float, 2, 2, false>, &rows_launch<__bf16, 2, 2, false>}};
const RowsTile kRowsX = {16, 32, {&rows_launch<float, 1, 2, true>, &rows_launch<__bf16, 1, 2, true>}};

double rows_groups(const RowsTile& t, int64_t rows, int64_t groups, int N) {
  return likely_tiles(rows, groups, t.bm) * ((N + t.bn - 1) / t.bn);
}

// As many tiles as fit the CUs at once: eight waves a tile then read b as fast as it
// comes (8192 x 8192 with 16 rows: 9.9 us, DMA tiles 13.8; with 32: 12.3, 14.4;
// 64 x 4096 x 4096: 7.3, 8.3; 1000 x 8192 x 128: 8.9, 15.1), beyond that whole slabs
// go to tiles that read their operands once for 64 rows (64 x 8192 x 8192: 22.6,
// 15.0).  By group twice as many, some of which stay empty (8 rows over 8 experts of
// 4096 x 2048: 7.3, 9.6; 32 over 16: 16.4, 13.2).  Blocks of no whole slabs stay
// here up to 32 rows a group (32 rows over 16 experts of 4128 x 2048: 14.1, the
// kernel of any blocks 20.5).
const RowsTile* rows_tile(int64_t rows, int64_t groups, int N, bool slabs) {
  const double most = groups > 1 ? 512 : 256;
  for (const RowsTile* t : {&kRows16, &kRows32})
    if (rows_groups(*t, rows, groups, N) <= most) return t;
  if (slabs) return nullptr;
  return rows <= 16 * groups ? &kRows16 : rows <= 32 * groups ? &kRows32 : nullptr;
}

// Whole quarters of blocks, no more workgroups than the CUs take at once, since each
// quantises its rows, and rows short enough: lanes read 64 bytes of different ones,
// which costs more than a launch (4 us) from some 32768 elements on.  16 rows x 1024
// x 2048 7.7 us in two launches, 4.9 in one; x 2048 x 8192 7.9, 7.0; x 4096 x 4096
// 8.4, 10.2.  Rows of 8192 and more are no faster in one launch, however few: 1, 2 and
// 4 x 8192 x 8192 11.2, 11.2 and 11.4 us in two, 11.1, 11.4 and 11.7 in one; 1 x 16384 x
// 4096 15.7, 16.6; 1 x 32768 x 1024 23.8, 28.2.
bool quantizes_on_the_way(int64_t rows, int64_t groups, int N, int K) {
  const int64_t each = (rows + groups - 1) / groups;
  return K % 8 == 0 && K < 8192 && (each < 16 ? each : 16) * K <= 32768 && rows_groups(kRowsX, rows, groups, N) <= 256;
}

int launch_rows(const xtc_hip_mx4_matmul_desc& d, const RowsTile& t, Mx4Args& a, const char* what) {
  a.tiles_n = (d.N + t.bn - 1) / t.bn;
  const int64_t groups = a.tiles_n * (a.sizes ? most_tiles(d.M, d.E, t.bm) : ((int64_t)d.M + t.bm - 1) / t.bm);
  if (groups >= (int64_t)1 << 31) return fail("%s: %lld workgroups are too many", what, (long long)groups);
  t.run[d.out_dtype](a, (unsigned)groups, core::pick_stream(d.stream));
  return done(what);
}

// ---- products

int check(const xtc_hip_mx4_matmul_desc* desc, const int32_t* sizes, const char* what) {
  if (!core::ready()) return fail("xtc_hip_init not called");
  if (!desc) return fail("%s: null descriptor", what);
  const xtc_hip_mx4_matmul_desc& d = *desc;
  if (d.out_dtype != XTC_HIP_F32 && d.out_dtype != XTC_HIP_BF16) return fail("%s: unsupported result dtype %d", what, d.out_dtype);
  if (d.E < 0 || d.M < 0 || d.N < 1 || d.blocks < 1)
    return fail("%s: invalid sizes E=%d M=%d N=%d blocks=%d", what, d.E, d.M, d.N, d.blocks);
  if (d.E > kMost || d.M > kMost || d.N > kMost || d.blocks > kMost / 32)
    return fail("%s: sizes E=%d M=%d N=%d blocks=%d are too many", what, d.E, d.M, d.N, d.blocks);
  if ((d.E > 0) != (sizes != nullptr)) return fail("%s: E=%d groups %s sizes", what, d.E, sizes ? "with" : "without");
  if (d.ldc && d.ldc < d.N) return fail("%s: row stride %d of c is below its %d columns", what, d.ldc, d.N);
  return 0;
}

Mx4Args args_of(const xtc_hip_mx4_matmul_desc& d, const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                const uint8_t* b_scales, const int32_t* sizes, void* c) {
  Mx4Args a{};
  a.a_codes = a_codes, a.a_scales = a_scales, a.b_codes = b_codes, a.b_scales = b_scales, a.sizes = sizes, a.c = c;
  a.E = d.E > 0 ? d.E : 1, a.M = d.M, a.N = d.N, a.blocks = d.blocks, a.ldc = d.ldc ? d.ldc : d.N;
  return a;
}

int product(const xtc_hip_mx4_matmul_desc& d, Mx4Args& a, const char* what) {
  const bool slabs = d.blocks % 4 == 0 && d.blocks < (1 << 19) && ((uintptr_t)a.a_scales & 3) == 0 && ((uintptr_t)a.b_scales & 3) == 0;
  if (const RowsTile* t = rows_tile(d.M, a.E, d.N, slabs)) return launch_rows(d, *t, a, what);
  if (slabs) {
    const DmaTile& t = dma_tile(d.M, a.E, d.N, d.blocks, d.out_dtype == XTC_HIP_BF16 ? 2 : 4);
    DmaArgs v{};
    v.a = a.a_codes, v.b = a.b_codes, v.sa = a.a_scales, v.sb = a.b_scales, v.sizes = a.sizes, v.c = a.c;
    v.E = a.E, v.M = d.M, v.N = d.N, v.K = d.blocks;
    v.lda = v.ldb = 16 * d.blocks, v.ldc = a.ldc;
    v.stride_b = (int64_t)d.N * v.ldb, v.stride_sb = (int64_t)d.N * d.blocks;
    v.tiles_m = (int)(a.sizes ? most_tiles(d.M, d.E, t.cost.bm) : ((int64_t)d.M + t.cost.bm - 1) / t.cost.bm);
    v.tiles_n = (d.N + t.cost.bn - 1) / t.cost.bn;
    v.band = v.tiles_m < 8 ? v.tiles_m : 8;
    v.out16 = d.out_dtype == XTC_HIP_BF16;
    const int64_t groups = dma_groups(v, 1);
    if (groups >= (int64_t)1 << 31) return fail("%s: %lld workgroups are too many", what, (long long)groups);
    t.launch(v, (unsigned)groups, core::pick_stream(d.stream));
    return done(what);
  }
  a.tiles_n = (d.N + mx4::BN - 1) / mx4::BN;
  const int64_t rows = a.sizes ? most_tiles(d.M, d.E, mx4::BM) : ((int64_t)d.M + mx4::BM - 1) / mx4::BM;
  if (rows * a.tiles_n < 1 || rows * a.tiles_n >= (int64_t)1 << 31)
    return fail("%s: %lld workgroups are too many", what, (long long)(rows * a.tiles_n));
  const dim3 grid((unsigned)(rows * a.tiles_n));
  if (d.out_dtype == XTC_HIP_F32) hipLaunchKernelGGL(mx4_any<float>, grid, dim3(256), 0, core::pick_stream(d.stream), a);
  else hipLaunchKernelGGL(mx4_any<__bf16>, grid, dim3(256), 0, core::pick_stream(d.stream), a);
  return done(what);
}

}  // namespace

extern "C" {

int xtc_hip_mx4_desc_size(void) { return (int)sizeof(xtc_hip_mx4_desc); }
int xtc_hip_mx4_matmul_desc_size(void) { return (int)sizeof(xtc_hip_mx4_matmul_desc); }

int xtc_hip_mx4_quantize(const xtc_hip_mx4_desc* desc, const void* x, uint8_t* codes, uint8_t* scales, void* values) {
  const char* const what = "mx4_quantize";
  if (check(desc, what)) return 1;
  if (desc->rows == 0) return 0;
  if (!x || (!codes && !scales && !values)) return fail("%s: null operand", what);
  Mx4QuantArgs a = args_of(*desc);
  a.x = x, a.codes = codes, a.scales = scales, a.values = values;
  return quantize(*desc, a, what);
}

int xtc_hip_mx4_encode(const xtc_hip_mx4_desc* desc, const void* x, const uint8_t* scales, uint8_t* codes) {
  const char* const what = "mx4_encode";
  if (check(desc, what)) return 1;
  if (desc->rows == 0) return 0;
  if (!x || !scales || !codes) return fail("%s: null operand", what);
  Mx4QuantArgs a = args_of(*desc);
  a.x = x, a.scales_in = scales, a.codes = codes;
  return quantize(*desc, a, what);
}

int xtc_hip_mx4_dequantize(const xtc_hip_mx4_desc* desc, const uint8_t* codes, const uint8_t* scales, void* values) {
  const char* const what = "mx4_dequantize";
  if (check(desc, what)) return 1;
  if (desc->rows == 0) return 0;
  if (!codes || !scales || !values) return fail("%s: null operand", what);
  if (!aligned16(codes)) return fail("%s: codes must be 16-byte aligned", what);
  Mx4QuantArgs a = args_of(*desc);
  a.codes_in = codes, a.scales_in = scales, a.values = values;
  a.ldv = a.ldx;
  if (desc->dtype == XTC_HIP_F32)
    hipLaunchKernelGGL(mx4_dequantize<float>, grid_of(a), dim3(256), 0, core::pick_stream(desc->stream), a);
  else
    hipLaunchKernelGGL(mx4_dequantize<__bf16>, grid_of(a), dim3(256), 0, core::pick_stream(desc->stream), a);
  return done(what);
}

int xtc_hip_mx4_matmul(const xtc_hip_mx4_matmul_desc* desc, const uint8_t* a_codes, const uint8_t* a_scales,
                       const uint8_t* b_codes, const uint8_t* b_scales, const int32_t* sizes, void* c) {
  const char* const what = "mx4_matmul";
  if (check(desc, sizes, what)) return 1;
  if (desc->M == 0) return 0;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !c) return fail("%s: null operand", what);
  if (!aligned16(a_codes) || !aligned16(b_codes)) return fail("%s: codes must be 16-byte aligned", what);
  Mx4Args a = args_of(*desc, a_codes, a_scales, b_codes, b_scales, sizes, c);
  return product(*desc, a, what);
}

int xtc_hip_mx4_quantize_matmul(const xtc_hip_mx4_desc* rows, const xtc_hip_mx4_matmul_desc* desc, const void* x,
                                uint8_t* a_codes, uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales,
                                const int32_t* sizes, void* c) {
  const char* const what = "mx4_quantize_matmul";
  if (check(rows, what) || check(desc, sizes, what)) return 1;
  if (rows->rows != desc->M || (rows->K + 31) / 32 != desc->blocks || rows->stream != desc->stream)
    return fail("%s: %lld rows of %d elements to quantise, %d rows of %d blocks to multiply, or two streams", what,
                (long long)rows->rows, rows->K, desc->M, desc->blocks);
  if (desc->M == 0) return 0;
  if (!x || !a_codes || !a_scales || !b_codes || !b_scales || !c) return fail("%s: null operand", what);
  if (!aligned16(a_codes) || !aligned16(b_codes)) return fail("%s: codes must be 16-byte aligned", what);
  Mx4Args a = args_of(*desc, a_codes, a_scales, b_codes, b_scales, sizes, c);
  if (rows->dtype == XTC_HIP_BF16 && quantizes_on_the_way(desc->M, a.E, desc->N, rows->K)) {
    a.x = (const __bf16*)x, a.K = rows->K, a.ldx = rows->ld ? rows->ld : rows->K;
    return launch_rows(*desc, kRowsX, a, what);
  }
  Mx4QuantArgs q = args_of(*rows);
  q.x = x, q.codes = a_codes, q.scales = a_scales;
  return quantize(*rows, q, what) || product(*desc, a, what);
}

}  // extern "C"
