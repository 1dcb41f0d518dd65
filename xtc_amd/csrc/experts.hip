// SPDX-License-Identifier: BSD-3-Clause
// Entry points of the products by group (rows sorted by expert).
#include "xtc_hip.h"
#include "core.hpp"
#include "grouped_any.hpp"
#include "grouped_dma.hpp"

using namespace xtc_hip;
using core::fail;

namespace {

// Largest extent: tiles and slabs past it stay within 32 bits.
constexpr int kMost = 0x7fffffff - 1023;
// 64 x 64 tiles of any operands that make them worth their barriers.
constexpr int64_t kSmallTiles = 512;

int check(const xtc_hip_grouped_matmul_desc* d, const char* what) {
  if (!core::ready()) return fail("xtc_hip_init not called");
  if (!d) return fail("%s: null descriptor", what);
  if (d->dtype != XTC_HIP_F32 && d->dtype != XTC_HIP_BF16) return fail("%s: unsupported dtype %d", what, d->dtype);
  if (d->out_dtype != XTC_HIP_F32 && !(d->out_dtype == XTC_HIP_BF16 && d->dtype == XTC_HIP_BF16))
    return fail("%s: unsupported result dtype %d for operands of dtype %d", what, d->out_dtype, d->dtype);
  if (d->E < 1 || d->T < 0 || d->N < 1 || d->K < 1)
    return fail("%s: invalid sizes E=%d T=%d N=%d K=%d", what, d->E, d->T, d->N, d->K);
  if (d->E > kMost || d->T > kMost || d->N > kMost || d->K > kMost)
    return fail("%s: sizes E=%d T=%d N=%d K=%d are too many, past %d", what, d->E, d->T, d->N, d->K, kMost);
  return 0;
}

int stride(int given, int dense, const char* what, const char* name, int* out) {
  *out = given ? given : dense;
  if (*out < dense) return fail("%s: row stride %d of %s is below its %d columns", what, given, name, dense);
  return 0;
}

// ---- bf16 in whole vectors

typedef void (*DmaLaunch)(const DmaArgs&, unsigned, hipStream_t);
template <bool GRAD, bool B_ROW, int WGM, int WGN, int TM, int TN, int STAGES, bool PP>
void dma_launch(const DmaArgs& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((grouped_dma<false, GRAD, B_ROW, WGM, WGN, TM, TN, STAGES, PP>), dim3(groups), dim3(WGM * WGN * 64), 0, s, a);
}
struct DmaTile {
  int bm, bn;
  DmaLaunch natural, transposed, grad;
};
#define XTC_DMA(...) &dma_launch<false, false, __VA_ARGS__>, &dma_launch<false, true, __VA_ARGS__>, &dma_launch<true, false, __VA_ARGS__>
const DmaTile kDmaTiles[] = {
    {256, 256, XTC_DMA(2, 4, 8, 4, 4, true)},
    {128, 128, XTC_DMA(2, 2, 4, 4, 4, false)},
    {64, 64, XTC_DMA(2, 2, 2, 2, 4, false)},
};
#undef XTC_DMA

// Strides of whole vectors whose offsets within a tile stay within 2^31 bytes.
bool vectors(const void* p, int ld) { return core::aligned16(p) && ld % 8 == 0 && ld < (1 << 22) - 8; }

const DmaTile* dma_tile(int64_t rows, int64_t groups, int N, bool grad, int K) {
  for (const DmaTile& t : kDmaTiles) {
    const int64_t tn = (N + t.bn - 1) / t.bn;
    const int64_t tm = grad ? groups * ((K + t.bm - 1) / t.bm) : rows / t.bm + 1;
    if (tm * tn >= 192) return &t;
  }
  return &kDmaTiles[2];
}

int launch_dma(const DmaTile& t, DmaLaunch run, DmaArgs& a, int64_t matrices, hipStream_t s) {
  a.tiles_n = (a.N + t.bn - 1) / t.bn;
  a.band = a.tiles_m < 8 ? a.tiles_m : 8;
  const int64_t groups = dma_groups(a, matrices);
  if (groups < 1 || groups >= (int64_t)1 << 31) return fail("grouped_matmul: %lld workgroups are too many", (long long)groups);
  run(a, (unsigned)groups, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("grouped_matmul: launch failed: %s", hipGetErrorString(e));
}

// ---- any operands: 64 x 64 tiles, or 32 x 32 tiles of split depth where those
// would leave the CUs idle
template <bool GRAD>
int launch_any(const xtc_hip_grouped_matmul_desc& d, GroupedArgs& a, hipStream_t s) {
  auto tiles = [&](int bm, int bn) {
    a.tiles_n = (a.N + bn - 1) / bn;
    a.tiles_k = (a.K + bm - 1) / bm;
    return a.tiles_n * (GRAD ? (int64_t)a.E * a.tiles_k : most_tiles(a.T, a.E, bm));
  };
  const bool small = tiles(gany::BM, gany::BN) < kSmallTiles;
  const int64_t groups = small ? tiles(gany::SM, gany::SN) : tiles(gany::BM, gany::BN);
  if (groups < 1 || groups >= (int64_t)1 << 31) return fail("grouped_matmul: %lld workgroups are too many", (long long)groups);
  const dim3 grid((unsigned)groups), block(small ? 64 * gany::SWAVES : gany::NT);
  const bool wt = !GRAD && d.trans_w, out16 = d.out_dtype == XTC_HIP_BF16;
#define XTC_ANY_OF(KERNEL, T, U)                                                      \
  do {                                                                                \
    if (wt) hipLaunchKernelGGL((KERNEL<T, U, !GRAD, GRAD>), grid, block, 0, s, a);    \
    else hipLaunchKernelGGL((KERNEL<T, U, false, GRAD>), grid, block, 0, s, a);       \
  } while (0)
#define XTC_ANY(T, U)                                  \
  do {                                                 \
    if (small) XTC_ANY_OF(grouped_small, T, U);        \
    else XTC_ANY_OF(grouped_any, T, U);                \
  } while (0)
  if (d.dtype == XTC_HIP_F32) XTC_ANY(float, float);
  else if (out16) XTC_ANY(__bf16, __bf16);
  else XTC_ANY(__bf16, float);
#undef XTC_ANY
#undef XTC_ANY_OF
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("grouped_matmul: launch failed: %s", hipGetErrorString(e));
}

}  // namespace

extern "C" {

int xtc_hip_grouped_matmul_desc_size(void) { return (int)sizeof(xtc_hip_grouped_matmul_desc); }

int xtc_hip_grouped_matmul(const xtc_hip_grouped_matmul_desc* desc, const void* x, const void* w, const int32_t* sizes,
                           void* y) {
  const char* const what = "grouped_matmul";
  if (check(desc, what)) return 1;
  const xtc_hip_grouped_matmul_desc& d = *desc;
  if (d.T == 0) return 0;
  if (!x || !w || !sizes || !y) return fail("%s: null operand", what);
  GroupedArgs a{};
  a.x = x, a.w = w, a.sizes = sizes, a.y = y;
  a.E = d.E, a.T = d.T, a.N = d.N, a.K = d.K;
  if (stride(d.ldx, d.K, what, "x", &a.ldx) || stride(d.ldw, d.trans_w ? d.K : d.N, what, "w", &a.ldw) ||
      stride(d.ldy, d.N, what, "y", &a.ldy))
    return 1;
  const int64_t matrix = (int64_t)(d.trans_w ? d.N : d.K) * a.ldw;
  a.stride_w = d.stride_w ? d.stride_w : matrix;
  if (a.stride_w < 0) return fail("%s: negative stride between matrices", what);
  if (d.dtype == XTC_HIP_BF16 && d.K % 8 == 0 && (d.trans_w || d.N % 8 == 0) && vectors(x, a.ldx) && vectors(w, a.ldw) &&
      a.stride_w % 8 == 0) {
    const DmaTile& t = *dma_tile(d.T, d.E, d.N, false, d.K);
    DmaArgs v{};
    v.a = (const uint8_t*)x, v.b = (const uint8_t*)w, v.sizes = sizes, v.c = y;
    v.stride_b = 2 * a.stride_w;
    v.E = d.E, v.M = d.T, v.N = d.N, v.K = d.K / 8;
    v.lda = 2 * a.ldx, v.ldb = 2 * a.ldw, v.ldc = a.ldy, v.out16 = d.out_dtype == XTC_HIP_BF16;
    v.tiles_m = (int)most_tiles(d.T, d.E, t.bm);
    return launch_dma(t, d.trans_w ? t.transposed : t.natural, v, 1, core::pick_stream(d.stream));
  }
  return launch_any<false>(d, a, core::pick_stream(d.stream));
}

int xtc_hip_grouped_matmul_grad_w(const xtc_hip_grouped_matmul_desc* desc, const void* x, const void* dy,
                                  const int32_t* sizes, void* dw) {
  const char* const what = "grouped_matmul_grad_w";
  if (check(desc, what)) return 1;
  const xtc_hip_grouped_matmul_desc& d = *desc;
  if (d.trans_w) return fail("%s: a transposed gradient is the gradient with x and dy exchanged", what);
  if (!sizes || !dw || (d.T > 0 && (!x || !dy))) return fail("%s: null operand", what);
  GroupedArgs a{};
  a.x = x, a.w = dy, a.sizes = sizes, a.y = dw;
  a.E = d.E, a.T = d.T, a.N = d.N, a.K = d.K;
  if (stride(d.ldx, d.K, what, "x", &a.ldx) || stride(d.ldy, d.N, what, "dy", &a.ldw) ||
      stride(d.ldw, d.N, what, "dw", &a.ldy))
    return 1;
  const int64_t matrix = (int64_t)d.K * a.ldy;
  a.stride_y = d.stride_w ? d.stride_w : matrix;
  if (a.stride_y < matrix) return fail("%s: a stride of %lld lets the gradients of two groups overlap", what, (long long)d.stride_w);
  if (d.dtype == XTC_HIP_BF16 && d.K % 8 == 0 && d.N % 8 == 0 && vectors(x, a.ldx) && vectors(dy, a.ldw)) {
    const DmaTile& t = *dma_tile(d.T, d.E, d.N, true, d.K);
    DmaArgs v{};
    v.a = (const uint8_t*)x, v.b = (const uint8_t*)dy, v.sizes = sizes, v.c = dw;
    v.stride_c = a.stride_y;
    v.E = d.E, v.M = d.T, v.N = d.N, v.K = d.K;
    v.lda = 2 * a.ldx, v.ldb = 2 * a.ldw, v.ldc = a.ldy, v.out16 = d.out_dtype == XTC_HIP_BF16;
    v.tiles_m = (d.K + t.bm - 1) / t.bm;
    return launch_dma(t, t.grad, v, d.E, core::pick_stream(d.stream));
  }
  return launch_any<true>(d, a, core::pick_stream(d.stream));
}

}  // extern "C"
