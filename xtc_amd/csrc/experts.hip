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
// Bytes of partial sums that a split gradient may write and read.
constexpr double kMostPartial = 1 << 28;
// Workgroups that fill the card, two a CU.
constexpr int64_t kFill = 512;

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
  DmaCost cost;
  DmaLaunch natural, transposed, grad;
};
#define XTC_DMA(...) &dma_launch<false, false, __VA_ARGS__>, &dma_launch<false, true, __VA_ARGS__>, &dma_launch<true, false, __VA_ARGS__>
// Costs as measured: 8 rows over 8 experts, 1024 and 4096 deep (light), 8192^3 and
// 4096 rows over 32 experts of 4096 x 2048 (full).
const DmaTile kDmaTiles[] = {
    {{256, 256, 1, 0.57, 0.80}, XTC_DMA(2, 4, 8, 4, 4, true)},
    {{128, 128, 2, 0.29, 0.62}, XTC_DMA(2, 2, 4, 4, 4, false)},
    {{64, 64, 4, 0.13, 0.73}, XTC_DMA(2, 2, 2, 2, 4, false)},
};
#undef XTC_DMA

// Strides of whole vectors whose offsets within a tile stay within 2^31 bytes.
bool vectors(const void* p, int ld) { return core::aligned16(p) && ld % 8 == 0 && ld < (1 << 22) - 8; }

const DmaTile& dma_tile(int64_t T, int64_t E, int K, int N, int out_bytes, double* cost) {
  const DmaTile* best = nullptr;
  for (const DmaTile& t : kDmaTiles) {
    const double tiles = likely_tiles(T, E, t.cost.bm) * ((N + t.cost.bn - 1) / t.cost.bn);
    const double c = dma_cost(t.cost, tiles, (K + 31) / 32, out_bytes);
    if (!best || c < *cost) best = &t, *cost = c;
  }
  return *best;
}

// The tile of E gradients of K x N and into how many parts each group's rows go.
// The largest group decides where tiles are few, the sum of all where they are many;
// the host does not know the sizes and takes 1.7 times the mean for the largest (shares
// drawn from a Dirichlet distribution of parameter 2: 1.4 times at 2 groups, 2.2 at 8, 3.4
// at 64); starting on a
// round of tiles and writing them out take 5 (64 rows) to 15 us (256): 512 rows, 32
// of 640 x 512, 21 us in 64 x 64 tiles, 14 in 128 x 128.  A part pays for writing and
// reading its partial sums (4 MB a microsecond), all together for one more launch,
// 4 us.  32768 rows: 1 matrix of 128 x 128 163 us whole, 18 in 16 parts of 64 x 64
// tiles; 8 of 512 x 512 55 and 49 (4 parts of 128 x 128); 4096 rows, 8 of 512 x
// 512, 11 us whole, 25 in parts.
const DmaTile& grad_tile(int64_t T, int64_t E, int K, int N, int* splits) {
  const DmaTile* best = nullptr;
  double least = 0;
  const double all = T / (32.0 * E) + 1, skew = E > 1 ? 1.7 : 1, plane = 8.0 * E * K * N;
  for (const DmaTile& t : kDmaTiles) {
    const DmaCost& c = t.cost;
    const double tiles = E * (double)((K + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    for (int s = 1; s <= 16 && (s == 1 || (all / s >= 4 && s * plane <= kMostPartial)); s *= 2) {
      const double slabs = all / s, load = tiles * s / (256.0 * c.per_cu);
      const double cost = slabs * fmax(c.light * skew, c.full * load) + (2 + 0.05 * c.bm) * fmax(load, 1) +
                          (s > 1 ? 4 + s * plane / 4e6 : 0);
      if (!best || cost < least) best = &t, least = cost, *splits = s;
    }
  }
  return *best;
}

int launch_dma(const DmaTile& t, DmaLaunch run, DmaArgs& a, int64_t matrices, hipStream_t s, const char* what) {
  a.tiles_n = (a.N + t.cost.bn - 1) / t.cost.bn;
  a.band = a.tiles_m < 8 ? a.tiles_m : 8;
  const int64_t groups = dma_groups(a, matrices);
  if (groups < 1 || groups >= (int64_t)1 << 31) return fail("%s: %lld workgroups are too many", what, (long long)groups);
  run(a, (unsigned)groups, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

// ---- any operands

typedef void (*AnyLaunch)(const GroupedArgs&, unsigned, hipStream_t);
template <typename T, typename U, bool WT, bool GRAD>
void any_launch(const GroupedArgs& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((grouped_any<T, U, WT, GRAD>), dim3(groups), dim3(gany::NT), 0, s, a);
}
template <typename T, typename U, bool WT, bool GRAD, int TM, int TN>
void small_launch(const GroupedArgs& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((grouped_small<T, U, WT, GRAD, TM, TN>), dim3(groups), dim3(64 * gany::SWAVES), 0, s, a);
}
struct AnyTile {
  int bm, bn;
  AnyLaunch run[3][3];  // natural, transposed, gradient of w; fp32, bf16 to fp32, bf16
};
#define XTC_TYPES(F, ...) {&F<float, float, __VA_ARGS__>, &F<__bf16, float, __VA_ARGS__>, &F<__bf16, __bf16, __VA_ARGS__>}
#define XTC_SMALL(TM, TN) \
  {16 * TM, 16 * TN, {XTC_TYPES(small_launch, false, false, TM, TN), XTC_TYPES(small_launch, true, false, TM, TN), {}}}
const AnyTile kSlabs = {gany::BM, gany::BN, {XTC_TYPES(any_launch, false, false), XTC_TYPES(any_launch, true, false),
                                            XTC_TYPES(any_launch, false, true)}};
const AnyTile kSmall16 = {16, 16, {{}, XTC_TYPES(small_launch, true, false, 1, 1), {}}};  // streams transposed matrices
const AnyTile kSmall32 = XTC_SMALL(1, 2), kSmall64 = XTC_SMALL(1, 4);
const AnyTile kSmallGrad = {32, 32, {{}, {}, XTC_TYPES(small_launch, false, true, 2, 2)}};
#undef XTC_SMALL
#undef XTC_TYPES

int launch_any(const xtc_hip_grouped_matmul_desc& d, const AnyTile& t, bool grad, GroupedArgs& a, hipStream_t s, const char* what) {
  a.tiles_n = (a.N + t.bn - 1) / t.bn;
  a.tiles_k = (a.K + t.bm - 1) / t.bm;
  const int64_t groups = a.tiles_n * (grad ? (int64_t)a.E * a.tiles_k : most_tiles(a.T, a.E, t.bm));
  if (groups < 1 || groups >= (int64_t)1 << 31) return fail("%s: %lld workgroups are too many", what, (long long)groups);
  t.run[grad ? 2 : d.trans_w ? 1 : 0][d.dtype == XTC_HIP_F32 ? 0 : 1 + d.out_dtype](a, (unsigned)groups, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

// Tiles that a call has at most.
int64_t tiles_of(const AnyTile& t, bool grad, const GroupedArgs& a) {
  const int64_t n = (a.N + t.bn - 1) / t.bn;
  return n * (grad ? (int64_t)a.E * ((a.K + t.bm - 1) / t.bm) : most_tiles(a.T, a.E, t.bm));
}

// Few rows a group: the matrices are streamed once, by waves that share out their
// depth.  Matrices in rows of n are read 64 columns wide (8 rows over 8 experts of
// 4096 x 2048: 19 us, 25 at 32 columns, DMA tiles 27), matrices in rows of k 16
// columns a tile (16 us, 22; DMA 21).  From 8 and 4 rows a group on DMA tiles are
// as fast (8: 31 and 35 us against 35 and 33).  With more matrices the natural ones lose
// from fewer rows on (bf16, 8 rows at each of 16 of 4096 x 2048: 75 us, DMA tiles 49; of
// 64 of 1024 x 1024: 38, 29), the transposed ones do not (4 rows at each of 32 of 4096 x
// 2048: 97, 96; one: 56, 73).
// fp32 has slabs only to turn to: 64 rows over 8 of 4096 x 2048 51 us, 121 in slabs,
// 56 at 32 columns, which are faster for a row or two (1 x 4096 x 4096 18 us, 27).
// The rows of each group are not known here, only their mean: 512 rows that all fall to
// one of 64 groups stream its matrix once per 16, 70 us (DMA tiles 29), where they spread
// 243 (192).
const AnyTile* stream_tile(bool trans_w, const GroupedArgs& a) {
  const int rows = trans_w ? 4 : 8;
  return a.T > rows * (int64_t)a.E ? nullptr : trans_w ? &kSmall16 : &kSmall64;
}

// Any operands: tiles of shared depth where those of slabs would not fill the
// card, the wider ones where they do.  777 fp32 rows over 5 experts of 509 x 301:
// 10 us (32 columns), 22 in slabs; 4096 bf16 rows over 8 of 1001 x 999: 103, 68.
const AnyTile& any_tile(bool grad, const GroupedArgs& a) {
  if (tiles_of(kSlabs, grad, a) >= kFill) return kSlabs;
  if (grad) return kSmallGrad;
  return tiles_of(kSmall64, false, a) >= kFill ? kSmall64 : kSmall32;
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
  const hipStream_t s = core::pick_stream(d.stream);
  if (const AnyTile* t = stream_tile(d.trans_w, a)) return launch_any(d, *t, false, a, s, what);
  if (d.dtype == XTC_HIP_BF16 && d.K % 8 == 0 && (d.trans_w || d.N % 8 == 0) && vectors(x, a.ldx) && vectors(w, a.ldw) &&
      a.stride_w % 8 == 0) {
    double cost;
    const DmaTile& t = dma_tile(d.T, d.E, d.K, d.N, d.out_dtype == XTC_HIP_BF16 ? 2 : 4, &cost);
    // few tiles of deep K: waves that share out the depth, 256 of it a step of at
    // least .8 us, 3 in a round of 512 tiles (two a CU, one after the other in the natural
    // bf16 kernel, whose registers leave room for one; 512 rows over 2 experts of
    // 3584 x 256: 25 us on DMA tiles, 15 so), and a round of tiles has 4 us of its own:
    // finding the rows, the first loads, adding up and storing the sums (fp32 results:
    // 4100 rows over 6 of 32 x 3336 113 us so, 19 on DMA tiles; 9000 of 8 x 4104 456, 40)
    const double load = likely_tiles(d.T, d.E, 16) * ((d.N + 63) / 64) / 512;
    if (d.K / 256.0 * fmax(0.8, 3 * load) + 4 * load < cost) return launch_any(d, kSmall64, false, a, s, what);
    DmaArgs v{};
    v.a = (const uint8_t*)x, v.b = (const uint8_t*)w, v.sizes = sizes, v.c = y;
    v.stride_b = 2 * a.stride_w;
    v.E = d.E, v.M = d.T, v.N = d.N, v.K = d.K / 8;
    v.lda = 2 * a.ldx, v.ldb = 2 * a.ldw, v.ldc = a.ldy, v.out16 = d.out_dtype == XTC_HIP_BF16;
    v.tiles_m = (int)most_tiles(d.T, d.E, t.cost.bm);
    return launch_dma(t, d.trans_w ? t.transposed : t.natural, v, 1, s, what);
  }
  return launch_any(d, any_tile(false, a), false, a, s, what);
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
    const hipStream_t s = core::pick_stream(d.stream);
    int splits = 1;
    const DmaTile* t = &grad_tile(d.T, d.E, d.K, d.N, &splits);
    DmaArgs v{};
    v.a = (const uint8_t*)x, v.b = (const uint8_t*)dy, v.sizes = sizes, v.c = dw;
    v.stride_c = a.stride_y;
    v.E = d.E, v.M = d.T, v.N = d.N, v.K = d.K;
    v.lda = 2 * a.ldx, v.ldb = 2 * a.ldw, v.ldc = a.ldy, v.out16 = d.out_dtype == XTC_HIP_BF16;
    v.tiles_m = (d.K + t->cost.bm - 1) / t->cost.bm;
    v.splits = splits;
    if (splits > 1) {
      v.partial = core::partial_sums((size_t)splits * d.E * d.K * d.N * 4, s);
      if (!v.partial) v.splits = 1;
    }
    if (launch_dma(*t, t->grad, v, (int64_t)d.E * v.splits, s, what)) return 1;
    if (v.splits == 1) return 0;
    const int chunks = (int)(((int64_t)d.K * (d.N / 4) + 255) / 256);  // partial sums are small: kMostPartial
    hipLaunchKernelGGL(grouped_grad_sum, dim3((unsigned)(d.E * chunks)), dim3(256), 0, s, v, chunks);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(e));
  }
  return launch_any(d, any_tile(true, a), true, a, core::pick_stream(d.stream), what);
}

}  // extern "C"
