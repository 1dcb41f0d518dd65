// SPDX-License-Identifier: BSD-3-Clause
// Entry points of layer norm.
#include "xtc_hip.h"
#include "core.hpp"
#include "norm.hpp"

using namespace xtc_hip;
using core::fail;

namespace {

constexpr int kMost = 0x7fffffff - 16383;  // of K: a walk's step past it stays within 32 bits
constexpr int kLong = 16384;               // elements of a row that registers hold
constexpr int64_t kMostGroups = 1 << 20;   // of a launch: its threads stay within 32 bits
constexpr int64_t kWalks = 1024;           // workgroups of 256 threads that walk over the rows: four a CU (a
                                           // row each and no walk: 149 us of 32768 x 4096, this 129, both
                                           // with the rows read through the caches)
constexpr int kMostParts = XTC_HIP_LAYER_NORM_PARTS;

constexpr int64_t kMostColumns = 65535ll * 2048;  // of the parameters' sums: a launch's second extent

int check(const xtc_hip_layer_norm_desc* d, const char* what) {
  if (!core::ready()) return fail("xtc_hip_init not called");
  if (!d) return fail("%s: null descriptor", what);
  if (d->dtype != XTC_HIP_F32 && d->dtype != XTC_HIP_BF16) return fail("%s: unsupported dtype %d", what, d->dtype);
  if (d->param_dtype != XTC_HIP_F32 && !(d->param_dtype == XTC_HIP_BF16 && d->dtype == XTC_HIP_BF16))
    return fail("%s: unsupported dtype %d of the parameters for rows of dtype %d", what, d->param_dtype, d->dtype);
  if (d->rows < 0 || d->K < 1) return fail("%s: invalid sizes rows=%lld K=%d", what, (long long)d->rows, d->K);
  if (!(d->eps >= 0) || d->eps > 3.4e38f) return fail("%s: eps %g is not a finite number from 0 on", what, d->eps);
  if ((d->ldx && d->ldx < d->K) || (d->ldy && d->ldy < d->K))
    return fail("%s: row strides %d and %d are below the %d elements of a row", what, d->ldx, d->ldy, d->K);
  const int64_t ld = d->ldx > d->ldy ? d->ldx : d->ldy;
  if (d->K > kMost || d->rows >= (int64_t)1 << 31 || d->rows > INT64_MAX / 8 / (ld > d->K ? ld : d->K))
    return fail("%s: sizes rows=%lld K=%d are too many", what, (long long)d->rows, d->K);
  return 0;
}

int done(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

NormArgs args_of(const xtc_hip_layer_norm_desc& d, const void* x, const void* w) {
  NormArgs a{};
  a.x = x, a.w = w, a.rows = d.rows, a.K = d.K, a.eps = d.eps;
  a.ldx = d.ldx ? d.ldx : d.K, a.ldy = d.ldy ? d.ldy : d.K;
  return a;
}

// Threads that share a row: as few as hold it in two runs of 8 elements each; the backward
// pass, whose registers then leave two workgroups a CU little to run, in one run from 2048
// elements to 4096.
int threads_of(int K, bool grad) { return K <= 1024 ? 64 : K <= (grad ? 2048 : 4096) ? 256 : grad && K <= 4096 ? 512 : 1024; }

template <typename T, typename P, int THREADS, int VECS>
void run_forward(const NormArgs& a, unsigned groups, hipStream_t s) {
  hipLaunchKernelGGL((layer_norm<T, P, THREADS, VECS>), dim3(groups), dim3(THREADS < 256 ? 256 : THREADS), 0, s, a);
}
template <typename T, typename P, int THREADS, int VECS>
void run_grad(const NormArgs& a, unsigned groups, hipStream_t s) {
  const dim3 threads(THREADS < 256 ? 256 : THREADS);
  if constexpr (sizeof(T) == 4 && THREADS == 1024)
    // a dx that the caches do not hold beside what was read (stream.hpp)
    if (a.y && a.rows * a.K * 4 >= stream::LARGE) {
      hipLaunchKernelGGL((layer_norm_grad<true, T, P, THREADS, VECS>), dim3(groups), threads, 0, s, a);
      return;
    }
  hipLaunchKernelGGL((layer_norm_grad<false, T, P, THREADS, VECS>), dim3(groups), threads, 0, s, a);
}
template <typename T, typename P, int THREADS, int VECS>
void run_rows(const NormArgs& a, bool grad, unsigned groups, hipStream_t s) {
  if (grad) run_grad<T, P, THREADS, VECS>(a, groups, s);
  else run_forward<T, P, THREADS, VECS>(a, groups, s);
}

template <typename T, typename P>
void run(const NormArgs& a, bool grad, unsigned groups, hipStream_t s) {
  if (a.K > kLong) {
    if (grad) hipLaunchKernelGGL((layer_norm_long<T, P, true>), dim3(groups), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((layer_norm_long<T, P, false>), dim3(groups), dim3(1024), 0, s, a);
    return;
  }
  const int threads = threads_of(a.K, grad);
  const bool one = a.K <= 8 * threads;
  if (threads == 64) return one ? run_rows<T, P, 64, 1>(a, grad, groups, s) : run_rows<T, P, 64, 2>(a, grad, groups, s);
  if (threads == 256) return one ? run_rows<T, P, 256, 1>(a, grad, groups, s) : run_forward<T, P, 256, 2>(a, groups, s);
  if (threads == 512) return run_grad<T, P, 512, 1>(a, groups, s);
  return one ? run_rows<T, P, 1024, 1>(a, grad, groups, s) : run_rows<T, P, 1024, 2>(a, grad, groups, s);
}

void launch(const xtc_hip_layer_norm_desc& d, const NormArgs& a, bool grad, unsigned groups) {
  const hipStream_t s = core::pick_stream(d.stream);
  if (d.dtype == XTC_HIP_F32) run<float, float>(a, grad, groups, s);
  else if (d.param_dtype == XTC_HIP_F32) run<__bf16, float>(a, grad, groups, s);
  else run<__bf16, __bf16>(a, grad, groups, s);
}

// Workgroups of the backward pass, each with a part of the parameters' sums.
int64_t parts_of(const xtc_hip_layer_norm_desc& d) {
  const int64_t rows = d.K <= 1024 ? (d.rows + 3) / 4 : d.rows;
  return rows < kMostParts ? rows : kMostParts;
}

}  // namespace

extern "C" {

int xtc_hip_layer_norm_desc_size(void) { return (int)sizeof(xtc_hip_layer_norm_desc); }

int xtc_hip_layer_norm(const xtc_hip_layer_norm_desc* desc, const void* x, const void* w, const void* b, void* y) {
  const char* const what = "layer_norm";
  if (check(desc, what)) return 1;
  if (desc->rows == 0) return 0;
  if (!x || !y) return fail("%s: null operand", what);
  NormArgs a = args_of(*desc, x, w);
  a.b = b, a.y = y;
  const int64_t groups = a.K > 1024 ? a.rows : (a.rows + 3) / 4, most = a.K > kLong ? kMostGroups : a.K > 4096 ? 512 : kWalks;
  launch(*desc, a, false, (unsigned)(groups < most ? groups : most));
  return done(what);
}

int xtc_hip_layer_norm_grad(const xtc_hip_layer_norm_desc* desc, const void* x, const void* w, const void* dy, void* dx,
                            float* dw, float* db, float* workspace) {
  const char* const what = "layer_norm_grad";
  if (check(desc, what)) return 1;
  const bool sums = dw || db;
  if (!dx && !sums) return fail("%s: no result is asked for", what);
  if (desc->rows && (!x || !dy)) return fail("%s: null operand", what);
  if (desc->rows && sums && !workspace) return fail("%s: sums over the rows need a workspace", what);
  if (sums && desc->K > kMostColumns) return fail("%s: rows of %d elements are too many to sum over", what, desc->K);
  const hipStream_t s = core::pick_stream(desc->stream);
  NormArgs a = args_of(*desc, x, w);
  const int parts = (int)parts_of(*desc);
  if (parts) {
    a.dy = dy, a.y = dx, a.parts = sums ? workspace : nullptr;
    if (a.K > kLong) {
      a.stats = sums ? workspace + 2 * (size_t)parts * a.K : nullptr;
      launch(*desc, a, true, (unsigned)(a.rows < kMostGroups ? a.rows : kMostGroups));
      if (sums) {
        const dim3 grid((unsigned)parts, (unsigned)(((int64_t)a.K + 2047) / 2048));
        if (desc->dtype == XTC_HIP_F32) hipLaunchKernelGGL(layer_norm_grad_columns<float>, grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL(layer_norm_grad_columns<__bf16>, grid, dim3(256), 0, s, a);
      }
    } else {
      launch(*desc, a, true, (unsigned)parts);
    }
    if (done(what)) return 1;
  }
  if (sums) {
    hipLaunchKernelGGL(layer_norm_grad_sum, dim3((unsigned)(((int64_t)a.K + 63) / 64), 2), dim3(1024), 0, s, workspace, dw, db, parts, a.K);
    return done(what);
  }
  return 0;
}

}  // extern "C"
