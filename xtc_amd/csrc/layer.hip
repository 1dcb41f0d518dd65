// SPDX-License-Identifier: BSD-3-Clause
// Entry points of the layer of experts for a few tokens.
#include "xtc_hip.h"
#include "core.hpp"
#include "layer.hpp"

using namespace xtc_hip;
using core::aligned16;
using core::fail;

namespace {

constexpr int kMost = 0x7fffffff - 1023;
constexpr int kMostTokens = 64, kMostExperts = 256, kMostChosen = 16, kMostLogitParts = 8;
// Workgroups of a launch, as many as the CUs hold at once: they walk over all pieces.
int64_t groups_of(const xtc_hip_expert_layer_desc& d) { return d.weights == XTC_HIP_WEIGHTS_MX4 ? 512 : 768; }

int check(const xtc_hip_expert_layer_desc* d, const char* what) {
  if (!d) return fail("%s: null descriptor", what);
  if (d->dtype != XTC_HIP_F32 && d->dtype != XTC_HIP_BF16) return fail("%s: unsupported dtype %d", what, d->dtype);
  if (d->weights != XTC_HIP_WEIGHTS_DENSE && d->weights != XTC_HIP_WEIGHTS_FP8 && d->weights != XTC_HIP_WEIGHTS_MX4)
    return fail("%s: unsupported kind %d of matrices", what, d->weights);
  if (d->weights != XTC_HIP_WEIGHTS_DENSE && d->dtype != XTC_HIP_BF16)
    return fail("%s: 8-bit and 4-bit matrices take bf16 rows, not dtype %d", what, d->dtype);
  if (d->activation != XTC_HIP_RELU && d->activation != XTC_HIP_SWIGLU) return fail("%s: unsupported activation %d", what, d->activation);
  if (d->T < 0 || d->E < 1 || d->K < 1 || d->H < 1 || d->top_k < 1)
    return fail("%s: invalid sizes T=%d E=%d K=%d H=%d top_k=%d", what, d->T, d->E, d->K, d->H, d->top_k);
  if (d->T > kMostTokens || d->E > kMostExperts || d->top_k > kMostChosen || d->top_k > d->E)
    return fail("%s: T=%d, E=%d or top_k=%d are too many: at most %d tokens, %d experts, and %d of them a token", what, d->T, d->E,
                d->top_k, kMostTokens, kMostExperts, kMostChosen);
  if (d->K > kMost || d->H > kMost / 2) return fail("%s: sizes K=%d H=%d are too many", what, d->K, d->H);
  if ((d->ldx && d->ldx < d->K) || (d->ldy && d->ldy < d->K))
    return fail("%s: row strides %d and %d are below the %d columns", what, d->ldx, d->ldy, d->K);
  if (d->hidden_f32 != 0 && d->hidden_f32 != 1) return fail("%s: hidden_f32 %d is neither 0 nor 1", what, d->hidden_f32);
  return 0;
}

uint64_t padded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

struct Workspace {
  uint64_t mid, parts, logits, choice, counters, total;
};
Workspace workspace_of(const xtc_hip_expert_layer_desc& d) {
  const uint64_t slots = (uint64_t)d.T * d.top_k, hidden = ((uint64_t)d.H + 31) / 32 * 32;
  Workspace w{};
  // an activation is an fp32 number, or up to three bf16 ones
  w.parts = w.mid + padded((d.dtype == XTC_HIP_F32 ? 4 : 6) * slots * hidden);
  w.logits = w.parts + padded(4 * slots * d.K);
  w.choice = w.logits + padded(4ull * kMostLogitParts * d.T * d.E);
  w.counters = w.choice + padded(4 * slots);
  w.total = w.counters + padded(4 * (((uint64_t)d.K + 15) / 16));
  return w;
}

}  // namespace

extern "C" {

int xtc_hip_expert_layer_desc_size(void) { return (int)sizeof(xtc_hip_expert_layer_desc); }

uint64_t xtc_hip_expert_layer_workspace(const xtc_hip_expert_layer_desc* desc) {
  return check(desc, "expert_layer_workspace") ? 0 : workspace_of(*desc).total;
}

int xtc_hip_expert_layer(const xtc_hip_expert_layer_desc* desc, const void* x, const void* router, const void* up,
                         const uint8_t* up_scales, const void* down, const uint8_t* down_scales, void* workspace,
                         uint64_t workspace_bytes, void* y) {
  const char* const what = "expert_layer";
  if (!core::ready()) return fail("xtc_hip_init not called");
  if (check(desc, what)) return 1;
  const xtc_hip_expert_layer_desc& d = *desc;
  if (d.T == 0) return 0;
  const bool packed = d.weights != XTC_HIP_WEIGHTS_DENSE;
  if (!x || !router || !up || !down || !y || !workspace || (packed && (!up_scales || !down_scales))) return fail("%s: null operand", what);
  if (!packed && (up_scales || down_scales)) return fail("%s: scales with matrices that have none", what);
  if (packed && (!aligned16(up) || !aligned16(down))) return fail("%s: codes must be 16-byte aligned", what);
  if (!aligned16(workspace)) return fail("%s: the workspace must be 16-byte aligned", what);
  const Workspace w = workspace_of(d);
  if (workspace_bytes < w.total)
    return fail("%s: a workspace of %llu bytes, %llu are needed", what, (unsigned long long)workspace_bytes, (unsigned long long)w.total);
  char* const ws = (char*)workspace;
  LayerArgs a{};
  a.x = x, a.router = router, a.up = up, a.down = down, a.up_scales = up_scales, a.down_scales = down_scales, a.y = y;
  a.mid = ws + w.mid, a.parts = (float*)(ws + w.parts), a.choice = (int*)(ws + w.choice), a.counters = (unsigned*)(ws + w.counters);
  a.T = d.T, a.E = d.E, a.K = d.K, a.H = d.H, a.Hp = (d.H + 31) / 32 * 32, a.top_k = d.top_k;
  a.ldx = d.ldx ? d.ldx : d.K, a.ldy = d.ldy ? d.ldy : d.K;
  a.normalize = d.normalize != 0, a.swiglu = d.activation == XTC_HIP_SWIGLU;
  a.planes = d.dtype == XTC_HIP_BF16 && d.hidden_f32 ? 3 : 1;
  const hipStream_t s = core::pick_stream(d.stream);

  LayerGrid grid{};
  // experts that tokens may choose, and the tiles of 16 rows of all of them
  const int most = d.T * d.top_k < d.E ? d.T * d.top_k : d.E;
  const int64_t tiles = most * (((int64_t)d.H * (a.swiglu ? 2 : 1) + 15) / 16);
  // Waves that share k, four or two, us: dense matrices always take four (bf16, 512 tiles 19.8,
  // 24.8, 2048 tiles 43.6, 47.7, 8192 tiles 109, 114); packed ones, whose tokens go through LDS
  // twice as often a byte, two from 2048 tiles (4 bits, 256 tiles 23.2, 27.3, 1024 tiles 23.5,
  // 25.0, 2048 tiles of 8 tokens 45.7, 43.9 and of 32 60.7, 54.8; 8 bits, 2048 tiles 41.6, 38.2)
  grid.shared = !packed || tiles < 2048;
  // pieces of 32 rows of `down` that leave CUs idle are halved (64 of them 9.1 us, 128 of 16 rows
  // 7.0; from 256 on, a piece a CU, halves would only read the tokens twice)
  grid.narrow = grid.shared && ((int64_t)d.K + 31) / 32 * most < 256;
  const int up_rows = (a.swiglu ? 16 : 32) * (grid.shared ? 1 : 2), down_rows = (grid.narrow ? 16 : 32) * (grid.shared ? 1 : 2);
  const int64_t up_slices = ((int64_t)a.Hp + up_rows - 1) / up_rows, down_slices = ((int64_t)d.K + down_rows - 1) / down_rows;
  if (up_slices * most >= 1 << 30 || down_slices * most >= 1 << 30)
    return fail("%s: %lld pieces of work are too many", what, (long long)((up_slices > down_slices ? up_slices : down_slices) * most));
  const int64_t groups = groups_of(d);
  grid.up_slices = (int)up_slices, grid.down_slices = (int)down_slices;
  grid.up = (unsigned)(up_slices * most < groups ? up_slices * most : groups);
  grid.down = (unsigned)(down_slices * most < groups ? down_slices * most : groups);

  // router and tokens that every workgroup of layer_up reads again: in a launch of their own
  // from 64 KB (us, within layer_up and by themselves: 18 KB 19.8, 21.3, 34 KB 22.2, 24.7, 72 KB
  // 37.2, 35.8, 96 KB 43.6, 42.3, 272 KB 56.9, 38.2)
  const int esz = d.dtype == XTC_HIP_F32 ? 4 : 2;
  const int pairs = (d.E + 15) / 16 * ((d.T + 15) / 16);
  if (d.T > layer::ROUND || d.T * d.E > layer::LOGITS || pairs > 4 || ((int64_t)d.T + d.E) * d.K * esz > 64 << 10) {
    a.logits = (float*)(ws + w.logits);
    a.logit_parts = pairs >= 16 ? 2 : pairs >= 4 ? 4 : 8;
    const dim3 logits((unsigned)((d.T + 15) / 16), (unsigned)((d.E + 15) / 16), (unsigned)a.logit_parts);
    if (d.dtype == XTC_HIP_F32) hipLaunchKernelGGL(layer_logits<float>, logits, dim3(layer::THREADS), 0, s, a);
    else hipLaunchKernelGGL(layer_logits<__bf16>, logits, dim3(layer::THREADS), 0, s, a);
  }
  if (d.dtype == XTC_HIP_F32) layer_launch<layer::F32>(a, grid, s);
  else if (d.weights == XTC_HIP_WEIGHTS_FP8) layer_launch<layer::FP8>(a, grid, s);
  else if (d.weights == XTC_HIP_WEIGHTS_MX4) layer_launch<layer::MX4>(a, grid, s);
  else layer_launch<layer::BF16>(a, grid, s);
  const hipError_t err = hipGetLastError();
  return err == hipSuccess ? 0 : fail("%s: launch failed: %s", what, hipGetErrorString(err));
}

}  // extern "C"
