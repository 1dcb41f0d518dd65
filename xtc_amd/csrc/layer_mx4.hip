// SPDX-License-Identifier: BSD-3-Clause
// The expert layer's kernels for matrices of one kind.
#include "layer.hpp"

namespace xtc_hip {
XTC_HIP_LAYER_LAUNCH(layer::MX4)
}  // namespace xtc_hip
