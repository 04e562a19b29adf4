// pd_decode_var_f32.cu -- CUDA-core decode kernels for float K/V that take a window and store scores
// (variant 3: each by its arguments): head dims 8..256, q-head chunks of 1, 2, 4 or 8.
#include "pd_decode_kernel.cuh"

namespace pd {

#define PD_VAR_ROW(D)                                                                                  \
  {launch_decode<float, D, 1, false, false, 3>, launch_decode<float, D, 2, false, false, 3>, \
   launch_decode<float, D, 4, false, false, 3>, launch_decode<float, D, 8, false, false, 3>}

static const DecodeLaunchFn kVarTable[6][4] = {PD_VAR_ROW(8),  PD_VAR_ROW(16),  PD_VAR_ROW(32),
                                              PD_VAR_ROW(64), PD_VAR_ROW(128), PD_VAR_ROW(256)};
#undef PD_VAR_ROW

DecodeLaunchFn decode_launcher_var_f32(int d_index, int gt_index) {
  if (d_index < 0 || d_index >= 6 || gt_index < 0 || gt_index >= 4) return nullptr;
  return kVarTable[d_index][gt_index];
}

}  // namespace pd
