// pd_decode_var_mma_bf16.cu -- tensor-core decode kernels for __nv_bfloat16 K/V with a window (variant 1) or with
// stored scores (variant 2): head dims 64, 128 and 256, q-head chunks of 1, 2, 4 or 8.
#include "pd_decode_kernel.cuh"

namespace pd {

#define PD_VAR_ROW(D, V)                                                                                 \
  {launch_decode<__nv_bfloat16, D, 1, false, true, V>, launch_decode<__nv_bfloat16, D, 2, false, true, V>, \
   launch_decode<__nv_bfloat16, D, 4, false, true, V>, launch_decode<__nv_bfloat16, D, 8, false, true, V>}

static const DecodeLaunchFn kVarTable[2][3][4] = {{PD_VAR_ROW(64, 1), PD_VAR_ROW(128, 1), PD_VAR_ROW(256, 1)},
                                                 {PD_VAR_ROW(64, 2), PD_VAR_ROW(128, 2), PD_VAR_ROW(256, 2)}};
#undef PD_VAR_ROW

DecodeLaunchFn decode_launcher_var_mma_bf16(int variant, int d_index, int gt_index) {
  if (variant < 1 || variant > 2 || d_index < 3 || d_index >= 6 || gt_index < 0 || gt_index >= 4) return nullptr;
  return kVarTable[variant - 1][d_index - 3][gt_index];
}

}  // namespace pd
