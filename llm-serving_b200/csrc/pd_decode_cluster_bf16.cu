// pd_decode_cluster_bf16.cu -- decode kernels of few rows for __nv_bfloat16 K/V: with a window, with weights.
#include "pd_decode_cluster.cuh"

namespace pd {

#define PD_CLUSTER_ROW(D, LOG)                                                              \
  {launch_cluster<__nv_bfloat16, D, 1, LOG>, launch_cluster<__nv_bfloat16, D, 2, LOG>, \
   launch_cluster<__nv_bfloat16, D, 4, LOG>, launch_cluster<__nv_bfloat16, D, 8, LOG>}

static const ClusterLaunchFn kClusterTable[2][3][4] = {
    {PD_CLUSTER_ROW(64, false), PD_CLUSTER_ROW(128, false), PD_CLUSTER_ROW(256, false)},
    {PD_CLUSTER_ROW(64, true), PD_CLUSTER_ROW(128, true), PD_CLUSTER_ROW(256, true)}};
#undef PD_CLUSTER_ROW

ClusterLaunchFn cluster_launcher_bf16(bool weights, int d_index, int gt_index) {
  if (d_index < 3 || d_index >= 6 || gt_index < 0 || gt_index >= 4) return nullptr;
  return kClusterTable[weights ? 1 : 0][d_index - 3][gt_index];
}

int cluster_room(int warps, int log2_split) {
  return warps == 4 ? cluster_room_of<__nv_bfloat16, 4>(log2_split) : cluster_room_of<__nv_bfloat16, 8>(log2_split);
}

}  // namespace pd
