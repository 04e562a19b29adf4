// pd_decode_cluster_f32.cu -- decode kernels of few rows for float K/V: with a window, with weights.
#include "pd_decode_cluster.cuh"

namespace pd {

#define PD_CLUSTER_ROW(D, LOG)                                                              \
  {launch_cluster<float, D, 1, LOG>, launch_cluster<float, D, 2, LOG>, \
   launch_cluster<float, D, 4, LOG>, launch_cluster<float, D, 8, LOG>}

static const ClusterLaunchFn kClusterTable[2][3][4] = {
    {PD_CLUSTER_ROW(64, false), PD_CLUSTER_ROW(128, false), PD_CLUSTER_ROW(256, false)},
    {PD_CLUSTER_ROW(64, true), PD_CLUSTER_ROW(128, true), PD_CLUSTER_ROW(256, true)}};
#undef PD_CLUSTER_ROW

ClusterLaunchFn cluster_launcher_f32(bool weights, int d_index, int gt_index) {
  if (d_index < 3 || d_index >= 6 || gt_index < 0 || gt_index >= 4) return nullptr;
  return kClusterTable[weights ? 1 : 0][d_index - 3][gt_index];
}

}  // namespace pd
