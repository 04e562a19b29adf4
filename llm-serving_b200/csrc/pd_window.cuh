// pd_window.cuh -- host-side declarations of the windowed chunk kernel (pd_window_prefill.cu).
#pragma once

#include "pd_common.cuh"

namespace pd {

struct WindowPrefillParams {
  const void* q;  // (total_q, H, D)
  int64_t q_st, q_sh;
  void* out;
  int64_t o_st, o_sh;
  const int32_t* cu_q;    // (B + 1) query-token offsets
  const int32_t* seqlen;  // (B) keys per row, the chunk included
  const int32_t* table;
  int64_t bt_stride;
  int64_t n_blocks;
  const void *k, *v;  // the pools, for rows that are computed again (pd_window_prefill.cu)
  int64_t k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;  // block, token, head
  int32_t total_q, max_seqlen_q;
  int32_t batch, n_kv_head, group;
  uint32_t group_mul;  // division by group (set by the launch)
  int32_t group_shift;
  int32_t max_blocks, capacity;
  int32_t log2_bs, log2_box;  // tokens of a block, and of a copy: min(block, WINDOW_BOX)
  int32_t window, sinks;
  int32_t grouped;  // pool maps: a copy is 8-token groups of all pieces, or one piece
  int32_t sms;
  float scale_log2;
  unsigned* err;
  unsigned long long wait_ns;
};

constexpr int WINDOW_BOX = 16;    // most tokens of a copy
constexpr int WINDOW_ROWS = 128;  // query rows of a block (the MMA's M)

cudaError_t launch_window_prefill(const WindowPrefillParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                  int dtype, int head_dim, cudaStream_t stream);

}  // namespace pd
