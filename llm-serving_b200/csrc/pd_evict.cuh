// pd_evict.cuh -- host-side declarations of the eviction kernels (pd_evict.cu).
#pragma once

#include "pd_common.cuh"

namespace pd {

constexpr int EVICT_LAYERS = 64;  // layers of one launch: their pool pointers travel in the parameters
constexpr int EVICT_UNITS = 256;  // most 16-byte units of a row: the move gives each a thread of a CTA

struct EvictParams {
  void* k[EVICT_LAYERS];
  void* v[EVICT_LAYERS];
  int64_t k_sb, k_sn, k_sh, v_sb, v_sn, v_sh;  // pool strides in 16-byte units: block, token, head
  int64_t n_blocks;
  const int32_t* table;  // where the tokens are
  int64_t bt_stride;
  const int32_t* new_table;  // where the kept ones go (the same table: in place)
  int64_t nbt_stride;
  const int32_t* seqlen;
  int32_t* seqlen_out;  // written by the move kernel, which does not read seqlen; nullptr: not by this launch
  const float* weights;
  float* weights_out;
  int64_t w_sl, w_sb, w_sh, wo_sl, wo_sb, wo_sh;
  int64_t w_len;
  int32_t* order;  // (layers, B, H_kv, keep): the kept tokens, from the first that moves
  int2* info;      // (layers, B, H_kv): tokens before the first that moves, tokens kept
  unsigned* err;
  int32_t layers, batch, n_kv_head, chunks;  // chunks: 16-byte units of a row
  int32_t log2_bs, max_blocks, new_max_blocks, capacity;
  int32_t keep, recent, sinks;
  int32_t fresh;  // new pages: every kept token is copied
  int32_t sms;
};

cudaError_t launch_evict(const EvictParams& p, cudaStream_t stream);

}  // namespace pd
