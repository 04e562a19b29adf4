// pd_norm_rope.cuh -- parameter block of the head norm + rotation kernel (pd_norm_rope.cu).
#pragma once

#include "pd_common.cuh"

namespace pd {

// A position outside the cos/sin tables (mirrors PD_DEVERR_ROPE_RANGE).
constexpr unsigned DEVERR_ROPE_RANGE = 4u;

// Element strides; q, k, the weights, the tables and the outputs share one dtype.
struct NormRopeParams {
  const void* q;
  const void* k;
  int64_t q_st, q_sh, k_st, k_sh;
  void* q_out;
  void* k_out;
  int64_t qo_st, qo_sh, ko_st, ko_sh;
  const void* wq;
  const void* wk;
  const void* cos;
  const void* sin;
  int64_t cos_st, sin_st;
  int64_t n_pos;    // rows of the tables
  const void* pos;  // (n_tokens) int32 / int64, or nullptr: token t at position t
  int32_t pos_i64;
  int64_t n_tokens;
  int32_t n_head, n_kv_head, head_dim, rotary_dim;
  float eps;
  unsigned* err;
};

cudaError_t launch_norm_rope(const NormRopeParams& p, int dtype, bool vec, int sms, cudaStream_t stream);

}  // namespace pd
