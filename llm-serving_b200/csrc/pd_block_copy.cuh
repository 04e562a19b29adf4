// pd_block_copy.cuh -- parameter block of the page copy kernel (pd_block_copy.cu).
#pragma once

#include "pd_common.cuh"

namespace pd {

// A block id outside the pool in a copy (mirrors PD_DEVERR_COPY_RANGE).
constexpr unsigned DEVERR_COPY_RANGE = 8u;

constexpr int COPY_PIECE = 8192;      // bytes one CTA moves at a time
constexpr int COPY_MAX_POOLS = 128;   // pools of one launch (their addresses are kernel parameters)

struct BlockCopyParams {
  unsigned char* pools[COPY_MAX_POOLS];
  int32_t n_pools;
  int32_t ids_i64;
  int64_t n_blocks;
  int64_t block_bytes;
  const void* src;
  const void* dst;
  int64_t n_pairs;
  int32_t* table;  // or nullptr
  int64_t table_rows, table_cols, table_st;
  const int32_t* remap;
  int32_t vec16;  // pools and block size are multiples of 16 bytes
  unsigned* err;
};

cudaError_t launch_block_copy(const BlockCopyParams& p, int sms, cudaStream_t stream);

}  // namespace pd
