// pd_fp4.cuh -- the 4-bit page format, its conversions, and the parameter blocks of the kernels
// that write, read and attend over it (sm_100a).
//
// A pool is uint8 (n_blocks, n_kv_head, block_size / 16, 18 * head_dim): the last dimension is the
// record of 16 consecutive tokens of one kv head. With W = min(head_dim, 128):
//   K codes   8 D bytes  [D / W][16 tokens][W / 2]
//   K scales    D bytes  [D / W][16 tokens][W / 16]
//   V codes   8 D bytes  [2 halves][D / 16 groups][8 tokens][8]
//   V scales    D bytes  [2 halves][D / 16 groups][8 tokens]
// A code is e2m1 (sign, two exponent bits, one mantissa bit: 0 .5 1 1.5 2 3 4 6), two to a byte, the
// lower element in the low nibble; a scale is e4m3, one for 16 neighbouring elements. An element
// stands for code * scale * unit, unit a power of two kept per (K or V, kv head). A code has 2
// significant bits and a scale 4, so code * scale is exact in fp16 and in bf16.
//
// Why this layout: one (page, head) record holds K, V and their scales contiguously, so a tile is
// one run of 18 D bytes in memory. Inside it the bytes stand in the order in which a warp's lanes
// read them as MMA operands: lane (g, c) = (lane / 4, lane % 4) takes K token g's 32 elements from
// 32 c (one 16-byte load, quarter-warps on 128 consecutive bytes), and V group g's elements of
// tokens 2 c, 2 c + 1 (again one 16-byte load of consecutive bytes), so no shared-memory read has
// a bank conflict and no operand needs a transposing load.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>

#include "pd_common.cuh"
#include "pd_smem_limit.cuh"

namespace pd {

constexpr int FP4_TILE = 16;   // tokens of a record
constexpr int FP4_GROUP = 16;  // elements that share a scale

// Attention weights are kept as 2^(s - m + SHIFT), m the running maximum, and the sums carry the same factor.
// The maximum moves only when a score passes it by 2^HEADROOM, so a weight stays below 2^15, inside fp16, and one
// of 2^-21 of the largest is still a normal fp16 number. (Without the factor that end was 2^-14: rows with
// one key far above the others lost the others' bits.)
constexpr float FP4_HEADROOM = 8.f;
constexpr float FP4_P_SHIFT = 7.f;

__host__ __device__ constexpr int fp4_record_bytes(int d) { return 18 * d; }

// Byte offsets inside a record: of the 8 code bytes of group `gr` (16 elements) of token `t`, and
// of its scale byte.
__host__ __device__ __forceinline__ int fp4_k_code(int d, int t, int gr) {
  const int w = d < 128 ? d : 128, per = w / 16;
  return (gr / per) * 8 * w + t * (w / 2) + (gr % per) * 8;
}
__host__ __device__ __forceinline__ int fp4_k_scale(int d, int t, int gr) {
  const int w = d < 128 ? d : 128, per = w / 16;
  return 8 * d + (gr / per) * w + t * per + gr % per;
}
__host__ __device__ __forceinline__ int fp4_v_code(int d, int t, int gr) {
  return 9 * d + (t >> 3) * 4 * d + gr * 64 + (t & 7) * 8;
}
__host__ __device__ __forceinline__ int fp4_v_scale(int d, int t, int gr) {
  return 17 * d + (t >> 3) * (d / 2) + gr * 8 + (t & 7);
}

// Four code bytes -> four pairs of fp16 (low nibble in the low half), exact.
__device__ __forceinline__ void e2m1x8_to_half2x4(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}

// Two e4m3 scale bytes -> a pair of fp16, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
  uint32_t r;
  const uint16_t h = uint16_t(two);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
  return r;
}

// fp32 -> e4m3 byte, to nearest even, saturating at 448.
__device__ __forceinline__ uint32_t float_to_e4m3(float x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(x));
  return uint32_t(r) & 0xffu;
}

// Eight fp32 -> four code bytes (lower element in the low nibble), to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t floats_to_e2m1x8(const float* f) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}

__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// ------------------------------------------------------------------ parameter blocks

// Write of tokens into 4-bit pages, and the read back. Element strides of the 16/32-bit side.
struct Fp4RowsParams {
  unsigned char* pages;
  int64_t n_blocks;
  int32_t block_size;
  int32_t n_kv_head;
  int32_t head_dim;
  const float* units;  // (2, n_kv_head) or nullptr (all 1)
  const void* slots;   // slot of token i, int32 or int64, unless `table`
  int32_t slot_i64;
  const int32_t* table;  // decode step: slot from table[i, pos[i] / block_size] and pos[i]
  int64_t bt_stride;
  int32_t max_blocks;
  const int64_t* pos;
  void* k;
  void* v;
  int64_t k_s0, k_s1, v_s0, v_s1;
  int64_t n_tokens;
  unsigned* err;
};

// Attention of query tokens over 4-bit pages.
struct Fp4AttendParams {
  const void* q;  // (total_q, H, D)
  int64_t q_st, q_sh;
  int32_t total_q;
  void* out;
  int64_t o_st, o_sh;
  const unsigned char* pages;
  int64_t n_blocks;
  const float* units;  // (2, n_kv_head) or nullptr
  const int32_t* table;
  int64_t bt_stride;
  const int32_t* seqlen;  // keys per row, the chunk included
  const int32_t* cu_q;    // (B + 1), or nullptr: one query token per row
  int32_t max_seqlen_q;
  int32_t max_blocks;
  int32_t capacity;
  int32_t batch;
  int32_t n_kv_head;
  int32_t group;
  int32_t log2_tpb;  // log2(block_size / 16)
  float scale_log2;
  unsigned* counters;  // one per CTA, zero between launches
  float* partials;     // two slots per CTA
  unsigned* err;
  unsigned long long wait_ns;
};

// Launchers. sms: multiprocessors of the current device.
cudaError_t launch_fp4_rows(const Fp4RowsParams& p, int dtype, bool read, bool vec, int sms, cudaStream_t stream);
cudaError_t launch_fp4_attend(const Fp4AttendParams& p, int dtype, int head_dim, int sms, cudaStream_t stream);
// The same for long chunks, on tcgen05 tiles (pd_fp4_prefill.cu); needs cu_q.
cudaError_t launch_fp4_prefill(const Fp4AttendParams& p, int dtype, int head_dim, cudaStream_t stream);
int fp4_max_rows();  // rows of one attention launch
size_t fp4_counter_bytes(int sms);
size_t fp4_workspace_bytes(int head_dim, int sms);

}  // namespace pd
