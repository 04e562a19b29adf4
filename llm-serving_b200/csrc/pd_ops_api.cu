// pd_ops_api.cu -- the extern "C" boundary of the head norm with rotation, the 4-bit pages, the
// page copies and the eviction (declared in include/paged_decode.h): argument checks on the host, then the launch.
#include <algorithm>
#include <atomic>
#include <exception>
#include <vector>

#include "paged_decode.h"
#include "pd_api_internal.h"
#include "pd_block_copy.cuh"
#include "pd_evict.cuh"
#include "pd_fp4.cuh"
#include "pd_norm_rope.cuh"

namespace pd {

namespace {

// Kernel of pd_fp4_prefill: 0 chooses, 1 warp kernel, 2 tcgen05 tiles.
std::atomic<int> g_fp4_prefill_mode{0};

bool valid_dtype(int dtype) { return dtype == PD_F32 || dtype == PD_F16 || dtype == PD_BF16; }
int elem_size(int dtype) { return dtype == PD_F32 ? 4 : 2; }
bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1u)) == 0; }
bool pow2(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }
int ilog2_host(int64_t x) {
  int r = 0;
  while ((int64_t(1) << (r + 1)) <= x) ++r;
  return r;
}
bool fp4_head_dim(int d) { return d == 64 || d == 128 || d == 256; }

int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) return api_cuda_fail(e, what);
  api_count_launch();
  return PD_OK;
}

// What every entry point over 4-bit pages asks of the pool.
int check_pool(const void* pages, int64_t n_blocks, int32_t block_size, int32_t n_kv_head, int32_t head_dim) {
  if (n_blocks < 1 || n_kv_head < 1 || !pow2(block_size)) return PD_ERR_INVALID;
  if (!fp4_head_dim(head_dim) || block_size < FP4_TILE) return PD_ERR_UNSUPPORTED;
  // the kernels hold a block's bytes and offsets in it in 32 bits
  if (int64_t(n_kv_head) * (block_size / FP4_TILE) > 0x7fffffff / fp4_record_bytes(head_dim)) return PD_ERR_UNSUPPORTED;
  if (pages == nullptr || !aligned(pages, 16)) return PD_ERR_INVALID;
  return PD_OK;
}

int rows_common(Fp4RowsParams& p, int dtype, bool read, const int64_t* k_strides, const int64_t* v_strides,
                void* stream) {
  if (!valid_dtype(dtype) || p.n_tokens < 0 || k_strides == nullptr || v_strides == nullptr) return PD_ERR_INVALID;
  const int st = check_pool(p.pages, p.n_blocks, p.block_size, p.n_kv_head, p.head_dim);
  if (st != PD_OK) return st;
  if (p.n_tokens == 0) return PD_OK;
  if (p.k == nullptr || p.v == nullptr) return PD_ERR_INVALID;
  p.k_s0 = k_strides[0];
  p.k_s1 = k_strides[1];
  p.v_s0 = v_strides[0];
  p.v_s1 = v_strides[1];
  int sms = 0;
  if (api_device(&sms, &p.err) != PD_OK) return PD_ERR_CUDA;
  const int es = elem_size(dtype);
  bool vec = aligned(p.k, 16) && aligned(p.v, 16);
  for (const int64_t s : {p.k_s0, p.k_s1, p.v_s0, p.v_s1}) vec = vec && (s * es) % 16 == 0;
  return launched(launch_fp4_rows(p, dtype, read, vec, sms, static_cast<cudaStream_t>(stream)),
                  read ? "4-bit read launch" : "4-bit write launch");
}

// Whether a chunk call runs on tcgen05 tiles. Per visible key, the warp kernel's time goes with the
// 8-column units of query rows per SM, the tile kernel's with the waves of its CTAs, one block of 256
// (at head_dim 256: 128) query rows each, whatever part of the block is filled; a wave costs what
// WAVE_UNITS units per SM cost. Lengths stay on the device, but both times are proportional to them, so the
// comparison needs only the counts the host has. Measured, warp kernel and tiles, 16 heads on 8 of 128
// with 2048 keys: 16 rows of 8 tokens (2.2 units per SM, one wave) 28.5 and 38.1 us, of 16 (3.9) 42.4 and
// 38.5, of 32 (7.4) 72.8 and 38.9, one row of 1024 tokens (13.9) 185 and 52; 8 heads on 2 of 256: 16 rows
// of 16 tokens (1.8) 43.6 and 48.3, of 32 (3.6) 72.3 and 48.6; 4 heads on 4 of 64: one row of 1024 tokens
// (3.5) 39.2 and 47.1, 16 rows of 128 (7.1) 51.9 and 31.1. In fp16 P's second part slows both: 16 rows of
// 8 tokens 30.9 and 48.0, of 16 47.5 and 48.2, of 32 80.3 and 48.3; with the same constants the choice is within
// 12 % of the better kernel over 64 such shapes (the worst, 32 rows of 16 tokens with 1024 keys, 49.4 and
// 55.0), but for one with few keys, where the warp kernel's start counts more (in both types: 4 rows of 64
// tokens with 512 keys at head_dim 256, 25.2 and 21.0).
bool use_tiles(int64_t total_q, int32_t max_seqlen_q, int32_t batch, int32_t n_kv_head, int32_t group,
               int32_t head_dim, int sms) {
  const double WAVE_UNITS = head_dim == 256 ? 2.1 : head_dim == 128 ? 3.3 : 4.3;
  const int64_t block = head_dim == 256 ? 128 : 256;
  const double units = double(n_kv_head) * (double(total_q) * group / 8 + 0.5 * batch);
  const int64_t ctas = int64_t(batch) * n_kv_head * ((int64_t(max_seqlen_q) * group + block - 1) / block);
  return double((ctas + sms - 1) / sms) * WAVE_UNITS < units / sms;
}

int attend_common(const void* q, int64_t total_q, int64_t q_st, int64_t q_sh, const void* pages, int64_t n_blocks, int32_t block_size,
                  const float* units, const int32_t* block_table, int64_t bt_stride, int32_t max_blocks,
                  const int32_t* cu_q, int32_t max_seqlen_q, const int32_t* seqlen, void* out, int64_t o_st,
                  int64_t o_sh, int32_t batch, int32_t n_head, int32_t n_kv_head, int32_t head_dim, int32_t dtype,
                  float scale_log2, void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_dtype(dtype) || n_head < 1 || n_kv_head < 1 || n_head % n_kv_head != 0) return PD_ERR_INVALID;
  if (batch < 0 || max_seqlen_q < 0 || max_blocks < 0 || total_q < 0 || total_q > 0x7fffffff) return PD_ERR_INVALID;
  if (dtype == PD_F32) return PD_ERR_UNSUPPORTED;
  int st = check_pool(pages, n_blocks, block_size, n_kv_head, head_dim);
  if (st != PD_OK) return st;
  if (max_blocks > 0 && bt_stride < max_blocks) return PD_ERR_INVALID;
  const int64_t capacity = int64_t(max_blocks) * block_size;
  if (capacity > (int64_t(1) << 30)) return PD_ERR_INVALID;
  // the kernels index query rows (a token's heads side by side) in 32 bits, up to a block of rows past the last
  if (total_q * n_head > (int64_t(1) << 30)) return PD_ERR_UNSUPPORTED;
  // no chunk is longer than the packed tensor: a loose bound neither changes the choice of the kernel nor
  // launches blocks past the last row
  max_seqlen_q = int32_t(max_seqlen_q < total_q ? max_seqlen_q : total_q);
  if (batch == 0 || max_seqlen_q == 0) return PD_OK;
  if (seqlen == nullptr || (block_table == nullptr && max_blocks > 0)) return PD_ERR_INVALID;
  if (q == nullptr || out == nullptr || !aligned(q, 16) || !aligned(out, 16)) return PD_ERR_INVALID;
  for (const int64_t s : {q_st, q_sh, o_st, o_sh})
    if ((s * 2) % 16 != 0) return PD_ERR_INVALID;
  int sms = 0;
  unsigned* err = nullptr;
  if (api_device(&sms, &err) != PD_OK) return PD_ERR_CUDA;
  if (workspace == nullptr || workspace_bytes < fp4_workspace_bytes(head_dim, sms))
    return api_message(PD_ERR_WORKSPACE, "workspace is smaller than pd_fp4_workspace_bytes");
  if (!aligned(workspace, 256)) return api_message(PD_ERR_WORKSPACE, "workspace is not 256-byte aligned");
  Fp4AttendParams p{};
  p.total_q = int32_t(total_q);
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.pages = static_cast<const unsigned char*>(pages);
  p.n_blocks = n_blocks;
  p.units = units;
  p.bt_stride = bt_stride;
  p.max_seqlen_q = max_seqlen_q;
  p.max_blocks = max_blocks;
  p.capacity = int32_t(capacity);
  p.n_kv_head = n_kv_head;
  p.group = n_head / n_kv_head;
  p.log2_tpb = ilog2_host(block_size / FP4_TILE);
  p.scale_log2 = scale_log2;
  p.counters = static_cast<unsigned*>(workspace);
  p.partials = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + fp4_counter_bytes(sms));
  p.err = err;
  p.wait_ns = api_wait_limit_ns();
  const int mode = g_fp4_prefill_mode.load(std::memory_order_relaxed);
  const bool tiles = cu_q != nullptr && (mode == 2 || (mode == 0 && use_tiles(total_q, max_seqlen_q, batch, n_kv_head,
                                                                             p.group, head_dim, sms)));
  for (int b0 = 0; b0 < batch; b0 += fp4_max_rows()) {
    p.batch = batch - b0 < fp4_max_rows() ? batch - b0 : fp4_max_rows();
    // a chunk's offsets are absolute, a decode step's row b is q row b
    const int64_t at = cu_q != nullptr ? 0 : b0;
    p.q = static_cast<const unsigned char*>(q) + at * q_st * 2;
    p.out = static_cast<unsigned char*>(out) + at * o_st * 2;
    p.cu_q = cu_q != nullptr ? cu_q + b0 : nullptr;
    p.seqlen = seqlen + b0;
    p.table = block_table != nullptr ? block_table + int64_t(b0) * bt_stride : nullptr;
    const cudaStream_t on = static_cast<cudaStream_t>(stream);
    st = launched(tiles ? launch_fp4_prefill(p, dtype, head_dim, on) : launch_fp4_attend(p, dtype, head_dim, sms, on),
                  "4-bit attention launch");
    if (st != PD_OK) return st;
  }
  return PD_OK;
}

}  // namespace
}  // namespace pd

using namespace pd;

extern "C" {

int pd_qk_norm_rope(const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, void* q_out,
                    int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh, const void* q_weight,
                    const void* k_weight, const void* rope_cos, const void* rope_sin, int64_t cos_stride,
                    int64_t sin_stride, int64_t n_pos, const void* positions, int32_t pos_dtype, int64_t n_tokens,
                    int32_t n_head, int32_t n_kv_head, int32_t head_dim, int32_t rotary_dim, float eps, int32_t dtype,
                    void* stream) {
  if (!valid_dtype(dtype) || n_head < 1 || n_kv_head < 1 || n_tokens < 0 || n_pos < 0) return PD_ERR_INVALID;
  if (pos_dtype != PD_SLOT_I32 && pos_dtype != PD_SLOT_I64) return PD_ERR_INVALID;
  if (head_dim < 2 || rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim) return PD_ERR_INVALID;
  if (head_dim > 256) return PD_ERR_UNSUPPORTED;
  if (n_tokens == 0) return PD_OK;
  if (q == nullptr || k == nullptr || q_out == nullptr || k_out == nullptr || q_weight == nullptr ||
      k_weight == nullptr || (rotary_dim > 0 && (rope_cos == nullptr || rope_sin == nullptr)))
    return PD_ERR_INVALID;
  NormRopeParams p{};
  int sms = 0;
  if (api_device(&sms, &p.err) != PD_OK) return PD_ERR_CUDA;
  p.q = q;
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.k = k;
  p.k_st = k_st;
  p.k_sh = k_sh;
  p.q_out = q_out;
  p.qo_st = qo_st;
  p.qo_sh = qo_sh;
  p.k_out = k_out;
  p.ko_st = ko_st;
  p.ko_sh = ko_sh;
  p.wq = q_weight;
  p.wk = k_weight;
  p.cos = rope_cos;
  p.sin = rope_sin;
  p.cos_st = cos_stride;
  p.sin_st = sin_stride;
  p.n_pos = n_pos;
  p.pos = positions;
  p.pos_i64 = pos_dtype == PD_SLOT_I64;
  p.n_tokens = n_tokens;
  p.n_head = n_head;
  p.n_kv_head = n_kv_head;
  p.head_dim = head_dim;
  p.rotary_dim = rotary_dim;
  p.eps = eps;
  // The vector kernel loads 4 elements at a time: 8 bytes of 16-bit types, 16 of fp32.
  const unsigned n = unsigned(4 * elem_size(dtype));
  bool vec = (head_dim == 64 || head_dim == 128 || head_dim == 256) && rotary_dim % 8 == 0 &&
             cos_stride % 4 == 0 && sin_stride % 4 == 0;
  for (const void* a : {q, k, static_cast<const void*>(q_out), static_cast<const void*>(k_out), q_weight, k_weight,
                        rope_cos, rope_sin})
    vec = vec && aligned(a, n);
  for (const int64_t s : {q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh}) vec = vec && s % 4 == 0;
  return launched(launch_norm_rope(p, dtype, vec, sms, static_cast<cudaStream_t>(stream)), "norm and rotation launch");
}

int pd_fp4_write_slots(void* pages, int64_t n_blocks, int32_t block_size, const void* slot_ids, int32_t slot_dtype,
                       const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                       const float* units, int32_t src_dtype, int64_t n_tokens, int32_t n_kv_head, int32_t head_dim,
                       void* stream) {
  if (slot_dtype != PD_SLOT_I32 && slot_dtype != PD_SLOT_I64) return PD_ERR_INVALID;
  if (slot_ids == nullptr && n_tokens > 0) return PD_ERR_INVALID;
  Fp4RowsParams p{};
  p.pages = static_cast<unsigned char*>(pages);
  p.n_blocks = n_blocks;
  p.block_size = block_size;
  p.n_kv_head = n_kv_head;
  p.head_dim = head_dim;
  p.units = units;
  p.slots = slot_ids;
  p.slot_i64 = slot_dtype == PD_SLOT_I64;
  p.k = const_cast<void*>(k);
  p.v = const_cast<void*>(v);
  p.n_tokens = n_tokens;
  return rows_common(p, src_dtype, false, k_strides, v_strides, stream);
}

int pd_fp4_write_table(void* pages, int64_t n_blocks, int32_t block_size, const int32_t* block_table,
                       int64_t bt_stride, int32_t max_blocks, const int64_t* pos, const void* k,
                       const int64_t* k_strides, const void* v, const int64_t* v_strides, const float* units,
                       int32_t src_dtype, int32_t batch, int32_t n_kv_head, int32_t head_dim, void* stream) {
  if (batch > 0 && (block_table == nullptr || pos == nullptr || max_blocks < 1)) return PD_ERR_INVALID;
  Fp4RowsParams p{};
  p.pages = static_cast<unsigned char*>(pages);
  p.n_blocks = n_blocks;
  p.block_size = block_size;
  p.n_kv_head = n_kv_head;
  p.head_dim = head_dim;
  p.units = units;
  p.table = block_table;
  p.bt_stride = bt_stride;
  p.max_blocks = max_blocks;
  p.pos = pos;
  p.k = const_cast<void*>(k);
  p.v = const_cast<void*>(v);
  p.n_tokens = batch;
  return rows_common(p, src_dtype, false, k_strides, v_strides, stream);
}

int pd_fp4_read_slots(const void* pages, int64_t n_blocks, int32_t block_size, const void* slot_ids,
                      int32_t slot_dtype, void* k, const int64_t* k_strides, void* v, const int64_t* v_strides,
                      const float* units, int32_t dst_dtype, int64_t n_tokens, int32_t n_kv_head, int32_t head_dim,
                      void* stream) {
  if (slot_dtype != PD_SLOT_I32 && slot_dtype != PD_SLOT_I64) return PD_ERR_INVALID;
  if (slot_ids == nullptr && n_tokens > 0) return PD_ERR_INVALID;
  Fp4RowsParams p{};
  p.pages = static_cast<unsigned char*>(const_cast<void*>(pages));
  p.n_blocks = n_blocks;
  p.block_size = block_size;
  p.n_kv_head = n_kv_head;
  p.head_dim = head_dim;
  p.units = units;
  p.slots = slot_ids;
  p.slot_i64 = slot_dtype == PD_SLOT_I64;
  p.k = k;
  p.v = v;
  p.n_tokens = n_tokens;
  return rows_common(p, dst_dtype, true, k_strides, v_strides, stream);
}

size_t pd_fp4_workspace_bytes(int32_t head_dim) {
  int sms = 0;
  unsigned* err = nullptr;
  if (!fp4_head_dim(head_dim) || api_device(&sms, &err) != PD_OK) return 0;
  return fp4_workspace_bytes(head_dim, sms);
}

int pd_fp4_decode(const void* q, int64_t q_sb, int64_t q_sh, const void* pages, int64_t n_blocks, int32_t block_size,
                  const float* units, const int32_t* block_table, int64_t bt_stride, int32_t max_blocks,
                  const int32_t* seqlen, void* out, int64_t o_sb, int64_t o_sh, int32_t batch, int32_t n_head,
                  int32_t n_kv_head, int32_t head_dim, int32_t dtype, float scale_log2, void* workspace,
                  size_t workspace_bytes, void* stream) {
  return attend_common(q, batch, q_sb, q_sh, pages, n_blocks, block_size, units, block_table, bt_stride, max_blocks, nullptr,
                       1, seqlen, out, o_sb, o_sh, batch, n_head, n_kv_head, head_dim, dtype, scale_log2, workspace,
                       workspace_bytes, stream);
}

int pd_fp4_prefill(const void* q, int64_t total_q, int64_t q_st, int64_t q_sh, const void* pages, int64_t n_blocks, int32_t block_size,
                   const float* units, const int32_t* block_table, int64_t bt_stride, int32_t max_blocks,
                   const int32_t* cu_seqlens_q, const int32_t* seqlen_k, void* out, int64_t o_st, int64_t o_sh,
                   int32_t batch, int32_t max_seqlen_q, int32_t n_head, int32_t n_kv_head, int32_t head_dim,
                   int32_t dtype, float scale_log2, void* workspace, size_t workspace_bytes, void* stream) {
  if (batch > 0 && max_seqlen_q > 0 && cu_seqlens_q == nullptr) return PD_ERR_INVALID;
  return attend_common(q, total_q, q_st, q_sh, pages, n_blocks, block_size, units, block_table, bt_stride, max_blocks,
                       cu_seqlens_q, max_seqlen_q, seqlen_k, out, o_st, o_sh, batch, n_head, n_kv_head, head_dim,
                       dtype, scale_log2, workspace, workspace_bytes, stream);
}

int pd_set_fp4_prefill_mode(int32_t mode) {
  if (mode < 0 || mode > 2) return PD_ERR_INVALID;
  g_fp4_prefill_mode.store(mode, std::memory_order_relaxed);
  return PD_OK;
}

int pd_get_fp4_prefill_mode(void) { return g_fp4_prefill_mode.load(std::memory_order_relaxed); }

size_t pd_evict_scratch_bytes(int32_t n_layer, int32_t batch, int32_t n_kv_head, int32_t keep) {
  if (n_layer < 0 || batch < 0 || n_kv_head < 1 || keep < 1) return 0;
  const size_t items = size_t(n_layer) * batch * n_kv_head;
  return items * 8 + items * size_t(keep) * 4;
}

int pd_evict(void* const* k_caches, void* const* v_caches, int32_t n_layer, int64_t n_blocks, int32_t block_size,
             int32_t n_kv_head, int32_t head_dim, int32_t dtype, const int64_t* k_strides, const int64_t* v_strides,
             const int32_t* block_table, int64_t bt_stride, int32_t max_blocks, const int32_t* new_table,
             int64_t nbt_stride, int32_t new_max_blocks, const int32_t* seqlen, int32_t* seqlen_out,
             const float* weights, const int64_t* w_strides, float* weights_out, const int64_t* wo_strides,
             int64_t w_len, int32_t batch, int32_t keep, int32_t recent, int32_t sinks, void* scratch,
             size_t scratch_bytes, void* stream) {
  if (!valid_dtype(dtype) || n_layer < 0 || n_blocks < 1 || n_kv_head < 1 || head_dim < 1 || !pow2(block_size))
    return PD_ERR_INVALID;
  if (batch < 0 || max_blocks < 0 || new_max_blocks < 0 || keep < 1 || recent < 0 || sinks < 0) return PD_ERR_INVALID;
  if (int64_t(recent) + sinks > keep) return PD_ERR_INVALID;
  const int64_t capacity = int64_t(max_blocks) * block_size;
  if (capacity > (int64_t(1) << 30) || int64_t(new_max_blocks) * block_size > (int64_t(1) << 30)) return PD_ERR_INVALID;
  if (w_len < capacity || bt_stride < max_blocks) return PD_ERR_INVALID;
  const int es = elem_size(dtype);
  if (head_dim > EVICT_UNITS * 16 / es || head_dim * es % 16 != 0) return PD_ERR_UNSUPPORTED;
  if (n_layer == 0 || batch == 0) return PD_OK;
  if (k_caches == nullptr || v_caches == nullptr || k_strides == nullptr || v_strides == nullptr ||
      w_strides == nullptr || wo_strides == nullptr || seqlen == nullptr || seqlen_out == nullptr ||
      (max_blocks > 0 && (block_table == nullptr || weights == nullptr)) || (w_len > 0 && weights_out == nullptr))
    return PD_ERR_INVALID;
  // What the kept tokens need of the new pages.
  if (new_table != nullptr &&
      (nbt_stride < new_max_blocks || int64_t(new_max_blocks) * block_size < (keep < capacity ? keep : capacity)))
    return PD_ERR_INVALID;
  // A row's own pages as its new ones: rows moved to new pages are moved by several CTAs in any order, which would read
  // what others have written. (Equal block ids elsewhere in the tables are on the device.)
  if (new_table != nullptr) {
    const int64_t apart = (reinterpret_cast<intptr_t>(new_table) - reinterpret_cast<intptr_t>(block_table)) / 4;
    for (int64_t b = 0; b < (nbt_stride == bt_stride ? 1 : batch); ++b) {
      const int64_t at = apart + b * (nbt_stride - bt_stride);
      if (at < max_blocks && at > -int64_t(new_max_blocks))
        return api_message(PD_ERR_INVALID, "new_table is a row's own block_table (NULL evicts in place)");
    }
  }
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] * es % 16 != 0 || v_strides[i] * es % 16 != 0) return PD_ERR_INVALID;
  for (int i = 0; i < n_layer; ++i)
    if (k_caches[i] == nullptr || v_caches[i] == nullptr || !aligned(k_caches[i], 16) || !aligned(v_caches[i], 16))
      return PD_ERR_INVALID;
  std::vector<const void*> pools;
  try {
    pools.reserve(2 * size_t(n_layer));
  } catch (const std::exception&) {
    return api_message(PD_ERR_INVALID, "no host memory for that many layers");
  }
  pools.insert(pools.end(), k_caches, k_caches + n_layer);
  pools.insert(pools.end(), v_caches, v_caches + n_layer);
  std::sort(pools.begin(), pools.end());
  if (std::adjacent_find(pools.begin(), pools.end()) != pools.end())
    return api_message(PD_ERR_INVALID, "a pool is named twice, and its tokens would be moved twice");
  // no row holds more than its table: a larger budget evicts nothing either
  keep = int32_t(keep < capacity + 1 ? keep : capacity + 1);
  if (recent + sinks > keep) recent = sinks = 0;
  const int64_t items = int64_t(batch) * n_kv_head;
  if (items > 0x7fffffff / (2 * EVICT_LAYERS * 128)) return PD_ERR_UNSUPPORTED;  // CTAs of a launch
  if (scratch == nullptr || !aligned(scratch, 16) || scratch_bytes < pd_evict_scratch_bytes(n_layer, batch, n_kv_head, keep))
    return api_message(PD_ERR_WORKSPACE, "scratch is smaller than pd_evict_scratch_bytes");
  EvictParams p{};
  if (api_device(&p.sms, &p.err) != PD_OK) return PD_ERR_CUDA;
  p.k_sb = k_strides[0] * es / 16;
  p.k_sn = k_strides[1] * es / 16;
  p.k_sh = k_strides[2] * es / 16;
  p.v_sb = v_strides[0] * es / 16;
  p.v_sn = v_strides[1] * es / 16;
  p.v_sh = v_strides[2] * es / 16;
  p.n_blocks = n_blocks;
  p.table = block_table;
  p.bt_stride = bt_stride;
  p.fresh = new_table != nullptr;
  p.new_table = p.fresh ? new_table : block_table;
  p.nbt_stride = p.fresh ? nbt_stride : bt_stride;
  p.seqlen = seqlen;
  p.w_sl = w_strides[0];
  p.w_sb = w_strides[1];
  p.w_sh = w_strides[2];
  p.wo_sl = wo_strides[0];
  p.wo_sb = wo_strides[1];
  p.wo_sh = wo_strides[2];
  p.w_len = w_len;
  p.batch = batch;
  p.n_kv_head = n_kv_head;
  p.chunks = head_dim * es / 16;
  p.log2_bs = ilog2_host(block_size);
  p.max_blocks = max_blocks;
  p.new_max_blocks = p.fresh ? new_max_blocks : max_blocks;
  p.capacity = int32_t(capacity);
  p.keep = keep;
  p.recent = recent;
  p.sinks = sinks;
  int2* info = static_cast<int2*>(scratch);
  int32_t* order = reinterpret_cast<int32_t*>(info + n_layer * items);
  for (int l0 = 0; l0 < n_layer; l0 += EVICT_LAYERS) {
    p.layers = n_layer - l0 < EVICT_LAYERS ? n_layer - l0 : EVICT_LAYERS;
    for (int i = 0; i < p.layers; ++i) {
      p.k[i] = k_caches[l0 + i];
      p.v[i] = v_caches[l0 + i];
    }
    p.weights = weights + l0 * p.w_sl;
    p.weights_out = weights_out + l0 * p.wo_sl;
    p.info = info + l0 * items;
    p.order = order + l0 * items * keep;
    p.seqlen_out = l0 + p.layers == n_layer ? seqlen_out : nullptr;  // every launch reads the old lengths
    const int st = launched(launch_evict(p, static_cast<cudaStream_t>(stream)), "eviction launch");
    if (st != PD_OK) return st;
    api_count_launch();  // two kernels
  }
  return PD_OK;
}

int pd_block_copy(void* const* pools, int32_t n_pools, int64_t n_blocks, int64_t block_bytes, const void* src,
                  const void* dst, int32_t id_dtype, int64_t n_pairs, int32_t* block_table, int64_t table_rows,
                  int64_t table_cols, int64_t bt_stride, const int32_t* remap, void* stream) {
  if (n_pools < 0 || n_blocks < 1 || block_bytes < 1 || n_pairs < 0) return PD_ERR_INVALID;
  if (id_dtype != PD_SLOT_I32 && id_dtype != PD_SLOT_I64) return PD_ERR_INVALID;
  if (n_pools > 0 && n_pairs > 0 && (pools == nullptr || src == nullptr || dst == nullptr)) return PD_ERR_INVALID;
  if (block_table != nullptr && (remap == nullptr || table_rows < 0 || table_cols < 0 || bt_stride < table_cols))
    return PD_ERR_INVALID;
  for (int i = 0; i < n_pools; ++i)
    if (n_pairs > 0 && pools[i] == nullptr) return PD_ERR_INVALID;
  BlockCopyParams p{};
  int sms = 0;
  if (api_device(&sms, &p.err) != PD_OK) return PD_ERR_CUDA;
  p.ids_i64 = id_dtype == PD_SLOT_I64;
  p.n_blocks = n_blocks;
  p.block_bytes = block_bytes;
  p.src = src;
  p.dst = dst;
  p.n_pairs = n_pairs;
  p.remap = remap;
  int at = 0;
  bool table_done = block_table == nullptr || table_rows * table_cols == 0;
  do {  // pools in launches of COPY_MAX_POOLS; the tables with the first
    p.n_pools = 0;
    p.vec16 = block_bytes % 16 == 0;
    for (; n_pairs > 0 && at < n_pools && p.n_pools < COPY_MAX_POOLS; ++at) {
      p.pools[p.n_pools++] = static_cast<unsigned char*>(pools[at]);
      p.vec16 = p.vec16 && aligned(pools[at], 16);
    }
    p.table = table_done ? nullptr : block_table;
    p.table_rows = table_rows;
    p.table_cols = table_cols;
    p.table_st = bt_stride;
    table_done = true;
    if (p.n_pools == 0 && p.table == nullptr) break;
    const int st = launched(launch_block_copy(p, sms, static_cast<cudaStream_t>(stream)), "page copy launch");
    if (st != PD_OK) return st;
  } while (n_pairs > 0 && at < n_pools);
  return PD_OK;
}

}  // extern "C"
