// pd_fp4_rows.cu -- keys and values of tokens written into 4-bit pages and read back (sm_100a).
//
// Write: for each 16 neighbouring elements x of a K or V head row, in units u of the head,
//   scale = e4m3(max |x / u| / 6),  code_i = e2m1(x_i / u / scale),
// both to nearest with ties to even and both saturating; a group whose scale rounds to zero stores
// zeros, a NaN element counts as zero and infinities saturate. Read: x_i = code_i * scale * u,
// which is exact in fp32 and, for u = 1, in fp16 and bf16.
//
// Bound by memory: a token's rows are read once and 9/16 of a byte per element written. One thread
// handles one group of 16: its maximum and its eight code bytes are its own, so there is no
// exchange between threads; consecutive threads take consecutive groups of a row, so a warp reads
// 1 KB of 16-bit source in one run.
//
// The rounding is exact, not approximately so, which is what lets a reader compare pages bit for bit.
// For 16-bit sources x has at most 11 significant bits and scale * tie at most 7, so x / scale is
// either a tie exactly or at least 2^-11 (relative) away from it: the quotient is formed with an
// approximate reciprocal, rounded to 16 bits (which restores exact ties) and converted. fp32
// sources have no such gap: their codes come from comparing |x| with scale * tie, products that
// are exact. The scale's quotient is rounded to odd, so the second rounding to e4m3 sees on
// which side of a tie it lies.
#include "pd_fp4.cuh"
#include "pd_internal.h"

namespace pd {

namespace {

template <typename T>
__device__ __forceinline__ T from_f(float x) { return Elem<T>::from_float(x); }

// 16 consecutive elements as fp32. VEC: 16-byte aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load16(const T* p, float (&f)[16]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = Elem<T>::to_float(p[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 a = reinterpret_cast<const float4*>(p)[i];
      f[4 * i] = a.x; f[4 * i + 1] = a.y; f[4 * i + 2] = a.z; f[4 * i + 3] = a.w;
    }
  } else {
    Elem<T>::unpack(reinterpret_cast<const uint4*>(p)[0], f);
    Elem<T>::unpack(reinterpret_cast<const uint4*>(p)[1], f + 8);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store16(T* p, const float (&f)[16]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = from_f<T>(f[i]);
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
  } else {
    reinterpret_cast<uint4*>(p)[0] = Elem<T>::pack(f);
    reinterpret_cast<uint4*>(p)[1] = Elem<T>::pack(f + 8);
  }
}

// Block and offset of token i; false (and the error bit, once per token) outside the pool.
__device__ __forceinline__ bool locate(const Fp4RowsParams& p, int64_t i, bool first, int64_t& blk, int& off) {
  int64_t slot_off = 0;
  bool ok = true;
  if (p.table != nullptr) {
    const int64_t pos = p.pos[i];
    const int64_t page = pos >= 0 ? pos / p.block_size : -1;
    ok = page >= 0 && page < p.max_blocks;
    blk = ok ? p.table[i * p.bt_stride + page] : -1;
    slot_off = pos - page * p.block_size;
  } else {
    const int64_t slot = p.slot_i64 ? reinterpret_cast<const int64_t*>(p.slots)[i]
                                    : int64_t(reinterpret_cast<const int32_t*>(p.slots)[i]);
    blk = slot >= 0 ? slot / p.block_size : -1;
    slot_off = slot - blk * p.block_size;
  }
  if (blk < 0 || blk >= p.n_blocks) {
    if (first) atomicOr(p.err, DEVERR_APPEND_RANGE);
    return false;
  }
  off = int(slot_off);
  return true;
}

// The scale byte of a group with maximum m (in units), to nearest even.
__device__ __forceinline__ uint32_t scale_byte(float m) {
  m = fminf(m, 8192.f);  // past the saturation point 448 * 6
  const float q = __fdiv_rz(m, 6.f);
  const bool inexact = fmaf(-q, 6.f, m) != 0.f;
  return float_to_e4m3(__uint_as_float(__float_as_uint(q) | (inexact ? 1u : 0u)));
}

template <typename T>
__device__ __forceinline__ uint32_t code_byte(float a, float b, float s, float inv) {
  if constexpr (sizeof(T) == 2) {
    const auto snap = [](float x) { return __uint_as_float((__float_as_uint(x) + 0x80u) & ~0xffu); };
    return floats_to_e2m1x2(snap(a * inv), snap(b * inv));
  } else {
    const auto code = [s](float x) {
      const float m = fabsf(x);
      const int c = int(m > 0.25f * s) + int(m >= 0.75f * s) + int(m > 1.25f * s) + int(m >= 1.75f * s) +
                    int(m > 2.5f * s) + int(m >= 3.5f * s) + int(m > 5.f * s);
      return s > 0.f ? uint32_t(c) | (x < 0.f ? 8u : 0u) : 0u;
    };
    return code(a) | (code(b) << 4);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) pd_fp4_write_kernel(const Fp4RowsParams p) {
  const int groups = p.head_dim / FP4_GROUP;
  const int per_token = p.n_kv_head * groups;  // of K, and again of V
  const int64_t total = p.n_tokens * per_token * 2;
  const int rec = fp4_record_bytes(p.head_dim), tpb = p.block_size / FP4_TILE;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t t = i / (2 * per_token);
    const int rem = int(i - t * (2 * per_token));
    const bool is_v = rem >= per_token;
    const int r = is_v ? rem - per_token : rem;
    const int h = r / groups, gr = r - h * groups;
    int64_t blk;
    int off;
    if (!locate(p, t, rem == 0, blk, off)) continue;
    const T* src = (is_v ? reinterpret_cast<const T*>(p.v) + t * p.v_s0 + h * p.v_s1
                         : reinterpret_cast<const T*>(p.k) + t * p.k_s0 + h * p.k_s1) + gr * FP4_GROUP;
    float x[16];
    load16<T, VEC>(src, x);
    const float unit = p.units != nullptr ? p.units[(is_v ? p.n_kv_head : 0) + h] : 1.f;
    const float inv_unit = 1.f / unit;  // a power of two: exact
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      x[j] = x[j] == x[j] ? x[j] * inv_unit : 0.f;
      m = fmaxf(m, fabsf(x[j]));
    }
    const uint32_t sb = scale_byte(m);
    const float s = __half2float(__ushort_as_half(uint16_t(e4m3x2_to_half2(sb) & 0xffffu)));
    const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j >> 2] |= code_byte<T>(x[2 * j], x[2 * j + 1], s, inv) << (8 * (j & 3));
    const int tok = off % FP4_TILE;
    unsigned char* dst = p.pages + ((blk * p.n_kv_head + h) * tpb + off / FP4_TILE) * rec;
    *reinterpret_cast<uint2*>(dst + (is_v ? fp4_v_code(p.head_dim, tok, gr) : fp4_k_code(p.head_dim, tok, gr))) =
        make_uint2(w[0], w[1]);
    dst[is_v ? fp4_v_scale(p.head_dim, tok, gr) : fp4_k_scale(p.head_dim, tok, gr)] = static_cast<unsigned char>(sb);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) pd_fp4_read_kernel(const Fp4RowsParams p) {
  const int groups = p.head_dim / FP4_GROUP;
  const int per_token = p.n_kv_head * groups;
  const int64_t total = p.n_tokens * per_token * 2;
  const int rec = fp4_record_bytes(p.head_dim), tpb = p.block_size / FP4_TILE;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t t = i / (2 * per_token);
    const int rem = int(i - t * (2 * per_token));
    const bool is_v = rem >= per_token;
    const int r = is_v ? rem - per_token : rem;
    const int h = r / groups, gr = r - h * groups;
    int64_t blk;
    int off;
    float x[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.f;
    if (locate(p, t, rem == 0, blk, off)) {  // a slot outside the pool reads zeros
      const int tok = off % FP4_TILE;
      const unsigned char* src = p.pages + ((blk * p.n_kv_head + h) * tpb + off / FP4_TILE) * rec;
      const uint2 w = *reinterpret_cast<const uint2*>(
          src + (is_v ? fp4_v_code(p.head_dim, tok, gr) : fp4_k_code(p.head_dim, tok, gr)));
      const uint32_t sb = src[is_v ? fp4_v_scale(p.head_dim, tok, gr) : fp4_k_scale(p.head_dim, tok, gr)];
      const float unit = p.units != nullptr ? p.units[(is_v ? p.n_kv_head : 0) + h] : 1.f;
      const float s = __half2float(__ushort_as_half(uint16_t(e4m3x2_to_half2(sb) & 0xffffu))) * unit;
      uint32_t c[8];
      e2m1x8_to_half2x4(w.x, *reinterpret_cast<uint32_t(*)[4]>(c));
      e2m1x8_to_half2x4(w.y, *reinterpret_cast<uint32_t(*)[4]>(c + 4));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&c[j]));
        x[2 * j] = f.x * s;
        x[2 * j + 1] = f.y * s;
      }
    }
    T* dst = (is_v ? reinterpret_cast<T*>(p.v) + t * p.v_s0 + h * p.v_s1
                   : reinterpret_cast<T*>(p.k) + t * p.k_s0 + h * p.k_s1) + gr * FP4_GROUP;
    store16<T, VEC>(dst, x);
  }
}

template <typename T>
cudaError_t launch_typed(const Fp4RowsParams& p, bool read, bool vec, int sms, cudaStream_t stream) {
  const int64_t total = p.n_tokens * p.n_kv_head * (p.head_dim / FP4_GROUP) * 2;
  const int threads = 256;
  int64_t blocks = (total + threads - 1) / threads;
  if (blocks > int64_t(sms) * 32) blocks = int64_t(sms) * 32;
  if (read && vec)
    pd_fp4_read_kernel<T, true><<<unsigned(blocks), threads, 0, stream>>>(p);
  else if (read)
    pd_fp4_read_kernel<T, false><<<unsigned(blocks), threads, 0, stream>>>(p);
  else if (vec)
    pd_fp4_write_kernel<T, true><<<unsigned(blocks), threads, 0, stream>>>(p);
  else
    pd_fp4_write_kernel<T, false><<<unsigned(blocks), threads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp4_rows(const Fp4RowsParams& p, int dtype, bool read, bool vec, int sms, cudaStream_t stream) {
  switch (dtype) {
    case 0: return launch_typed<float>(p, read, vec, sms, stream);
    case 1: return launch_typed<__half>(p, read, vec, sms, stream);
    case 2: return launch_typed<__nv_bfloat16>(p, read, vec, sms, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace pd
