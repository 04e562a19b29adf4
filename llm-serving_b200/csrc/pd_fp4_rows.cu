// pd_fp4_rows.cu -- keys and values of tokens written into 4-bit pages and read back (sm_100a).
//
// Write: for each 16 neighbouring elements x of a K or V head row, in units u of the head,
//   scale = e4m3(max |x / u| / 6),  code_i = e2m1(x_i / u / scale),
// both to nearest with ties to even and both saturating; a group whose scale rounds to zero stores
// zeros, a NaN element counts as zero and infinities saturate. Read: x_i = code_i * scale * u,
// which is exact in fp32 and, for u = 1, in fp16 and bf16.
//
// Bound by memory in bytes (a token's rows are read once and 9/16 of a byte per element written),
// in practice by instructions and latency: 16 elements are 41 bytes of traffic, so at the copy rate an SM has
// some 180 issue slots a warp's 512 elements; the write takes 193 and issues in 57 % of its active cycles
// (half of the warps fit: 45 registers, and most wait on their source), the read 155 in 41 %, held up by its
// loads of 8 bytes and of one. One thread handles one group of 16: its maximum and its
// eight code bytes are its own, so there is no exchange between threads; consecutive threads
// take consecutive groups of a row, so a warp reads 1 KB of 16-bit source in one run.
//
// Measured: 7001 bf16 tokens of 8 heads of 128 written into scattered slots and read back, two
// launches, 74 MB, 21.9 us (3.4 TB/s), apart 9.2 and 11.2; into slots in order 9.1 and 10.4. fp32 rows, whose
// codes come from comparisons, 22.8 and 19.3. 32 tokens 4.2 us for the two (fp32 6.1). A token is 8 or 64 bytes at a
// time of a record, so scattered writes meet each 32-byte sector of V several times in L2; tokens of one
// record written together do not.
//
// The rounding is exact, not approximately so, which is what lets a reader compare bit for bit what pages
// stand for. (Their bytes may differ in the sign of a zero code: a negative element below 2^-17 of a code
// step becomes +0 from 16 bits and -0 from fp32.) A 16-bit x has at most 11 significant bits and scale * tie at most 7, so x / scale is either a tie
// exactly or at least 2^-11 (relative) away from it: fma(x, 1 / scale, 192) - 192 rounds the quotient
// (which the reciprocal's 2 ulp leave within 2^-20) to a multiple of 2^-16, which restores exact ties and moves nothing across one, and the
// hardware conversion then rounds it to a code. fp32 sources have no such gap: their codes come
// from comparing |x| with scale * tie, products that are exact. The maximum / 6 goes to e4m3 the
// same two ways: rounded to 16 bits first, or (fp32) divided toward zero with the remainder kept in
// the last bit, so that the second rounding sees on which side of a tie it lies.
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
  const int log2_bs = __ffs(p.block_size) - 1;
  if (p.table != nullptr) {
    const int64_t pos = p.pos[i], page = pos >> log2_bs;
    blk = pos >= 0 && page < p.max_blocks ? p.table[i * p.bt_stride + page] : -1;
    off = int(pos & (p.block_size - 1));
  } else {
    const int64_t slot = p.slot_i64 ? reinterpret_cast<const int64_t*>(p.slots)[i]
                                    : int64_t(reinterpret_cast<const int32_t*>(p.slots)[i]);
    blk = slot >> log2_bs;
    off = int(slot & (p.block_size - 1));
  }
  if (blk < 0 || blk >= p.n_blocks) {
    if (first) atomicOr(p.err, DEVERR_APPEND_RANGE);
    return false;
  }
  return true;
}

// max |x| of a pair and a running pair of maxima, NaN if either holds one.
__device__ __forceinline__ uint32_t max_abs(uint32_t m, uint32_t x, __half) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&m), __habs2(*reinterpret_cast<const __half2*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max_abs(uint32_t m, uint32_t x, __nv_bfloat16) {
  const __nv_bfloat162 r =
      __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&m), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The scale byte of a group with maximum m (in units), to nearest even.
template <typename T>
__device__ __forceinline__ uint32_t scale_byte(float m) {
  m = fminf(m, 8192.f);  // past the saturation point 448 * 6
  if constexpr (sizeof(T) == 2) {
    const uint32_t q = __float_as_uint(m * (1.f / 6.f));
    return float_to_e4m3(__uint_as_float((q + 0x80u) & ~0xffu));
  } else {
    const float q = __fdiv_rz(m, 6.f);
    const bool inexact = fmaf(-q, 6.f, m) != 0.f;
    return float_to_e4m3(__uint_as_float(__float_as_uint(q) | (inexact ? 1u : 0u)));
  }
}

__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
  return __half2float(__ushort_as_half(uint16_t(e4m3x2_to_half2(byte) & 0xffffu)));
}

// 16 elements (in `inv_unit`s) -> their codes and scale byte.
template <typename T>
__device__ __forceinline__ void quantise(float (&x)[16], float m, float inv_unit, uint32_t (&w)[2], uint32_t& sb) {
  m *= inv_unit;  // a power of two: exact
  sb = scale_byte<T>(m);
  const float s = e4m3_to_float(sb);
  w[0] = w[1] = 0u;
  if constexpr (sizeof(T) == 2) {
    const float inv = s > 0.f ? __fdividef(inv_unit, s) : 0.f;  // 2 ulp
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = fmaf(x[j], inv, 192.f) - 192.f;
    w[0] = floats_to_e2m1x8(x);
    w[1] = floats_to_e2m1x8(x + 8);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float a = x[j] * inv_unit, y = fabsf(a);
      const int c = int(y > 0.25f * s) + int(y >= 0.75f * s) + int(y > 1.25f * s) + int(y >= 1.75f * s) +
                    int(y > 2.5f * s) + int(y >= 3.5f * s) + int(y > 5.f * s);
      if (s > 0.f) w[j >> 3] |= (uint32_t(c) | (a < 0.f ? 8u : 0u)) << (4 * (j & 7));
    }
  }
}

// Where thread i of the grid works: a token, a head and a group of 16 elements of its K and of its V.
// head_dim is a compile-time constant, so a record's offsets are a few shifts, and K and V share
// the slot's look-up: written with run-time divisions and apart, addresses cost more than the
// rounding.
struct Place {
  int64_t token;
  bool first;
  int h, gr;
};

template <int D>
__device__ __forceinline__ Place place_of(const Fp4RowsParams& p, int64_t i) {
  constexpr int GROUPS = D / FP4_GROUP;
  const uint32_t per_token = uint32_t(p.n_kv_head) * GROUPS;
  Place at;
  uint32_t rem;
  if (i < 0xffffffffll) {
    const uint32_t t = uint32_t(i) / per_token;
    rem = uint32_t(i) - t * per_token;
    at.token = t;
  } else {
    at.token = i / per_token;
    rem = uint32_t(i - at.token * per_token);
  }
  at.first = rem == 0;
  at.h = int(rem / GROUPS);
  at.gr = int(rem % GROUPS);
  return at;
}

// 1 / unit and the unit itself: powers of two, so the reciprocal is a subtraction of exponents.
__device__ __forceinline__ float unit_of(const Fp4RowsParams& p, bool is_v, int h) {
  return p.units != nullptr ? __ldg(p.units + (is_v ? p.n_kv_head : 0) + h) : 1.f;
}
__device__ __forceinline__ float reciprocal_of_power(float unit) {
  return __uint_as_float(0x7f000000u - __float_as_uint(unit));
}

// A group of 16 elements as it is in memory, so that every load of a thread can be under way before
// the first is looked at.
template <typename T, bool VEC>
struct Group {
  static constexpr bool PAIRS = VEC && sizeof(T) == 2;
  uint4 r[PAIRS ? 2 : 1];
  float f[PAIRS ? 1 : 16];

  __device__ __forceinline__ void load(const T* src) {
    if constexpr (PAIRS) {
      r[0] = __ldcs(reinterpret_cast<const uint4*>(src));
      r[1] = __ldcs(reinterpret_cast<const uint4*>(src) + 1);
    } else {
      load16<T, VEC>(src, f);
    }
  }

  // The elements, NaN replaced by zero; returns their largest absolute value.
  __device__ __forceinline__ float unpack(float (&x)[16]) const {
    if constexpr (PAIRS) {
      const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
      uint32_t top = 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max_abs(top, w[j], T{});
      Elem<T>::unpack(r[0], x);
      Elem<T>::unpack(r[1], x + 8);
      float m[2];
      Elem<T>::unpack2(max_abs(top, __byte_perm(top, 0, 0x1032), T{}), m);
      if (m[0] == m[0]) return m[0];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = f[j];
    }
    float m = 0.f;  // a NaN among them, or a source that is not read in pairs
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      x[j] = x[j] == x[j] ? x[j] : 0.f;
      m = fmaxf(m, fabsf(x[j]));
    }
    return m;
  }
};

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(128) pd_fp4_write_kernel(const Fp4RowsParams p) {
  const int64_t total = p.n_tokens * p.n_kv_head * (D / FP4_GROUP);
  constexpr int REC = fp4_record_bytes(D);
  const int log2_tpb = __ffs(p.block_size) - 5;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const Place a = place_of<D>(p, i);
    Group<T, VEC> raw[2];
    raw[0].load(reinterpret_cast<const T*>(p.k) + a.token * p.k_s0 + a.h * p.k_s1 + a.gr * FP4_GROUP);
    raw[1].load(reinterpret_cast<const T*>(p.v) + a.token * p.v_s0 + a.h * p.v_s1 + a.gr * FP4_GROUP);
    int64_t blk;
    int off;
    if (!locate(p, a.token, a.first, blk, off)) continue;
    const int tok = off % FP4_TILE;
    unsigned char* dst = p.pages + (((blk * p.n_kv_head + a.h) << log2_tpb) + off / FP4_TILE) * REC;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float x[16];
      const float m = raw[kv].unpack(x);
      uint32_t w[2], sb;
      quantise<T>(x, m, reciprocal_of_power(unit_of(p, kv, a.h)), w, sb);
      *reinterpret_cast<uint2*>(dst + (kv ? fp4_v_code(D, tok, a.gr) : fp4_k_code(D, tok, a.gr))) = make_uint2(w[0], w[1]);
      dst[kv ? fp4_v_scale(D, tok, a.gr) : fp4_k_scale(D, tok, a.gr)] = static_cast<unsigned char>(sb);
    }
  }
}

template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(128) pd_fp4_read_kernel(const Fp4RowsParams p) {
  const int64_t total = p.n_tokens * p.n_kv_head * (D / FP4_GROUP);
  constexpr int REC = fp4_record_bytes(D);
  const int log2_tpb = __ffs(p.block_size) - 5;
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const Place a = place_of<D>(p, i);
    int64_t blk;
    int off;
    const bool inside = locate(p, a.token, a.first, blk, off);  // a slot outside the pool reads zeros
    uint2 w[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
    uint32_t sb[2] = {0u, 0u};
    if (inside) {
      const int tok = off % FP4_TILE;
      const unsigned char* src = p.pages + (((blk * p.n_kv_head + a.h) << log2_tpb) + off / FP4_TILE) * REC;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        w[kv] = __ldg(reinterpret_cast<const uint2*>(src + (kv ? fp4_v_code(D, tok, a.gr) : fp4_k_code(D, tok, a.gr))));
        sb[kv] = __ldg(src + (kv ? fp4_v_scale(D, tok, a.gr) : fp4_k_scale(D, tok, a.gr)));
      }
    }
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const float s = e4m3_to_float(sb[kv]) * unit_of(p, kv, a.h);
      uint32_t c[8];
      e2m1x8_to_half2x4(w[kv].x, *reinterpret_cast<uint32_t(*)[4]>(c));
      e2m1x8_to_half2x4(w[kv].y, *reinterpret_cast<uint32_t(*)[4]>(c + 4));
      float x[16];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&c[j]));
        x[2 * j] = f.x * s;
        x[2 * j + 1] = f.y * s;
      }
      T* dst = kv ? reinterpret_cast<T*>(p.v) + a.token * p.v_s0 + a.h * p.v_s1
                  : reinterpret_cast<T*>(p.k) + a.token * p.k_s0 + a.h * p.k_s1;
      store16<T, VEC>(dst + a.gr * FP4_GROUP, x);
    }
  }
}

template <typename T, int D>
cudaError_t launch_dim(const Fp4RowsParams& p, bool read, bool vec, int sms, cudaStream_t stream) {
  const int64_t total = p.n_tokens * p.n_kv_head * (D / FP4_GROUP);
  const int threads = 128;
  int64_t blocks = (total + threads - 1) / threads;
  if (blocks > int64_t(sms) * 64) blocks = int64_t(sms) * 64;
  if (read && vec)
    pd_fp4_read_kernel<T, D, true><<<unsigned(blocks), threads, 0, stream>>>(p);
  else if (read)
    pd_fp4_read_kernel<T, D, false><<<unsigned(blocks), threads, 0, stream>>>(p);
  else if (vec)
    pd_fp4_write_kernel<T, D, true><<<unsigned(blocks), threads, 0, stream>>>(p);
  else
    pd_fp4_write_kernel<T, D, false><<<unsigned(blocks), threads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const Fp4RowsParams& p, bool read, bool vec, int sms, cudaStream_t stream) {
  switch (p.head_dim) {
    case 64: return launch_dim<T, 64>(p, read, vec, sms, stream);
    case 128: return launch_dim<T, 128>(p, read, vec, sms, stream);
    case 256: return launch_dim<T, 256>(p, read, vec, sms, stream);
  }
  return cudaErrorInvalidValue;
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
