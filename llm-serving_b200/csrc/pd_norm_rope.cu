// pd_norm_rope.cu -- RMS norm of each query and key head and its rotary rotation in one pass
// (sm_100a).
//
// For a head row x of D elements with weight w, position p and rotary dimension R:
//   y = x * rsqrt(mean(x^2) + eps) * w
//   out[i] = y[i] cos[p, i] - y[i + R/2] sin[p, i],  out[i + R/2] = y[i] sin[p, i] + y[i + R/2] cos[p, i]
// for i < R / 2, the elements from R on passing through (the model's q_norm / k_norm and
// apply_rotary_emb_partial, model/layers.py:59-117 and 200-211). Everything between the load and
// the one rounding of the result is fp32.
//
// Bound by memory: every element is read and written once. A lane holds the two halves of its
// rotary pairs itself (4 elements at i and 4 at i + R/2), so the rotation needs no exchange and the
// norm one shuffle reduction over the D / 8 lanes of a head. A warp takes NORM_HEADS heads of one
// token per lane group and issues their loads together: the cos/sin row is read once for
// them, and a lane has 64 bytes in flight.
#include "pd_internal.h"
#include "pd_norm_rope.cuh"

namespace pd {

namespace {

constexpr int NORM_HEADS = 4;  // heads in flight per lane group

// 4 consecutive elements as fp32.
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&f)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  } else {
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    Elem<T>::unpack2(r.x, f);
    Elem<T>::unpack2(r.y, f + 2);
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&f)[4]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]));
  }
}

__device__ __forceinline__ int64_t position_of(const NormRopeParams& p, int64_t t) {
  if (p.pos == nullptr) return t;
  return p.pos_i64 ? reinterpret_cast<const int64_t*>(p.pos)[t]
                   : int64_t(reinterpret_cast<const int32_t*>(p.pos)[t]);
}

// LANES = D / 8 lanes per head (8, 16 or 32). Lane l of a head holds elements e0 .. e0 + 3 and
// e1 .. e1 + 3: a rotary pair block while 4 l < R / 2, two blocks of the passed-through rest after.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) pd_norm_rope_kernel(const NormRopeParams p) {
  constexpr int D = LANES * 8;
  constexpr int GROUPS = 32 / LANES;  // heads of a warp at once
  const int lane = threadIdx.x & 31;
  const int l = lane % LANES, grp = lane / LANES;
  const int heads = p.n_head + p.n_kv_head;
  const int per_warp = GROUPS * NORM_HEADS;
  const int chunks = (heads + per_warp - 1) / per_warp;
  const int64_t items = p.n_tokens * chunks;
  const int half = p.rotary_dim >> 1;
  const bool rot = 4 * l < half;
  const int e0 = rot ? 4 * l : p.rotary_dim + 8 * (l - half / 4);
  const int e1 = rot ? half + 4 * l : e0 + 4;
  for (int64_t it = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items;
       it += int64_t(gridDim.x) * (blockDim.x >> 5)) {
    const int64_t t = it / chunks;
    const int h0 = int(it - t * chunks) * per_warp + grp;
    float a[NORM_HEADS][4], b[NORM_HEADS][4];
#pragma unroll
    for (int j = 0; j < NORM_HEADS; ++j) {
      const int h = h0 + j * GROUPS;
      if (h < heads) {
        const T* x = h < p.n_head ? reinterpret_cast<const T*>(p.q) + t * p.q_st + h * p.q_sh
                                  : reinterpret_cast<const T*>(p.k) + t * p.k_st + (h - p.n_head) * p.k_sh;
        load4(x + e0, a[j]);
        load4(x + e1, b[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[j][i] = b[j][i] = 0.f;
      }
    }
    const int64_t pos = position_of(p, t);
    const bool in_range = pos >= 0 && pos < p.n_pos;
    float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
    if (rot && in_range) {
      load4(reinterpret_cast<const T*>(p.cos) + pos * p.cos_st + 4 * l, c);
      load4(reinterpret_cast<const T*>(p.sin) + pos * p.sin_st + 4 * l, s);
    }
    if (!in_range && lane == 0) atomicOr(p.err, DEVERR_ROPE_RANGE);
#pragma unroll
    for (int j = 0; j < NORM_HEADS; ++j) {
      const int h = h0 + j * GROUPS;
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = fmaf(a[j][i], a[j][i], fmaf(b[j][i], b[j][i], ss));
#pragma unroll
      for (int o = LANES / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, o);
      // 1 / sqrt rather than the approximate rsqrt: fp32 rows then keep fp32's accuracy
      const float inv = in_range ? 1.f / sqrtf(ss * (1.f / D) + p.eps) : 0.f;
      if (h >= heads) continue;
      const bool is_q = h < p.n_head;
      const T* w = reinterpret_cast<const T*>(is_q ? p.wq : p.wk);
      float wa[4], wb[4], oa[4], ob[4];
      load4(w + e0, wa);
      load4(w + e1, wb);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ya = a[j][i] * inv * wa[i], yb = b[j][i] * inv * wb[i];
        oa[i] = rot ? ya * c[i] - yb * s[i] : ya;
        ob[i] = rot ? ya * s[i] + yb * c[i] : yb;
      }
      T* y = is_q ? reinterpret_cast<T*>(p.q_out) + t * p.qo_st + h * p.qo_sh
                  : reinterpret_cast<T*>(p.k_out) + t * p.ko_st + (h - p.n_head) * p.ko_sh;
      store4(y + e0, oa);
      store4(y + e1, ob);
    }
  }
}

// Any even head_dim up to 256 and any alignment: one warp per head, one element at a time.
template <typename T>
__global__ void __launch_bounds__(256) pd_norm_rope_any_kernel(const NormRopeParams p) {
  using E = Elem<T>;
  const int lane = threadIdx.x & 31;
  const int heads = p.n_head + p.n_kv_head;
  const int64_t items = p.n_tokens * heads;
  const int half = p.rotary_dim >> 1, d = p.head_dim;
  for (int64_t it = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items;
       it += int64_t(gridDim.x) * (blockDim.x >> 5)) {
    const int64_t t = it / heads;
    const int h = int(it - t * heads);
    const bool is_q = h < p.n_head;
    const T* x = is_q ? reinterpret_cast<const T*>(p.q) + t * p.q_st + h * p.q_sh
                      : reinterpret_cast<const T*>(p.k) + t * p.k_st + (h - p.n_head) * p.k_sh;
    T* y = is_q ? reinterpret_cast<T*>(p.q_out) + t * p.qo_st + h * p.qo_sh
                : reinterpret_cast<T*>(p.k_out) + t * p.ko_st + (h - p.n_head) * p.ko_sh;
    const T* w = reinterpret_cast<const T*>(is_q ? p.wq : p.wk);
    // Element lane + 32 n for n < 8; its rotary partner is read from memory again, before any
    // store of this head (the rows may be normalised in place).
    float v[8], u[8];
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int e = lane + 32 * n;
      const bool live = e < d;
      v[n] = live ? E::to_float(x[e]) : 0.f;
      ss = fmaf(v[n], v[n], ss);
      const int partner = e < half ? e + half : e - half;
      u[n] = live && e < p.rotary_dim ? E::to_float(x[partner]) * E::to_float(w[partner]) : 0.f;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, o);
    const int64_t pos = position_of(p, t);
    const bool in_range = pos >= 0 && pos < p.n_pos;
    if (!in_range && lane == 0) atomicOr(p.err, DEVERR_ROPE_RANGE);
    const float inv = in_range ? 1.f / sqrtf(ss / float(d) + p.eps) : 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const int e = lane + 32 * n;
      if (e >= d) continue;
      const float own = v[n] * inv * E::to_float(w[e]);
      float r = own;
      if (e < p.rotary_dim && in_range) {
        const int i = e < half ? e : e - half;
        const float c = E::to_float(reinterpret_cast<const T*>(p.cos)[pos * p.cos_st + i]);
        const float s = E::to_float(reinterpret_cast<const T*>(p.sin)[pos * p.sin_st + i]);
        const float other = u[n] * inv;
        r = e < half ? own * c - other * s : other * s + own * c;
      }
      y[e] = E::from_float(r);
    }
  }
}

template <typename T>
cudaError_t launch_typed(const NormRopeParams& p, bool vec, int sms, cudaStream_t stream) {
  const int threads = 256, warps = threads / 32;
  const int heads = p.n_head + p.n_kv_head;
  int64_t items = p.n_tokens * heads;
  if (vec) {
    const int per_warp = 32 / (p.head_dim / 8) * NORM_HEADS;
    items = p.n_tokens * ((heads + per_warp - 1) / per_warp);
  }
  int64_t blocks = (items + warps - 1) / warps;
  if (blocks > int64_t(sms) * 64) blocks = int64_t(sms) * 64;
  if (!vec)
    pd_norm_rope_any_kernel<T><<<unsigned(blocks), threads, 0, stream>>>(p);
  else if (p.head_dim == 64)
    pd_norm_rope_kernel<T, 8><<<unsigned(blocks), threads, 0, stream>>>(p);
  else if (p.head_dim == 128)
    pd_norm_rope_kernel<T, 16><<<unsigned(blocks), threads, 0, stream>>>(p);
  else
    pd_norm_rope_kernel<T, 32><<<unsigned(blocks), threads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeParams& p, int dtype, bool vec, int sms, cudaStream_t stream) {
  switch (dtype) {
    case 0: return launch_typed<float>(p, vec, sms, stream);
    case 1: return launch_typed<__half>(p, vec, sms, stream);
    case 2: return launch_typed<__nv_bfloat16>(p, vec, sms, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace pd
