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
// them, and a lane has 64 bytes in flight. Measured: 6001 tokens of 8 + 2 heads of 256, fp16, 62 MB,
// 14.0 us (4.4 TB/s, two thirds of the copy rate; some 2 us of it the launch); one token 2.2 us. Rows at
// any other head_dim or alignment take the second kernel, one element of 2 or 4 bytes at a time: 6001 tokens of
// 16 + 8 heads of 128, bf16, 14.5 us aligned and 89 us one element off; of 96, 84 us; one token 3.0 us.
#include "pd_internal.h"
#include "pd_norm_rope.cuh"

namespace pd {

namespace {

constexpr int NORM_HEADS = 4;  // heads in flight per lane group
constexpr int THREADS = 128;    // of a CTA: small, so that the last ones spread evenly (14.1 us, 14.4 with 256)

// 4 consecutive elements as they are in memory: 8 bytes of 16-bit types, 16 of fp32.
template <typename T>
struct Four {
  using Raw = uint2;
  __device__ __forceinline__ static void unpack(const Raw& r, float (&f)[4]) {
    Elem<T>::unpack2(r.x, f);
    Elem<T>::unpack2(r.y, f + 2);
  }
  __device__ __forceinline__ static Raw pack(const float (&f)[4]) {
    return make_uint2(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]));
  }
};
template <>
struct Four<float> {
  using Raw = float4;
  __device__ __forceinline__ static void unpack(const Raw& r, float (&f)[4]) {
    f[0] = r.x;
    f[1] = r.y;
    f[2] = r.z;
    f[3] = r.w;
  }
  __device__ __forceinline__ static Raw pack(const float (&f)[4]) { return make_float4(f[0], f[1], f[2], f[3]); }
};

__device__ __forceinline__ int64_t position_of(const NormRopeParams& p, int64_t t) {
  if (p.pos == nullptr) return t;
  return p.pos_i64 ? reinterpret_cast<const int64_t*>(p.pos)[t]
                   : int64_t(reinterpret_cast<const int32_t*>(p.pos)[t]);
}

// LANES = D / 8 lanes per head (8, 16 or 32). Lane l of a head holds elements e0 .. e0 + 3 and
// e1 .. e1 + 3: a rotary pair block while 4 l < R / 2, two blocks of the passed-through rest after.
// What is loaded stays packed until its head's turn: four heads in flight then cost 16 registers.
template <typename T, int LANES>
__global__ void __launch_bounds__(THREADS, 8) pd_norm_rope_kernel(const NormRopeParams p) {
  constexpr int D = LANES * 8;
  constexpr int GROUPS = 32 / LANES;  // heads of a warp at once
  using F = Four<T>;
  using Raw = typename F::Raw;
  const int lane = threadIdx.x & 31;
  const int l = lane % LANES, grp = lane / LANES;
  constexpr int PER_WARP = GROUPS * NORM_HEADS;
  // an item is a token and PER_WARP of its q heads, or of its k heads
  const uint32_t q_chunks = (p.n_head + PER_WARP - 1) / PER_WARP, k_chunks = (p.n_kv_head + PER_WARP - 1) / PER_WARP;
  const uint32_t chunks = q_chunks + k_chunks;
  const int64_t items = p.n_tokens * chunks;
  const int half = p.rotary_dim >> 1;
  const bool rot = 4 * l < half;
  const int e0 = rot ? 4 * l : p.rotary_dim + 8 * (l - half / 4);
  const int e1 = rot ? half + 4 * l : e0 + 4;
  for (int64_t it = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items;
       it += int64_t(gridDim.x) * (blockDim.x >> 5)) {
    const int64_t t = it < 0x7fffffff ? int64_t(uint32_t(it) / chunks) : it / chunks;
    const uint32_t ch = uint32_t(it - t * chunks);
    const int64_t pos = position_of(p, t);
    const bool is_q = ch < q_chunks;
    const int h0 = int(is_q ? ch : ch - q_chunks) * PER_WARP + grp;
    const int heads = is_q ? p.n_head : p.n_kv_head;
    const int64_t sh = (is_q ? p.q_sh : p.k_sh), so = (is_q ? p.qo_sh : p.ko_sh);
    const T* x = (is_q ? reinterpret_cast<const T*>(p.q) + t * p.q_st : reinterpret_cast<const T*>(p.k) + t * p.k_st) +
                 h0 * sh;
    T* y = (is_q ? reinterpret_cast<T*>(p.q_out) + t * p.qo_st : reinterpret_cast<T*>(p.k_out) + t * p.ko_st) + h0 * so;
    Raw a[NORM_HEADS], b[NORM_HEADS];
#pragma unroll
    for (int j = 0; j < NORM_HEADS; ++j) {
      a[j] = b[j] = Raw{};
      if (h0 + j * GROUPS < heads) {
        a[j] = __ldcs(reinterpret_cast<const Raw*>(x + e0));
        b[j] = __ldcs(reinterpret_cast<const Raw*>(x + e1));
      }
      x += GROUPS * sh;
    }
    const bool in_range = pos >= 0 && pos < p.n_pos;
    if (!in_range && lane == 0) atomicOr(p.err, DEVERR_ROPE_RANGE);
    // out_a = inv (x_a w_a cos - x_b w_b sin), out_b = inv (x_a w_a sin + x_b w_b cos): the four
    // products of weight and angle are the item's, not the head's
    float ac[4], as[4], bc[4], bs[4];
    {
      const T* w = reinterpret_cast<const T*>(is_q ? p.wq : p.wk);
      float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f}, wa[4], wb[4];
      F::unpack(__ldg(reinterpret_cast<const Raw*>(w + e0)), wa);
      F::unpack(__ldg(reinterpret_cast<const Raw*>(w + e1)), wb);
      if (rot && in_range) {
        F::unpack(__ldg(reinterpret_cast<const Raw*>(reinterpret_cast<const T*>(p.cos) + pos * p.cos_st + 4 * l)), c);
        F::unpack(__ldg(reinterpret_cast<const Raw*>(reinterpret_cast<const T*>(p.sin) + pos * p.sin_st + 4 * l)), s);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ac[i] = wa[i] * c[i];
        as[i] = wa[i] * s[i];
        bc[i] = wb[i] * c[i];
        bs[i] = wb[i] * s[i];
      }
    }
#pragma unroll
    for (int j = 0; j < NORM_HEADS; ++j) {
      float xa[4], xb[4];
      F::unpack(a[j], xa);
      F::unpack(b[j], xb);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) ss = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], ss));
#pragma unroll
      for (int o = LANES / 2; o >= 1; o >>= 1) ss += __shfl_xor_sync(FULL_MASK, ss, o);
      const float inv = rsqrtf(ss * (1.f / D) + p.eps);  // 2 ulp
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float u = (xa[i] * ac[i] - xb[i] * bs[i]) * inv;
        xb[i] = (xa[i] * as[i] + xb[i] * bc[i]) * inv;
        xa[i] = u;
      }
      if (h0 + j * GROUPS < heads) {
        // zeros by choice, not by a product: 0 times an infinity would be NaN
        *reinterpret_cast<Raw*>(y + e0) = in_range ? F::pack(xa) : Raw{};
        *reinterpret_cast<Raw*>(y + e1) = in_range ? F::pack(xb) : Raw{};
      }
      y += GROUPS * so;
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
    const float inv = rsqrtf(ss / float(d) + p.eps);
    __syncwarp();  // every lane has read its partners before a lane stores over them (shuffles order no memory)
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
      y[e] = E::from_float(in_range ? r : 0.f);
    }
  }
}

template <typename T>
cudaError_t launch_typed(const NormRopeParams& p, bool vec, int sms, cudaStream_t stream) {
  const int threads = vec ? THREADS : 256, warps = threads / 32;
  const int heads = p.n_head + p.n_kv_head;
  int64_t items = p.n_tokens * heads;
  if (vec) {
    const int per_warp = 32 / (p.head_dim / 8) * NORM_HEADS;
    items = p.n_tokens * ((p.n_head + per_warp - 1) / per_warp + (p.n_kv_head + per_warp - 1) / per_warp);
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
