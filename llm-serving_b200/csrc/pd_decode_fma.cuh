// pd_decode_fma.cuh -- tile math of the few rows' decode kernel for fp32 K/V (head_dim 64..256): fp32 multiply-adds.
//
// A row of K or V is spread over LPR lanes, 16 bytes a chunk, so a warp's load covers RPL tokens. Every lane of a row ends
// with the row's scores (an all-reduce over its lanes) and adds p v to accumulators of its own dimensions; with two
// rows to a load the halves' accumulators are added at the end. Registers hold all of a tile's scores, so no
// probability is exchanged. The tiles are few here: 8 rows of 1000 tokens on 8 heads of 128 are bound by the round trips
// around them, not by these instructions.
#pragma once

#include "pd_common.cuh"
#include "pd_tile.cuh"

namespace pd {

template <int D, int GT>
struct FmaWorker {
  static constexpr int TILE = 1024 / D;
  static constexpr int CHUNKS = D / 4;
  static constexpr int LPR = CHUNKS < 32 ? CHUNKS : 32;  // lanes of a row
  static constexpr int RPL = 32 / LPR;                   // rows of a load
  static constexpr int CPL = CHUNKS / LPR;               // chunks of a lane
  static constexpr int NT = TILE / RPL;                  // tokens of a lane
  static constexpr int R = NT * GT;                      // its scores: token i's of head g at i * GT + g
  static constexpr int AT_ONCE = 4;

  int pos, half;  // lane of the row, row of the load
  float4 q[GT][CPL], acc[GT][CPL];
  float m_run[GT], l_run[GT];  // l: this lane's tokens

  __device__ __forceinline__ void init(int lane, int, int) {
    pos = lane & (LPR - 1);
    half = lane / LPR;
  }

  __device__ __forceinline__ void start(const float* qrow, int64_t q_sh, int hq0, int heads) {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      m_run[g] = MAX_START;
      l_run[g] = 0.f;
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        acc[g][c] = make_float4(0.f, 0.f, 0.f, 0.f);
        q[g][c] = g < heads ? __ldg(reinterpret_cast<const float4*>(qrow + int64_t(hq0 + g) * q_sh) + c * LPR + pos)
                            : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }

  __device__ __forceinline__ float4 chunk(uint32_t base, int i, int c) const {
    const uint4 w = lds128(base + uint32_t((i * RPL + half) * (D * 4) + (c * LPR + pos) * 16));
    return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
  }

  template <typename Live>
  __device__ __forceinline__ void scores(uint32_t kbase, const Live& live, float scale_log2, float (&sc)[R]) const {
    // AT_ONCE tokens' loads, products and exchanges side by side, so that none waits for another's
#pragma unroll
    for (int i0 = 0; i0 < NT; i0 += AT_ONCE) {
      float4 k[AT_ONCE][CPL];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
        for (int c = 0; c < CPL; ++c) k[i][c] = chunk(kbase, i0 + i, c);
      float s[AT_ONCE * GT];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          float x = 0.f, y = 0.f;
#pragma unroll
          for (int c = 0; c < CPL; ++c) {
            x = fmaf(k[i][c].x, q[g][c].x, fmaf(k[i][c].y, q[g][c].y, x));
            y = fmaf(k[i][c].z, q[g][c].z, fmaf(k[i][c].w, q[g][c].w, y));
          }
          s[i * GT + g] = x + y;
        }
#pragma unroll
      for (int o = LPR / 2; o >= 1; o >>= 1)
#pragma unroll
        for (int e = 0; e < AT_ONCE * GT; ++e) s[e] += __shfl_xor_sync(FULL_MASK, s[e], o);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const bool counts = live((i0 + i) * RPL + half);
#pragma unroll
        for (int g = 0; g < GT; ++g) sc[(i0 + i) * GT + g] = counts ? s[i * GT + g] * scale_log2 : -INFINITY;
      }
    }
  }

  __device__ __forceinline__ void max_update(const float (&sc)[R]) {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      float t = sc[g];
#pragma unroll
      for (int i = 1; i < NT; ++i) t = fmaxf(t, sc[i * GT + g]);
      if constexpr (RPL == 2) t = fmaxf(t, __shfl_xor_sync(FULL_MASK, t, LPR));
      if (t > m_run[g]) {  // the same in every lane
        const float alpha = exp2f(m_run[g] - t);
        m_run[g] = t;
        l_run[g] *= alpha;
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          acc[g][c].x *= alpha;
          acc[g][c].y *= alpha;
          acc[g][c].z *= alpha;
          acc[g][c].w *= alpha;
        }
      }
    }
  }

  // Every lane picks one score of each LPR and stores it. (Written as selections: the compiler would make an indexed
  // read of local memory of the conditional expressions, and a tile twice as long.)
  template <typename Live>
  __device__ __forceinline__ void store_scores(float* dst, int, int, const Live&, const float (&sc)[R]) const {
#pragma unroll
    for (int j0 = 0; j0 < R; j0 += LPR) {
      float x = sc[j0];
#pragma unroll
      for (int j = j0 + 1; j < j0 + LPR && j < R; ++j)
        asm("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, %2;\n\tselp.f32 %0, %3, %0, p;\n\t}" : "+f"(x) : "r"(pos), "r"(j - j0), "f"(sc[j]));
      const int j = j0 + pos;
      if (j < R) dst[((j / GT) * RPL + half) * GT + j % GT] = x;
    }
  }

  // Tokens that do not count have P = 0 and their V is taken as zero, whatever the bytes.
  template <typename Live>
  __device__ __forceinline__ void pv(uint32_t vbase, const float (&sc)[R], const Live& live, bool full) {
#pragma unroll
    for (int i0 = 0; i0 < NT; i0 += AT_ONCE) {
      float4 v[AT_ONCE][CPL];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const bool counts = full || live((i0 + i) * RPL + half);
#pragma unroll
        for (int c = 0; c < CPL; ++c) {
          v[i][c] = chunk(vbase, i0 + i, c);
          if (!counts) v[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
#pragma unroll
        for (int g = 0; g < GT; ++g) {
          const float p = exp2f(sc[(i0 + i) * GT + g] - m_run[g]);
          l_run[g] += p;
#pragma unroll
          for (int c = 0; c < CPL; ++c) {
            acc[g][c].x = fmaf(p, v[i][c].x, acc[g][c].x);
            acc[g][c].y = fmaf(p, v[i][c].y, acc[g][c].y);
            acc[g][c].z = fmaf(p, v[i][c].z, acc[g][c].z);
            acc[g][c].w = fmaf(p, v[i][c].w, acc[g][c].w);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void total_l(float (&l_tot)[GT]) const {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      l_tot[g] = l_run[g];
      if constexpr (RPL == 2) l_tot[g] += __shfl_xor_sync(FULL_MASK, l_tot[g], LPR);
    }
  }

  __device__ __forceinline__ void store_ml(float* m_dst, float* l_dst, const float (&l_tot)[GT]) const {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
      if (pos == 0 && half == 0) {
        m_dst[g] = m_run[g];
        l_dst[g] = l_tot[g];
      }
    }
  }

  // Unnormalised accumulators, head-major rows of D floats.
  __device__ __forceinline__ void store_acc(float* dst) const {
#pragma unroll
    for (int g = 0; g < GT; ++g) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) {
        float4 a = acc[g][c];
        if constexpr (RPL == 2) {
          a.x += __shfl_xor_sync(FULL_MASK, a.x, LPR);
          a.y += __shfl_xor_sync(FULL_MASK, a.y, LPR);
          a.z += __shfl_xor_sync(FULL_MASK, a.z, LPR);
          a.w += __shfl_xor_sync(FULL_MASK, a.w, LPR);
        }
        if (half == 0) *reinterpret_cast<float4*>(dst + g * D + (c * LPR + pos) * 4) = a;
      }
    }
  }
};

}  // namespace pd
