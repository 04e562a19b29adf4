// pd_fp4_attend.cuh -- attention of few query tokens over 4-bit pages: the decode step, and short
// chunks (sm_100a; fp16 / bf16 queries, head_dim 64, 128 or 256, any group).
//
// For query token i of row b's chunk (one token in a decode step) and q head h, over the row's
// visible keys j <= lim = seqlen - chunk + i:
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp2(s_j - max s),  s_j = q . k_j * scale * log2(e)
// with fp32 scores, maxima, sums and accumulators; no visible key gives zeros.
//
// Bound by memory in a decode step: 9/16 of a byte per cached element is read once, and a lane has
// about 0.9 instruction slots per element at the copy rate, so the element's way into the
// matrix instruction has to be short. Per 16-token record a warp computes
//   S^T = K q^T    m16n8k16, M = tokens, N = 8 columns, K = head_dim
//   O^T += V^T P^T m16n8k16, M = head_dim, N = 8 columns, K = tokens
// where a column is one (query token, q head of the kv head's group) pair. Operands never pass
// through a transposing load: the record's byte order (pd_fp4.cuh) hands lane (g, c) exactly the
// codes of its A fragments. Which elements sit in which k slot or m row is free as long as the
// other operand agrees, so K's k slots are 32 c + 4 ks + .. (a lane's own 16 bytes), and V's rows
// 16 g + .. (a lane's own group), which also makes a lane's outputs consecutive in memory. Codes
// become fp16 by the hardware conversion and take their scale with one packed multiply: exact
// both, so the products are those of the values the cache stands for.
//  * q enters as fp16: a column is scaled by a power of two that puts its largest element near
//    2^13, exact for fp16 and for every bf16 element within 2^-27 of the largest.
//  * P enters as one fp16 for bf16 results: a result is off by at most 2^-11 of the weighted mean of |v|
//    (the weights' sum is kept unrounded in fp32), an eighth of a bf16 half ulp of that mean. fp16 results,
//    no coarser than that, get two fp16 parts (2^-22).
//  * tokens past the row are masked to P = 0 and their V scales to 0, so whatever bytes a page
//    holds there (a NaN scale included) never reaches the sums.
//
// Work split: the (row, kv head, column block, tile) sequence is cut into equal runs, one per
// CTA and in it one per warp, so every SM streams the same number of bytes whatever the lengths.
// Each warp prefetches its run through its own ring of tiles (two records, 32 keys) in shared
// memory by bulk copies of 18 D bytes per record, or of both where they share a page: no lane but
// a page's own spends instructions on it, and no warp waits for another's data. A unit (row, kv
// head, column block) cut between warps leaves partial (m, l, acc) pieces that the CTA joins in shared memory; a unit cut between CTAs goes through the
// workspace and the last CTA to arrive joins it, in piece order whoever arrives last, so results
// do not depend on timing, and a CTA that is not last leaves. Where there are no more units than
// CTAs, a unit may get a CTA of its own instead (JOIN_TILES).
//
// Measured, bf16, 16 heads on 8 of 128: 32 rows of 8192 tokens, 302 MB, 66.9 us (4.5 TB/s, 0.69 of the
// copy rate; the loads alone reach 0.95), 32 of 2048 25.2 us, one of 700 9.7 us; 61 rows of skewed lengths,
// 8 heads on 2 of 256, fp16, 59 MB, 28.6 us; in fp16 (P in two parts) the first two take 74.3 and 27.3. What is
// left over the bytes: 339 warp instructions per record, 312 in the loop and the rest what a warp spends
// outside it (64 conversions, 64 multiplies and 16 MMAs at least; schedulers issue in 0.62 of their
// cycles, with 4 warps each to choose from), and some 6 us of start, joins and launch.
#pragma once

#include "pd_fp4.cuh"
#include "pd_internal.h"

#include <type_traits>

namespace pd {

namespace fp4 {

constexpr int MAX_ROWS = 896;  // rows of one launch (their prefix sums are in shared memory)
constexpr int COLS = 8;         // columns of a unit
constexpr int TILE = 2 * FP4_TILE;  // keys of a warp's step: two records
// What a join between CTAs costs, in tiles of one CTA: where there are no more units than CTAs, units
// stay whole if the longest is at most this much more than an even share. One row of 700 tokens (22
// tiles, 8 units) takes 9.6 us whole and 9.9 cut, of 2048 (64 tiles) 14.5 and 10.0; 16 rows of 2048
// (128 units) 15.4 and 18.3.
constexpr int JOIN_TILES = 24;
// Fewest tiles of a CTA where units are cut: one row of 2048 tokens takes 10.0 us with 8, 10.7 with 4.
constexpr int CTA_TILES = 8;
// A running maximum below every score: finite, so that exp2(score - maximum) needs no special case
// for columns that have seen no key (their scores are -inf).
constexpr float NO_MAX = -3.0e38f;

// Floats of one CTA-level partial: m and l of 8 columns, then 8 x D accumulators.
__host__ __device__ constexpr int partial_floats(int d) { return 2 * COLS + COLS * d; }

// Bulk copy of `bytes` (a multiple of 16) into shared memory, counted on the mbarrier; the source
// is read once, so its lines are the first to leave the L2.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar), "l"(pol)
      : "memory");
}

__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp, subnormal results flushed to zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t r;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}

// One row's geometry.
struct Row {
  int q_begin;  // first query token in the packed tensor
  int sq;       // query tokens attended
  int chunk;    // query tokens of the row
  int lk;       // keys
};

__device__ __forceinline__ Row row_of(const Fp4AttendParams& p, int b) {
  Row r;
  r.q_begin = b;
  r.sq = 1;
  if (p.cu_q != nullptr) {  // offsets are held inside the packed tensor
    r.q_begin = min(max(__ldg(p.cu_q + b), 0), p.total_q);
    r.sq = min(max(__ldg(p.cu_q + b + 1), 0), p.total_q) - r.q_begin;
    r.sq = r.sq < 0 ? 0 : r.sq;
  }
  r.chunk = r.sq;  // a longer chunk than announced keeps its tokens' positions
  r.sq = r.sq > p.max_seqlen_q ? p.max_seqlen_q : r.sq;
  r.lk = __ldg(p.seqlen + b);
  r.lk = r.lk < 0 ? 0 : (r.lk > p.capacity ? p.capacity : r.lk);
  return r;
}

// One warp's columns: queries, running softmax and accumulators.
template <typename T, int D>
struct Worker {
  static constexpr int W = D < 128 ? D : 128;  // elements of a K code block
  static constexpr int BLK = D / W;
  static constexpr int KSB = W / 16;           // k steps of a block
  static constexpr int KS = D / 16;
  static constexpr int MT = D / 16;            // 16-row tiles of O^T
  using E = Elem<T>;
  using X = Mma<__half>;

  int lane, g, c;
  uint32_t qb[KS][2];
  float o[MT][4];
  float m_run[2], l_run[2];  // reference (a maximum less FP4_P_SHIFT) and sum of the weights
  float bar[2];  // the scores above it move the reference: FP4_HEADROOM over the maximum it was set from
  float mul[2];  // score multiplier of columns 2c, 2c + 1
  int lim[2];    // their last visible key
  int open_lim;  // keys up to this one are visible to every live column

  __device__ __forceinline__ void init(int lane_) {
    lane = lane_;
    g = lane >> 2;
    c = lane & 3;
  }

  // Opens a unit: column n = first + n is (token n / group, head n % group) of the row's chunk.
  __device__ __forceinline__ void start(const Fp4AttendParams& p, const Row& r, int h, int first) {
    const int cols = r.sq * p.group;
    const int n = first + g;
    const bool live = n < cols;
    const int tok = live ? n / p.group : 0, hg = live ? n - tok * p.group : 0;
    const T* src = reinterpret_cast<const T*>(p.q) + int64_t(r.q_begin + tok) * p.q_st +
                   int64_t(h * p.group + hg) * p.q_sh;
    float x[KS * 4];
    float top = 0.f;
#pragma unroll
    for (int b = 0; b < BLK; ++b) {
#pragma unroll
      for (int u = 0; u < KSB / 2; ++u) {  // 8 elements from W/4 c + 8 u
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (live) raw = __ldg(reinterpret_cast<const uint4*>(src + b * W + c * (W / 4) + u * 8));
        E::unpack(raw, x + (b * KSB / 2 + u) * 8);
      }
    }
#pragma unroll
    for (int i = 0; i < KS * 4; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 1));
    top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 2));
    // 2^(13 - floor(log2 top)), at most 2^126 (its inverse is a normal number); 1 for zero and for
    // non-finite columns
    int e = int(__float_as_uint(top) >> 23);
    e = e == 0 || e == 255 ? 140 : e;
    int shift = 140 - e;
    shift = shift > 126 ? 126 : shift;  // at least -114
    const float up = __uint_as_float(uint32_t(127 + shift) << 23);
    const float down = __uint_as_float(uint32_t(127 - shift) << 23);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qb[ks][0] = Elem<__half>::pack2(x[4 * ks] * up, x[4 * ks + 1] * up);
      qb[ks][1] = Elem<__half>::pack2(x[4 * ks + 2] * up, x[4 * ks + 3] * up);
    }
    const float unit = p.units != nullptr ? __ldg(p.units + h) : 1.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mul[j] = __shfl_sync(FULL_MASK, down, (2 * c + j) * 4) * (p.scale_log2 * unit);
      const int col = first + 2 * c + j;
      lim[j] = col < cols ? r.lk - r.chunk + col / p.group : -1;
      m_run[j] = bar[j] = NO_MAX;
      l_run[j] = 0.f;
    }
    open_lim = r.lk - r.chunk + first / p.group;  // columns are in token order: the first sees least
#pragma unroll
    for (int m = 0; m < MT; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
  }

  // q . k of the 16 tokens of the record at shared address `a`: acc[0], acc[1] token g of columns 2c,
  // 2c + 1; acc[2], acc[3] token g + 8.
  __device__ __forceinline__ void scores(uint32_t a, float (&acc)[4]) const {
    acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
#pragma unroll
    for (int b = 0; b < BLK; ++b) {
      alignas(16) uint32_t w0[KSB / 2], w1[KSB / 2];  // codes of tokens g and g + 8
      uint32_t s0[2], s1[2];              // their scale pairs, one per 16 elements
      const uint32_t ka = a + b * 8 * W + g * (W / 2) + c * (W / 8);
      const uint32_t sa = a + 8 * D + b * W + g * (W / 16);
      if constexpr (W == 128) {
        *reinterpret_cast<uint4*>(w0) = lds128(ka);
        *reinterpret_cast<uint4*>(w1) = lds128(ka + 4 * W);
        const uint32_t x0 = e4m3x2_to_half2(lds16(sa + 2 * c));
        const uint32_t x1 = e4m3x2_to_half2(lds16(sa + W / 2 + 2 * c));
        s0[0] = __byte_perm(x0, 0, 0x1010);
        s0[1] = __byte_perm(x0, 0, 0x3232);
        s1[0] = __byte_perm(x1, 0, 0x1010);
        s1[1] = __byte_perm(x1, 0, 0x3232);
      } else {
        *reinterpret_cast<uint2*>(w0) = lds64(ka);
        *reinterpret_cast<uint2*>(w1) = lds64(ka + 4 * W);
        s0[0] = s0[1] = __byte_perm(e4m3x2_to_half2(lds8(sa + c)), 0, 0x1010);
        s1[0] = s1[1] = __byte_perm(e4m3x2_to_half2(lds8(sa + W / 2 + c)), 0, 0x1010);
      }
#pragma unroll
      for (int u = 0; u < KSB / 2; ++u) {
        uint32_t x[4], y[4];
        e2m1x8_to_half2x4(w0[u], x);
        e2m1x8_to_half2x4(w1[u], y);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = hmul2_bits(x[i], s0[u >> 1]);
          y[i] = hmul2_bits(y[i], s1[u >> 1]);
        }
        const int ks = b * KSB + 2 * u;
        X::m16n8k16(acc, x[0], y[0], x[1], y[1], qb[ks][0], qb[ks][1]);
        X::m16n8k16(acc, x[2], y[2], x[3], y[3], qb[ks + 1][0], qb[ks + 1][1]);
      }
    }
  }

  // O^T += V^T P^T of the record at `a`, P as its fragment pair (pb0: tokens 0 .. 7, pb1: 8 .. 15);
  // its tokens from `rows` on count as zeros.
  template <int PARTS>
  __device__ __forceinline__ void values(uint32_t a, const uint32_t (&pb0)[PARTS], const uint32_t (&pb1)[PARTS],
                                         int rows) {
    // scales of tokens 2c, 2c + 1 and 2c + 8, 2c + 9; zero past the row
    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
    if (rows < FP4_TILE) {
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int t = 8 * hi + 2 * c;
        keep[hi] = (t < rows ? 0x0000ffffu : 0u) | (t + 1 < rows ? 0xffff0000u : 0u);
      }
    }
#pragma unroll
    for (int b = 0; b < BLK; ++b) {
      alignas(16) uint32_t v[2][4];
      uint32_t sv[2];
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const uint32_t va = a + 9 * D + hi * 4 * D;
        const uint32_t sa = a + 17 * D + hi * (D / 2);
        if constexpr (W == 128) {  // words 0, 1: token 2c; words 2, 3: token 2c + 1
          *reinterpret_cast<uint4*>(v[hi]) = lds128(va + (b * 8 + g) * 64 + c * 16);
          sv[hi] = e4m3x2_to_half2(lds16(sa + (b * 8 + g) * 8 + 2 * c)) & keep[hi];
        } else {  // a lane's 8 rows are half a group: one word per token
          const uint32_t q = va + (g >> 1) * 64 + c * 16 + (g & 1) * 4;
          v[hi][0] = lds32(q);
          v[hi][2] = lds32(q + 8);
          v[hi][1] = v[hi][3] = 0u;
          sv[hi] = e4m3x2_to_half2(lds16(sa + (g >> 1) * 8 + 2 * c)) & keep[hi];
        }
      }
#pragma unroll
      for (int u = 0; u < (W == 128 ? 2 : 1); ++u) {
        uint32_t even[2][4], odd[2][4];
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {
          // bytes of (token 2c, token 2c + 1) nibble pairs: even elements, then odd ones
          const uint32_t x = v[hi][u], y = v[hi][2 + u];
          e2m1x8_to_half2x4((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), even[hi]);
          e2m1x8_to_half2x4(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), odd[hi]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            even[hi][i] = hmul2_bits(even[hi][i], sv[hi]);
            odd[hi][i] = hmul2_bits(odd[hi][i], sv[hi]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            X::m16n8k16(o[b * 8 + u * 4 + i], even[0][i], odd[0][i], even[1][i], odd[1][i], pb0[part], pb1[part]);
      }
    }
  }

  // A tile of two records at shared address `a`: keys t0 .. t0 + 31, of which `rows` exist. Two
  // records share the maximum's test, the wait and the copy of a tile, and give the scheduler
  // two independent chains.
  __device__ __forceinline__ void tile(uint32_t a, int t0, int rows) {
    float sc[8];
    // both records whatever `rows`: what an absent one holds is masked below
    scores(a, *reinterpret_cast<float(*)[4]>(sc));
    scores(a + fp4_record_bytes(D), *reinterpret_cast<float(*)[4]>(sc + 4));
#pragma unroll
    for (int i = 0; i < 8; ++i) sc[i] *= mul[i & 1];
    if (t0 + 2 * FP4_TILE - 1 > open_lim) {  // some column's last key, or the row's, is in this tile
#pragma unroll
      for (int i = 0; i < 8; ++i)
        sc[i] = t0 + (i >> 2) * FP4_TILE + 8 * ((i >> 1) & 1) + g <= lim[i & 1] ? sc[i] : -INFINITY;
    }
    float top[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) top[j] = fmaxf(fmaxf(sc[j], sc[2 + j]), fmaxf(sc[4 + j], sc[6 + j]));
    if (__any_sync(FULL_MASK, top[0] > bar[0] || top[1] > bar[1])) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float t = top[j];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) t = fmaxf(t, __shfl_xor_sync(FULL_MASK, t, off));
        t = fmaxf(t - FP4_P_SHIFT, m_run[j]);
        const float alpha = ex2(m_run[j] - t);
        m_run[j] = t;
        bar[j] = t + (FP4_P_SHIFT + FP4_HEADROOM);  // rescaling the accumulators is then rare
        l_run[j] *= alpha;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          o[m][j] *= alpha;
          o[m][2 + j] *= alpha;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sc[i] = ex2(sc[i] - m_run[i & 1]);
      l_run[i & 1] += sc[i];
    }
    // P is one fp16 operand for bf16 outputs (2^-11 is an eighth of their half ulp) and a hi + lo pair
    // for fp16 outputs, whose rounding is no coarser than fp16 P's
    constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      uint32_t pb[2][PARTS];
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const float p0 = sc[4 * r + 2 * hi], p1 = sc[4 * r + 2 * hi + 1];
        const uint32_t whole = Elem<__half>::pack2(p0, p1);
        pb[hi][0] = movmatrix_trans(whole);
        if constexpr (PARTS == 2) {
          float f[2];
          Elem<__half>::unpack2(whole, f);
          pb[hi][1] = movmatrix_trans(Elem<__half>::pack2(p0 - f[0], p1 - f[1]));
        }
      }
      values<PARTS>(a + r * fp4_record_bytes(D), pb[0], pb[1], rows - r * FP4_TILE);
    }
  }

  __device__ __forceinline__ void total(float (&l)[2]) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x = l_run[j];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) x += __shfl_xor_sync(FULL_MASK, x, off);
      l[j] = x;
    }
  }

  // First head_dim element of this lane's run in 128-element block b, and the run's length.
  static constexpr int RUN = W / 8;  // 16, or 8 at head_dim 64
  __device__ __forceinline__ int run0(int b) const { return b * W + g * RUN; }

  // The finished unit: out rows of columns 2c and 2c + 1.
  __device__ __forceinline__ void finish(const Fp4AttendParams& p, const Row& r, int h, int first) const {
    float l[2];
    total(l);
    const float unit = p.units != nullptr ? __ldg(p.units + p.n_kv_head + h) : 1.f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = first + 2 * c + j;
      if (n >= r.sq * p.group) continue;
      const float inv = l[j] > 0.f ? unit / l[j] : 0.f;
      const int tok = n / p.group, hg = n - tok * p.group;
      T* dst = reinterpret_cast<T*>(p.out) + int64_t(r.q_begin + tok) * p.o_st + int64_t(h * p.group + hg) * p.o_sh;
#pragma unroll
      for (int b = 0; b < BLK; ++b) {
        uint32_t w[RUN / 2];
#pragma unroll
        for (int i = 0; i < RUN / 2; ++i) w[i] = E::pack2(o[b * 8 + i][j] * inv, o[b * 8 + i][2 + j] * inv);
#pragma unroll
        for (int i = 0; i < RUN / 8; ++i)
          *reinterpret_cast<uint4*>(dst + run0(b) + 8 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      }
    }
  }

  // A partial unit: m[8], l[8] and acc[cols][D] (fp32, unnormalised, without the V unit).
  __device__ __forceinline__ void store_piece(float* ml, float* acc, int cols) const {
    float l[2];
    total(l);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = 2 * c + j;
      if (n >= cols) continue;
      if (g == 0) {
        ml[n] = m_run[j];
        ml[COLS + n] = l[j];
      }
#pragma unroll
      for (int b = 0; b < BLK; ++b)
#pragma unroll
        for (int i = 0; i < RUN / 2; ++i)
          *reinterpret_cast<float2*>(acc + n * D + run0(b) + 2 * i) = make_float2(o[b * 8 + i][j], o[b * 8 + i][2 + j]);
    }
  }
};

// A partial unit of this CTA: tiles [t0, t1) of the `tiles` of unit `unit` of row `row`, with what a
// join needs to know of it, so that no join looks lengths up or divides again.
struct alignas(16) Piece {
  int row, unit, t0, t1;  // row < 0: none
  int tiles, h, first, cols;
  int q_begin, pad[3];
};

// Joins `n` pieces' four elements of column col: ml(i) is piece i's (m, l) block, acc(i) its elements.
template <typename Ml, typename Acc>
__device__ __forceinline__ void join4(int n, int col, Ml ml, Acc acc, float (&x)[4], float& m, float& l) {
  m = NO_MAX;
  for (int i = 0; i < n; ++i) m = fmaxf(m, ml(i)[col]);
  l = 0.f;
  x[0] = x[1] = x[2] = x[3] = 0.f;
  for (int i = 0; i < n; ++i) {
    const float f = ex2(ml(i)[col] - m);
    const float4 v = acc(i);
    l = fmaf(f, ml(i)[COLS + col], l);
    x[0] = fmaf(f, v.x, x[0]);
    x[1] = fmaf(f, v.y, x[1]);
    x[2] = fmaf(f, v.z, x[2]);
    x[3] = fmaf(f, v.w, x[3]);
  }
}

template <typename T>
__device__ __forceinline__ void store_out4(const Fp4AttendParams& p, const Piece& a, int col, int e, const float (&x)[4],
                                           float l) {
  const float unit = p.units != nullptr ? __ldg(p.units + p.n_kv_head + a.h) : 1.f;
  const float inv = l > 0.f ? unit / l : 0.f;
  const int n = a.first + col, tok = n / p.group, hg = n - tok * p.group;
  T* dst = reinterpret_cast<T*>(p.out) + int64_t(a.q_begin + tok) * p.o_st + int64_t(a.h * p.group + hg) * p.o_sh + e;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(Elem<T>::pack2(x[0] * inv, x[1] * inv), Elem<T>::pack2(x[2] * inv, x[3] * inv));
}

// Shared memory: [stage barriers (NW x stages) | prefix int64 (rows + 1) | tiles and units per row |
// pieces | piece (m, l) | leading pieces' accumulators (NW x cols x D) | rings (NW x stages x 2
// records)]. A warp's trailing piece is its last work: its accumulators take the warp's ring, which
// holds 18 D x 2 bytes a stage and so at least the 32 D of eight columns.
struct Smem {
  int pre_off, rows_off, piece_off, ml_off, acc_off, ring_off, bytes;
};

__host__ __device__ constexpr Smem smem_layout(int batch, int nw, int cols, int d, int stages) {
  Smem s{};
  s.pre_off = nw * stages * 8;
  s.rows_off = s.pre_off + (batch + 1) * 8;
  s.piece_off = (s.rows_off + batch * 8 + 15) & ~15;
  s.ml_off = s.piece_off + 2 * nw * int(sizeof(Piece));
  s.acc_off = s.ml_off + 2 * nw * 2 * COLS * 4;
  s.ring_off = (s.acc_off + nw * cols * d * 4 + 127) & ~127;
  s.bytes = s.ring_off + nw * stages * 2 * fp4_record_bytes(d);
  return s;
}

// A position in the tile sequence: tile `tile` of unit `unit` (kv head, column block) of row b.
struct Cursor {
  int b, unit, tile, tiles, units;
};

// a / b for a >= 0, b > 0; the 64-bit division only where it is needed.
__device__ __forceinline__ long long quotient(long long a, int b) {
  return (a >> 32) == 0 ? (long long)(uint32_t(a) / uint32_t(b)) : a / b;
}

// [0, total) cut into n runs whose lengths differ by one at most: where run c begins, and the run of f.
struct Split {
  long long q;
  int r;
  __device__ __forceinline__ Split(long long total, int n) : q(quotient(total, n)), r(int(total - q * n)) {}
  __device__ __forceinline__ long long begin(int c) const { return c * q + min(c, r); }
  __device__ __forceinline__ int run(long long f) const {
    const long long longer = r * (q + 1);  // runs below r have q + 1
    return f < longer ? int(quotient(f, int(q + 1))) : r + int(quotient(f - longer, int(q)));
  }
};

__device__ __forceinline__ unsigned atom_add_acq_rel(unsigned* p, unsigned v) {
  unsigned old;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

template <typename T, int D, int NW>
__global__ void __launch_bounds__(NW * 32, 1)
    pd_fp4_attend_kernel(const __grid_constant__ Fp4AttendParams p, int stages, int max_cols) {
  constexpr int REC = fp4_record_bytes(D);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long warp_sums[2][NW];
  __shared__ int arrival[2][3];  // per cut: last to arrive, first CTA, CTAs
  const Smem L = smem_layout(p.batch, NW, max_cols, D, stages);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long* pre = reinterpret_cast<long long*>(smem + L.pre_off);
  int2* rows = reinterpret_cast<int2*>(smem + L.rows_off);  // (tiles, units) per row
  Piece* pieces = reinterpret_cast<Piece*>(smem + L.piece_off);
  float* piece_ml = reinterpret_cast<float*>(smem + L.ml_off);
  auto piece_acc = [&](int slot) -> float* {  // slot 2 w: warp w's leading piece, 2 w + 1: its trailing one
    return slot & 1 ? reinterpret_cast<float*>(smem + L.ring_off) + size_t(slot >> 1) * stages * (2 * REC / 4)
                    : reinterpret_cast<float*>(smem + L.acc_off) + size_t(slot >> 1) * max_cols * D;
  };
  const uint32_t bars = smem_addr(smem) + uint32_t(warp * stages) * 8u;

  // ---- tiles of every row, their prefix sums, the unit count and the longest row
  long long total, units_total;
  int longest, row, row_unit;  // row and unit of the CTA's unit, where each CTA has one
  bool whole;
  if (lane < stages) mbar_init(bars + lane * 8u, 1);
  if (lane < 2) pieces[2 * warp + lane].row = -1;
  fence_barrier_init();
  auto row_work = [&](int b) -> int2 {
    const Row r = row_of(p, b);
    return make_int2(r.lk > TILE ? (r.lk + TILE - 1) / TILE : 1, p.n_kv_head * ((r.sq * p.group + COLS - 1) / COLS));
  };
  auto up = [&](long long x, int o) -> long long { return __shfl_up_sync(FULL_MASK, x, o); };
  if (p.batch <= 32) {
    // A row to a lane, and every warp for itself: all write the same values, each reads its own, and
    // no barrier is needed.
    const int2 w = lane < p.batch ? row_work(lane) : make_int2(0, 0);
    long long incl = (long long)w.x * w.y;
    int unit_incl = w.y;
    longest = w.y > 0 ? w.x : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long f = up(incl, o);
      const int g = __shfl_up_sync(FULL_MASK, unit_incl, o);
      if (lane >= o) {
        incl += f;
        unit_incl += g;
      }
      longest = max(longest, __shfl_xor_sync(FULL_MASK, longest, o));
    }
    total = __shfl_sync(FULL_MASK, incl, 31);
    units_total = __shfl_sync(FULL_MASK, unit_incl, 31);
    if (lane < p.batch) {
      pre[lane] = incl - (long long)w.x * w.y;
      rows[lane] = w;
    }
    __syncwarp();
    whole = units_total <= gridDim.x && longest <= quotient(total, gridDim.x) + JOIN_TILES;
    row = __ffs(__ballot_sync(FULL_MASK, unit_incl > int(blockIdx.x))) - 1;
    row_unit = int(blockIdx.x) - __shfl_sync(FULL_MASK, unit_incl - w.y, row < 0 ? 0 : row);
  } else {
    const int per = (p.batch + NW * 32 - 1) / (NW * 32);
    const int b0 = tid * per;
    long long sum = 0, usum = 0;
    int most = 0;
    for (int b = b0; b < b0 + per && b < p.batch; ++b) {
      const int2 w = row_work(b);
      rows[b] = w;
      sum += (long long)w.x * w.y;
      usum += w.y;
      most = w.y > 0 && w.x > most ? w.x : most;
    }
    long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long f = up(incl, o);
      if (lane >= o) incl += f;
      usum += __shfl_xor_sync(FULL_MASK, usum, o);
      most = max(most, __shfl_xor_sync(FULL_MASK, most, o));
    }
    if (lane == 31) {
      warp_sums[0][warp] = incl;
      warp_sums[1][warp] = (usum << 31) | most;  // both below 2^31
    }
    __syncthreads();
    long long at = incl - sum;
    total = units_total = 0;
    longest = 0;
#pragma unroll 1
    for (int w = 0; w < NW; ++w) {
      if (w < warp) at += warp_sums[0][w];
      total += warp_sums[0][w];
      units_total += warp_sums[1][w] >> 31;
      longest = max(longest, int(warp_sums[1][w] & 0x7fffffff));
    }
    for (int b = b0; b < b0 + per && b < p.batch; ++b) {
      pre[b] = at;
      at += (long long)rows[b].x * rows[b].y;
    }
    __syncthreads();
    whole = units_total <= gridDim.x && longest <= quotient(total, gridDim.x) + JOIN_TILES;
    row = 0;
    row_unit = int(blockIdx.x);
    if (whole)
      while (row < p.batch && row_unit >= rows[row].y) row_unit -= rows[row++].y;
  }
  if (total == 0) return;

  // ---- this CTA's run of tiles and this warp's part of it
  const long long wanted = whole ? units_total : quotient(total + CTA_TILES - 1, CTA_TILES);
  const int ctas = int(wanted < gridDim.x ? wanted : gridDim.x);
  if (int(blockIdx.x) >= ctas) return;
  const Split split(total, ctas);  // where units are not whole CTAs'
  long long c0, c1;
  if (whole) {
    c0 = pre[row] + (long long)row_unit * rows[row].x;
    c1 = c0 + rows[row].x;
  } else {
    c0 = split.begin(blockIdx.x);
    c1 = split.begin(blockIdx.x + 1);
  }
  const int in_cta = int(c1 - c0);
  const int warps = min(NW, in_cta);
  const int wq = in_cta / warps, wr = in_cta - wq * warps;
  const long long f0 = c0 + warp * wq + min(warp, wr);
  const int count = warp < warps ? wq + (warp < wr ? 1 : 0) : 0;

  if (count > 0) {
    constexpr uint32_t STAGE = 2 * REC;
    const uint32_t ring = smem_addr(smem + L.ring_off) + uint32_t(warp * stages) * STAGE;
    const uint64_t policy = l2_policy_evict_first();
    auto step_unit = [&](Cursor& k) {  // to the next unit's first tile
      k.tile = 0;
      if (++k.unit < k.units) return;
      k.unit = 0;
      do ++k.b; while (k.b < p.batch && rows[k.b].y == 0);
      if (k.b < p.batch) {
        k.tiles = rows[k.b].x;
        k.units = rows[k.b].y;
      }
    };
    Cursor at;
    if (p.batch <= 32) {  // the last row that begins at or before the tile
      at.b = 31 - __clz(__ballot_sync(FULL_MASK, lane < p.batch && pre[lane < p.batch ? lane : 0] <= f0));
    } else {
      int lo = 0, hi = p.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= f0) lo = mid; else hi = mid - 1;
      }
      at.b = lo;
    }
    {
      const long long r = f0 - pre[at.b];
      at.tiles = rows[at.b].x;
      at.units = rows[at.b].y;
      at.unit = int(quotient(r, at.tiles));
      at.tile = int(r - (long long)at.unit * at.tiles);
    }

    // ---- prefetch: tile `ahead`. Lane l holds the address of the unit's page win_page + l (this head's
    // records of it) and issues that page's copies itself; the block ids of the next 32 pages are
    // already loading. A window starts at a tile's first page, so a tile's two pages (block_size
    // 16) are in one window.
    Cursor ahead = at;
    const unsigned char* page_at = nullptr;
    int id_next = 0, win_page = 0, last_page = 0, records = 0;
    unsigned dead = 0;  // pages of the window that are outside the pool, or past the row
    const unsigned char* head_pages = nullptr;  // this head's first record of block 0
    const uint32_t block_stride = uint32_t(p.n_kv_head << p.log2_tpb) * REC;
    auto entry = [&](int page) -> int {
      return page <= last_page ? __ldg(p.table + int64_t(ahead.b) * p.bt_stride + page) : -1;
    };
    auto open_window = [&](int id) {  // the window at win_page, whose block ids are `id`
      const bool live = id >= 0 && id < p.n_blocks;
      page_at = head_pages + (live ? uint64_t(id) * block_stride : 0);
      dead = __ballot_sync(FULL_MASK, !live);
      id_next = entry(win_page + 32 + lane);
    };
    auto open_ahead = [&]() {
      const int h = ahead.unit / (ahead.units / p.n_kv_head);
      head_pages = p.pages + (int64_t(h) << p.log2_tpb) * REC;
      records = (row_of(p, ahead.b).lk + FP4_TILE - 1) / FP4_TILE;
      last_page = min(((records + (1 << p.log2_tpb) - 1) >> p.log2_tpb), p.max_blocks) - 1;
      win_page = (2 * ahead.tile) >> p.log2_tpb;
      open_window(entry(win_page + lane));
    };
    open_ahead();
    int issued = 0;
    uint32_t fill = 0;  // stage of the next copy
    auto issue = [&]() {
      if (issued == count) return;
      const int rec = 2 * ahead.tile;
      int page = (rec >> p.log2_tpb) - win_page;
      if (page >= 32) {
        win_page += 32;
        page -= 32;
        open_window(id_next);
      }
      const uint32_t dst = ring + fill * STAGE, bar = bars + fill * 8u;
      const bool two = rec + 1 < records;
      const unsigned needs = two && p.log2_tpb == 0 ? 3u : 1u;
      if (((dead >> page) & needs) == 0) {
        // the page's lane announces the bytes and copies; with one record to a page, the next lane copies
        // the second (its bytes may be counted before they are announced: the phase waits for the
        // announcing arrival)
        const int mine = lane - page;
        if (mine == 0) mbar_arrive_expect_tx(bar, two ? STAGE : REC);
        if (p.log2_tpb == 0) {
          if (mine == 0 || (mine == 1 && two)) bulk_load(dst + mine * REC, page_at, REC, bar, policy);
        } else if (mine == 0) {  // both records in one page, one after the other
          bulk_load(dst, page_at + (rec & ((1 << p.log2_tpb) - 1)) * REC, two ? STAGE : REC, bar, policy);
        }
      } else {  // a block outside the pool reads zeros
        const int in_page = rec & ((1 << p.log2_tpb) - 1);
#pragma unroll 1
        for (int r = 0; r < 2; ++r) {
          const int holder = p.log2_tpb == 0 ? (page + r) & 31 : page;
          const uint64_t at64 = __shfl_sync(FULL_MASK, reinterpret_cast<uint64_t>(page_at), holder);
          const bool live = (r == 0 || two) && !((dead >> holder) & 1u);
          const uint4* src = reinterpret_cast<const uint4*>(at64) + (p.log2_tpb == 0 ? 0 : (in_page + r) * (REC / 16));
          for (int i = lane; i < REC / 16; i += 32) {
            const uint4 v = live ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + r * REC + i * 16), "r"(v.x), "r"(v.y),
                         "r"(v.z), "r"(v.w)
                         : "memory");
          }
        }
        fence_proxy_async_smem();  // a later bulk copy writes the same bytes
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
      }
      fill = fill + 1 == uint32_t(stages) ? 0 : fill + 1;
      ++issued;
      if (++ahead.tile == ahead.tiles && issued < count) {
        step_unit(ahead);
        open_ahead();
      }
    };
    for (int s = 0; s < stages - 1; ++s) issue();

    Worker<T, D> wk;
    wk.init(lane);
    uint32_t stage = 0, phase = 0;
    int taken = 0;
    bool ok = true;
    for (int n = 0; n < count;) {
      const Row r = row_of(p, at.b);
      const int cbs = at.units / p.n_kv_head;
      const int h = at.unit / cbs, first = (at.unit - h * cbs) * COLS;
      const int begin = at.tile, end = min(at.tiles, at.tile + count - n);
      wk.start(p, r, h, first);
      for (int tile = begin; tile < end; ++tile) {
        if (ok && !warp_wait_phase(bars + stage * 8u, phase, p.wait_ns)) {
          ok = false;  // the rest of the run is left out; its pieces and arrivals still happen
          if (lane == 0) atomicOr(p.err, DEVERR_WAIT_TIMEOUT);
        }
        if (!ok) continue;
        __syncwarp();  // every lane is done with the stage that the next copy fills
        issue();
        wk.tile(ring + stage * STAGE, tile * TILE, r.lk - tile * TILE);
        ++taken;
        if (++stage == uint32_t(stages)) {
          stage = 0;
          phase ^= 1u;
        }
      }
      n += end - begin;
      if (begin == 0 && end == at.tiles) {
        wk.finish(p, r, h, first);
      } else {
        const int slot = 2 * warp + (begin == 0 ? 1 : 0);
        wk.store_piece(piece_ml + slot * 2 * COLS, piece_acc(slot), min(COLS, r.sq * p.group - first));
        if (lane == 0)
          pieces[slot] = Piece{at.b, at.unit, begin, end, at.tiles, h, first, min(COLS, r.sq * p.group - first), r.q_begin, {}};
      }
      if (n < count) step_unit(at);
    }
    if (!ok) {  // never leave with a copy in flight: stages in the order of their copies
      for (; taken < issued; ++taken) {
        warp_wait_phase(bars + stage * 8u, phase, DRAIN_LIMIT_NS);
        if (++stage == uint32_t(stages)) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  }

  // ---- joins within the CTA
  __syncthreads();
  static_assert(2 * NW <= 32, "one lane per piece");
  int2 mine = make_int2(-1, 0);
  if (lane < 2 * NW) mine = make_int2(pieces[lane].row, pieces[lane].unit);
  const unsigned valid = __ballot_sync(FULL_MASK, mine.x >= 0);
  if (valid == 0) return;  // uniform over the CTA
  const unsigned below = valid & ((1u << lane) - 1u);
  const int prev = below ? 31 - __clz(below) : lane;
  const int prev_row = __shfl_sync(FULL_MASK, mine.x, prev), prev_unit = __shfl_sync(FULL_MASK, mine.y, prev);
  unsigned heads =
      __ballot_sync(FULL_MASK, mine.x >= 0 && (below == 0 || prev_row != mine.x || prev_unit != mine.y));
  float* const cta_part = p.partials + size_t(blockIdx.x) * 2 * partial_floats(D);
  int task = 0;
  int cut0 = -1, cut1 = -1;  // first piece of the unit cut at the CTA's front, and at its back
#pragma unroll 1
  while (heads) {
    const int s0 = __ffs(heads) - 1;
    heads &= heads - 1;
    const unsigned upto = heads ? (1u << (__ffs(heads) - 1)) - 1u : 0xffffffffu;
    const unsigned members = valid & upto & ~((1u << s0) - 1u);
    const Piece a = pieces[s0];
    const bool complete = a.t0 == 0 && pieces[31 - __clz(members)].t1 == a.tiles;
    const int slot = a.t0 > 0 ? 0 : 1;
    if (!complete) {
      if (slot == 0) cut0 = s0; else cut1 = s0;
    }
    const int n = __popc(members), chunks = (a.cols * D + 127) / 128;
    // chunk c of the group is task + c: this warp's are those that leave remainder `warp`
#pragma unroll 1
    for (int ch = (warp - task % NW + NW) % NW; ch < chunks; ch += NW) {
      const int e = ch * 128 + lane * 4;
      if (e >= a.cols * D) continue;
      const int col = e / D;
      float x[4], m, l;
      // after the first piece, each further one is the next warp's leading piece
      auto index = [&](int i) -> int { return i == 0 ? s0 : 2 * ((s0 >> 1) + i); };
      join4(n, col, [&](int i) { return piece_ml + index(i) * 2 * COLS; },
            [&](int i) { return *reinterpret_cast<const float4*>(piece_acc(index(i)) + e); }, x, m, l);
      if (complete) {
        store_out4<T>(p, a, col, e - col * D, x, l);
      } else {
        float* part = cta_part + slot * partial_floats(D);
        if (e % D == 0) {
          part[col] = m;
          part[COLS + col] = l;
        }
        *reinterpret_cast<float4*>(part + 2 * COLS + e) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
    task += chunks;
  }
  if (cut0 < 0 && cut1 < 0) return;  // uniform

  // ---- joins between CTAs: the last one to arrive at a unit joins its partials, in CTA order. One
  // thread arrives for each cut; the barrier before it puts the CTA's stores ahead of its release.
  __syncthreads();
  if (lane == 0 && warp < 2) {
    const int at = warp == 0 ? cut0 : cut1;
    int last = 0;
    if (at >= 0) {
      const Piece& a = pieces[at];
      const long long u0 = pre[a.row] + (long long)a.unit * a.tiles;
      const int cta0 = split.run(u0), n = split.run(u0 + a.tiles - 1) - cta0 + 1;
      last = atom_add_acq_rel(p.counters + cta0, 1u) == unsigned(n - 1);
      if (last) p.counters[cta0] = 0u;  // zero again for the next launch
      arrival[warp][1] = cta0;
      arrival[warp][2] = n;
    }
    arrival[warp][0] = last;
  }
  __syncthreads();
#pragma unroll 1
  for (int s = 0; s < 2; ++s) {
    if (!arrival[s][0]) continue;
    const Piece a = pieces[s == 0 ? cut0 : cut1];
    const int cta0 = arrival[s][1], n = arrival[s][2];
    // the cuts' elements side by side: the second's on the threads that the first's leave
    for (int e = ((tid + (s == 0 ? 0 : NW * 16)) % (NW * 32)) * 4; e < a.cols * D; e += NW * 128) {
      const int col = e / D;
      float x[4], m, l;
      auto part = [&](int i) -> const float* {  // the first CTA's is its unit that goes on, the others' their first
        return p.partials + (size_t(cta0 + i) * 2 + (i == 0 ? 1 : 0)) * partial_floats(D);
      };
      join4(n, col, part,
            [&](int i) { return __ldcg(reinterpret_cast<const float4*>(part(i) + 2 * COLS + e)); }, x, m, l);
      store_out4<T>(p, a, col, e - col * D, x, l);
    }
  }
}

}  // namespace fp4

}  // namespace pd
