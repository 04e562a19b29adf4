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
//  * P enters as fp16 (2^-12 relative, on weights whose sum is kept unrounded in fp32): below half
//    an ulp of the 16-bit result.
//  * tokens past the row are masked to P = 0 and their V scales to 0, so whatever bytes a page
//    holds there (a NaN scale included) never reaches the sums.
//
// Work split: the (row, kv head, column block, record) sequence is cut into equal runs, one per
// warp, so every SM streams the same number of bytes whatever the lengths. Each warp prefetches
// its run through a ring of records in shared memory (cp.async, no barrier shared with other
// warps). A unit (row, kv head, column block) cut between warps leaves partial (m, l, acc) pieces:
// the CTA joins its own in shared memory; a unit cut between CTAs goes through the workspace and
// the last CTA to arrive joins it, in piece order whoever arrives last, so results do not depend
// on timing. Nothing waits: a CTA that is not last leaves.
#pragma once

#include "pd_fp4.cuh"
#include "pd_internal.h"

namespace pd {

namespace fp4 {

constexpr int MAX_ROWS = 1024;  // rows of one launch (their prefix sums are in shared memory)
constexpr int COLS = 8;         // columns of a unit

// Floats of one CTA-level partial: m and l of 8 columns, then 8 x D accumulators.
__host__ __device__ constexpr int partial_floats(int d) { return 2 * COLS + COLS * d; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  const int n = live ? 16 : 0;  // 0: fills with zeros, reads nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

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
  float m_run[2], l_run[2];
  float mul[2];  // score multiplier of columns 2c, 2c + 1
  int lim[2];    // their last visible key

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
    // 2^(13 - floor(log2 top)), within 2^+-100; 1 for zero and for non-finite columns
    int e = int(__float_as_uint(top) >> 23);
    e = e == 0 || e == 255 ? 140 : e;
    int shift = 140 - e;
    shift = shift > 100 ? 100 : (shift < -100 ? -100 : shift);
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
      m_run[j] = -INFINITY;
      l_run[j] = 0.f;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) o[m][0] = o[m][1] = o[m][2] = o[m][3] = 0.f;
  }

  // One record at shared address `a`; its first token is key `t0`, `rows` of its tokens exist.
  __device__ __forceinline__ void tile(uint32_t a, int t0, int rows) {
    float acc[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[0][i] = acc[1][i] = 0.f;
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
        X::m16n8k16(acc[0], x[0], y[0], x[1], y[1], qb[ks][0], qb[ks][1]);
        X::m16n8k16(acc[1], x[2], y[2], x[3], y[3], qb[ks + 1][0], qb[ks + 1][1]);
      }
    }
    float s[4];
    bool exceeds = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = i & 1, t = t0 + g + 8 * (i >> 1);
      s[i] = t <= lim[j] ? (acc[0][i] + acc[1][i]) * mul[j] : -INFINITY;
      exceeds |= s[i] > m_run[j];
    }
    if (__any_sync(FULL_MASK, exceeds)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float t = fmaxf(s[j], s[2 + j]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) t = fmaxf(t, __shfl_xor_sync(FULL_MASK, t, off));
        t = fmaxf(t, m_run[j]);
        const float alpha = t == -INFINITY ? 1.f : exp2f(m_run[j] - t);
        m_run[j] = t;
        l_run[j] *= alpha;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          o[m][j] *= alpha;
          o[m][2 + j] *= alpha;
        }
      }
    }
    float pr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = i & 1;
      pr[i] = s[i] == -INFINITY ? 0.f : exp2f(s[i] - m_run[j]);
      l_run[j] += pr[i];
    }
    const uint32_t pb0 = movmatrix_trans(Elem<__half>::pack2(pr[0], pr[1]));
    const uint32_t pb1 = movmatrix_trans(Elem<__half>::pack2(pr[2], pr[3]));
    // V scales of tokens 2c, 2c + 1 and 2c + 8, 2c + 9; zero past the row
    uint32_t keep[2];
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int t = 8 * hi + 2 * c;
      keep[hi] = (t < rows ? 0x0000ffffu : 0u) | (t + 1 < rows ? 0xffff0000u : 0u);
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
          X::m16n8k16(o[b * 8 + u * 4 + i], even[0][i], odd[0][i], even[1][i], odd[1][i], pb0, pb1);
      }
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

// A partial unit of this CTA: records [t0, t1) of unit `unit` (kv head, column block) of row b.
struct Piece {
  int row, unit, t0, t1;  // row < 0: none
};

// Joins `n` pieces' four elements of column col: ml(i) is piece i's (m, l) block, acc(i) its elements.
template <typename Ml, typename Acc>
__device__ __forceinline__ void join4(int n, int col, Ml ml, Acc acc, float (&x)[4], float& m, float& l) {
  m = -INFINITY;
  for (int i = 0; i < n; ++i) m = fmaxf(m, ml(i)[col]);
  l = 0.f;
  x[0] = x[1] = x[2] = x[3] = 0.f;
  if (m == -INFINITY) return;
  for (int i = 0; i < n; ++i) {
    const float f = exp2f(ml(i)[col] - m);
    const float4 v = acc(i);
    l = fmaf(f, ml(i)[COLS + col], l);
    x[0] = fmaf(f, v.x, x[0]);
    x[1] = fmaf(f, v.y, x[1]);
    x[2] = fmaf(f, v.z, x[2]);
    x[3] = fmaf(f, v.w, x[3]);
  }
}

template <typename T>
__device__ __forceinline__ void store_out4(const Fp4AttendParams& p, const Row& r, int h, int n, int e, float unit,
                                           const float (&x)[4], float l) {
  const float inv = l > 0.f ? unit / l : 0.f;
  const int tok = n / p.group, hg = n - tok * p.group;
  T* dst = reinterpret_cast<T*>(p.out) + int64_t(r.q_begin + tok) * p.o_st + int64_t(h * p.group + hg) * p.o_sh + e;
  *reinterpret_cast<uint2*>(dst) =
      make_uint2(Elem<T>::pack2(x[0] * inv, x[1] * inv), Elem<T>::pack2(x[2] * inv, x[3] * inv));
}

// Shared memory: [prefix int64 (rows + 1) | records and units per row | pieces | piece (m, l) |
// piece accumulators (2 NW x cols x D) | rings (NW x stages x record)].
struct Smem {
  int rows_off, piece_off, ml_off, acc_off, ring_off, bytes;
};

__host__ __device__ inline Smem smem_layout(int batch, int nw, int cols, int d, int stages) {
  Smem s;
  s.rows_off = (batch + 1) * 8;
  s.piece_off = (s.rows_off + batch * 8 + 15) & ~15;
  s.ml_off = s.piece_off + 2 * nw * int(sizeof(Piece));
  s.acc_off = s.ml_off + 2 * nw * 2 * COLS * 4;
  s.ring_off = (s.acc_off + 2 * nw * cols * d * 4 + 127) & ~127;
  s.bytes = s.ring_off + nw * stages * fp4_record_bytes(d);
  return s;
}

template <typename T, int D, int NW>
__global__ void __launch_bounds__(NW * 32, 1)
    pd_fp4_attend_kernel(const __grid_constant__ Fp4AttendParams p, int stages, int max_cols, int min_records) {
  constexpr int REC = fp4_record_bytes(D);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long warp_sums[NW];
  __shared__ unsigned last_flags[2];
  const Smem L = smem_layout(p.batch, NW, max_cols, D, stages);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  long long* pre = reinterpret_cast<long long*>(smem);
  int2* rows = reinterpret_cast<int2*>(smem + L.rows_off);  // (records, units) per row
  Piece* pieces = reinterpret_cast<Piece*>(smem + L.piece_off);
  float* piece_ml = reinterpret_cast<float*>(smem + L.ml_off);
  float* piece_acc = reinterpret_cast<float*>(smem + L.acc_off);

  // ---- records of every row, and their prefix sums
  {
    const int per = (p.batch + NW * 32 - 1) / (NW * 32);
    const int b0 = tid * per;
    long long sum = 0;
    for (int b = b0; b < b0 + per && b < p.batch; ++b) {
      const Row r = row_of(p, b);
      const int records = r.lk > FP4_TILE ? (r.lk + FP4_TILE - 1) / FP4_TILE : 1;
      const int units = p.n_kv_head * ((r.sq * p.group + COLS - 1) / COLS);
      rows[b] = make_int2(records, units);
      sum += (long long)records * units;
    }
    long long incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(FULL_MASK, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sums[warp] = incl;
    if (tid < 2 * NW) pieces[tid].row = -1;
    __syncthreads();
    long long at = incl - sum;
    for (int w = 0; w < warp; ++w) at += warp_sums[w];
    for (int b = b0; b < b0 + per && b < p.batch; ++b) {
      pre[b] = at;
      at += (long long)rows[b].x * rows[b].y;
      if (b == p.batch - 1) pre[p.batch] = at;
    }
    __syncthreads();
  }
  const long long total = pre[p.batch];
  if (total == 0) return;
  // Warps with work: all of them, unless that leaves a warp fewer than min_records.
  const long long all = (long long)gridDim.x * NW;
  long long active = (total + min_records - 1) / min_records;
  active = active < all ? active : all;
  const long long me = (long long)blockIdx.x * NW + warp;
  if ((long long)blockIdx.x * NW >= active) return;
  auto begin_of = [&](long long w) -> long long { return w >= active ? total : w * total / active; };
  auto find_row = [&](long long f) -> int {  // last b with pre[b] <= f that has work
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= f) lo = mid; else hi = mid - 1;
    }
    return lo;
  };

  const long long f0 = begin_of(me), f1 = begin_of(me + 1);
  const int count = int(f1 - f0);
  if (count > 0) {
    const uint32_t ring = smem_addr(smem + L.ring_off) + uint32_t(warp * stages) * REC;
    const int tpb_mask = (1 << p.log2_tpb) - 1;
    // Lookup cursor: the record whose block id is being fetched; one record ahead of the copies.
    struct Cursor {
      int b, unit, rec, records, units;
    };
    auto place = [&](Cursor& k, long long f) {
      k.b = find_row(f);
      const long long r = f - pre[k.b];
      k.records = rows[k.b].x;
      k.units = rows[k.b].y;
      k.unit = int(r / k.records);
      k.rec = int(r - (long long)k.unit * k.records);
    };
    auto step = [&](Cursor& k) {
      if (++k.rec < k.records) return;
      k.rec = 0;
      if (++k.unit < k.units) return;
      k.unit = 0;
      do ++k.b; while (k.b < p.batch && rows[k.b].y == 0);
      if (k.b < p.batch) {
        k.records = rows[k.b].x;
        k.units = rows[k.b].y;
      }
    };
    Cursor look, at;
    place(look, f0);
    at = look;
    int next_blk = -1, next_sub = 0;
    int looked = 0;
    auto lookup = [&]() {
      if (looked >= count) return;
      const int page = look.rec >> p.log2_tpb;
      const int cbs = look.units / p.n_kv_head;
      next_sub = ((look.unit / cbs) << p.log2_tpb) + (look.rec & tpb_mask);
      next_blk = page < p.max_blocks ? __ldg(p.table + int64_t(look.b) * p.bt_stride + page) : -1;
      ++looked;
      step(look);
    };
    lookup();
    int issued = 0;
    auto issue = [&]() {
      if (issued < count) {
        const bool live = next_blk >= 0 && next_blk < p.n_blocks;
        const unsigned char* src =
            p.pages + (((live ? int64_t(next_blk) : 0) * p.n_kv_head << p.log2_tpb) + next_sub) * REC;
        const uint32_t dst = ring + uint32_t(issued % stages) * REC;
        lookup();
#pragma unroll
        for (int i = 0; i < (REC / 16 + 31) / 32; ++i) {
          const int ch = i * 32 + lane;
          if (ch < REC / 16) cp_async16(dst + ch * 16, src + (live ? ch * 16 : 0), live);
        }
        ++issued;
      }
      cp_async_commit();
    };
    for (int s = 0; s < stages - 1; ++s) issue();

    Worker<T, D> wk;
    wk.init(lane);
    Row row{};
    int h = 0, first = 0, t_begin = 0;
    for (int n = 0; n < count; ++n) {
      if (n == 0 || at.rec == 0) {  // a unit opens
        row = row_of(p, at.b);
        const int cbs = at.units / p.n_kv_head;
        h = at.unit / cbs;
        first = (at.unit - h * cbs) * COLS;
        t_begin = at.rec;
        wk.start(p, row, h, first);
      }
      // record n has landed once at most stages - 2 later groups are pending
      switch (stages) {
        case 2: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 3: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 4: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        case 5: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
      }
      __syncwarp();  // every lane's bytes are in, and every lane is done with the stage refilled next
      issue();
      const int t0 = at.rec * FP4_TILE;
      wk.tile(ring + uint32_t(n % stages) * REC, t0, row.lk - t0);
      const bool unit_ends = at.rec + 1 == at.records;
      if (unit_ends || n == count - 1) {
        if (unit_ends && t_begin == 0) {
          wk.finish(p, row, h, first);
        } else {
          const int slot = 2 * warp + (t_begin == 0 ? 1 : 0);
          const int cols = min(COLS, row.sq * p.group - first);
          wk.store_piece(piece_ml + slot * 2 * COLS, piece_acc + size_t(slot) * max_cols * D, cols);
          if (lane == 0) {
            Piece pc;
            pc.row = at.b;
            pc.unit = at.unit;
            pc.t0 = t_begin;
            pc.t1 = at.rec + 1;
            pieces[slot] = pc;
          }
        }
      }
      step(at);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }

  // ---- joins within the CTA
  __syncthreads();
  static_assert(2 * NW <= 32, "one lane per piece");
  Piece mine{-1, 0, 0, 0};
  if (lane < 2 * NW) mine = pieces[lane];
  const unsigned valid = __ballot_sync(FULL_MASK, mine.row >= 0);
  if (valid == 0) return;  // uniform over the CTA
  const unsigned below = valid & ((1u << lane) - 1u);
  const int prev = below ? 31 - __clz(below) : lane;
  const int prev_row = __shfl_sync(FULL_MASK, mine.row, prev), prev_unit = __shfl_sync(FULL_MASK, mine.unit, prev);
  const bool opens = mine.row >= 0 && (below == 0 || prev_row != mine.row || prev_unit != mine.unit);
  unsigned heads = __ballot_sync(FULL_MASK, opens);
  float* const cta_part = p.partials + size_t(blockIdx.x) * 2 * partial_floats(D);
  int task = 0;
  bool cut[2] = {false, false};
  Piece cut_piece[2] = {};
  while (heads) {
    const int s0 = __ffs(heads) - 1;
    heads &= heads - 1;
    const unsigned upto = heads ? (1u << (__ffs(heads) - 1)) - 1u : 0xffffffffu;
    const unsigned members = valid & upto & ~((1u << s0) - 1u);
    const int s1 = 31 - __clz(members);
    const Piece a = pieces[s0], z = pieces[s1];
    const bool complete = a.t0 == 0 && z.t1 == rows[a.row].x;
    const Row r = row_of(p, a.row);
    const int cbs = rows[a.row].y / p.n_kv_head;
    const int h = a.unit / cbs, first = (a.unit - h * cbs) * COLS;
    const int cols = min(COLS, r.sq * p.group - first);
    const int slot = a.t0 > 0 ? 0 : 1;
    if (!complete) {
      cut[slot] = true;
      cut_piece[slot] = a;
    }
    const float unit = p.units != nullptr ? __ldg(p.units + p.n_kv_head + h) : 1.f;
    const int n = __popc(members);
    for (int ch = 0; ch * 128 < cols * D; ++ch, ++task) {
      if (task % NW != warp) continue;
      const int e = ch * 128 + lane * 4;
      if (e >= cols * D) continue;
      const int col = e / D;
      float x[4], m, l;
      // after the first piece, each further one is the next warp's leading piece
      auto index = [&](int i) -> int { return i == 0 ? s0 : 2 * ((s0 >> 1) + i); };
      join4(n, col, [&](int i) { return piece_ml + index(i) * 2 * COLS; },
            [&](int i) { return *reinterpret_cast<const float4*>(piece_acc + size_t(index(i)) * max_cols * D + e); }, x,
            m, l);
      if (complete) {
        store_out4<T>(p, r, h, first + col, e - col * D, unit, x, l);
      } else {
        float* part = cta_part + slot * partial_floats(D);
        if (e % D == 0) {
          part[col] = m;
          part[COLS + col] = l;
        }
        *reinterpret_cast<float4*>(part + 2 * COLS + e) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
  }
  if (!cut[0] && !cut[1]) return;  // uniform

  // ---- joins between CTAs: the last one to arrive at a unit joins its partials, in CTA order
  __threadfence();
  __syncthreads();
  int cta0[2] = {0, 0}, n_cta[2] = {0, 0};
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (!cut[s]) continue;
    const long long u0 = pre[cut_piece[s].row] + (long long)cut_piece[s].unit * rows[cut_piece[s].row].x;
    const long long u1 = u0 + rows[cut_piece[s].row].x - 1;
    // the warp of record f: the largest w with w * total / active <= f
    cta0[s] = int((((u0 + 1) * active + total - 1) / total - 1) / NW);
    n_cta[s] = int((((u1 + 1) * active + total - 1) / total - 1) / NW) - cta0[s] + 1;
    if (tid == 0) {
      const unsigned old = atomicAdd(p.counters + cta0[s], 1u);
      last_flags[s] = old == unsigned(n_cta[s] - 1);
      if (last_flags[s]) p.counters[cta0[s]] = 0u;  // zero again for the next launch
    }
  }
  __threadfence();
  __syncthreads();
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (!cut[s] || !last_flags[s]) continue;
    const Piece a = cut_piece[s];
    const Row r = row_of(p, a.row);
    const int cbs = rows[a.row].y / p.n_kv_head;
    const int h = a.unit / cbs, first = (a.unit - h * cbs) * COLS;
    const int cols = min(COLS, r.sq * p.group - first);
    const float unit = p.units != nullptr ? __ldg(p.units + p.n_kv_head + h) : 1.f;
    const int n = n_cta[s];
    for (int e = tid * 4; e < cols * D; e += NW * 128) {
      const int col = e / D;
      float x[4], m, l;
      auto part = [&](int i) -> const float* {  // the first CTA's is its unit that goes on, the others' their first
        return p.partials + (size_t(cta0[s] + i) * 2 + (i == 0 ? 1 : 0)) * partial_floats(D);
      };
      join4(n, col, part,
            [&](int i) { return __ldcg(reinterpret_cast<const float4*>(part(i) + 2 * COLS + e)); }, x, m, l);
      store_out4<T>(p, r, h, first + col, e - col * D, unit, x, l);
    }
  }
}

}  // namespace fp4

}  // namespace pd
