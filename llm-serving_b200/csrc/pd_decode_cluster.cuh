// pd_decode_cluster.cuh -- paged GQA decode of few rows for sm_100a: windows and attention weights, head_dim 64..256;
// bf16 / fp16 in blocks of at least 8 tokens, fp32 in any.
//
// The function of pd_decode_kernel.cuh's variants where that kernel's start costs more than its work: with so few
// (row, kv head, q-head chunk) items that all their CTAs run at once, nothing has to be dealt. A cluster of `split` CTAs
// takes one item and each of its warps an even run of the row's visible tiles (VisibleTiles), through a TMA
// ring of its own into the tensor-core consumer of pd_decode_mma.cuh (fp32: pd_decode_fma.cuh). The warps' (m, l, acc) meet in shared memory
// and the CTAs' in distributed shared memory: no workspace, no counter, no second pass over global memory. With
// weights (LOG) the scores wait in shared memory until the row's m and l are known, and are added in the same launch
// (one q-head chunk per kv head, so that a sum has one writer).
//
// Bound by latency: length, block ids, tiles, merge, each a round trip; every warp's first loads go out before it
// waits for anything. One row, 8 kv heads of 128, a window of 1024: 6.2 us in a graph of such calls, of which 4 are its
// 4 MB's round trips and 2 the merge (0.65 would move the bytes), 7.4 launched one by one; with weights over 700 tokens
// 7.7 either way. 61 rows of 2 kv heads of 256, windows of 777: 23.4 and 24.4 us, 95 MB at 4.1 TB/s: the longest rows'
// runs of 13 tiles a warp.
#pragma once

#include "pd_decode_fma.cuh"
#include "pd_decode_kernel.cuh"

namespace pd {

// Tile math: tensor cores for 16-bit K/V, multiply-adds for fp32; scores and normalisers that a lane holds.
template <typename T, int D, int GT>
struct ClusterMath {
  using W = MmaWorker<T, D, GT>;
  static constexpr int R = MmaCfg<T, D, GT>::R, L = 2;
};
template <int D, int GT>
struct ClusterMath<float, D, GT> {
  using W = FmaWorker<D, GT>;
  static constexpr int R = W::R, L = GT;
};

// W warps a CTA: eight of one CTA on an SM, or four of two, so that more items run at once.
template <typename T, int D, int GT, bool LOG, int W>
__global__ void __launch_bounds__(W * 32, 8 / W)
    pd_decode_cluster_kernel(const __grid_constant__ DecodeParams p, const __grid_constant__ ClusterDecode c,
                             const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using C = DecodeCfg<T, D, GT>;
  using E = Elem<T>;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ float s_m[W][GT], s_l[W][GT];           // the warps'
  __shared__ __align__(16) float s_cta[2 * GT];      // the CTA's m, then l
  __shared__ float s_final[2][GT];                   // the row's m and 1 / l
  __shared__ __align__(16) float s_acc[GT * D];      // the CTA's accumulators
  __shared__ __align__(8) uint64_t s_bars[W * 4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int S = p.stages;
  const uint32_t base = smem_addr(smem);
  const uint32_t stages_off = (((base + uint32_t(c.scores_bytes) + 1023u) & ~1023u) - base) + uint32_t(warp * S * C::STAGE_BYTES);
  unsigned char* const my_stages = smem + stages_off;
  const uint32_t stages_addr = base + stages_off;
  float* const my_scores = reinterpret_cast<float*>(smem) + warp * (c.scores_bytes / (4 * W));
  uint64_t* const my_bars = s_bars + warp * 4;
  if (lane == 0) {
    for (int s = 0; s < S; ++s) mbar_init(smem_addr(my_bars + s), 1);
    fence_barrier_init();
    if (warp == 0) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
    }
  }
  __syncwarp();
  griddep_wait();
  griddep_launch_dependents();

  const int split = 1 << c.log2_split, rank = int(blockIdx.x) & (split - 1);
  const int item = int(blockIdx.x) >> c.log2_split;
  const int gc = item % p.n_gchunks, h = item / p.n_gchunks % p.n_kv_head, b = item / p.n_gchunks / p.n_kv_head;
  const int heads = min(GT, p.group - gc * GT), hq0 = h * p.group + gc * GT;
  int len = __ldg(p.seqlen + b);
  len = len < 0 ? 0 : (len > p.capacity ? p.capacity : len);
  const VisibleTiles<C::LOG_TILE> vis(p.window, p.sinks);
  const int ntile = vis.count(len);
  const int workers = split * W, g = rank * W + warp;
  const int t0 = int(int64_t(g) * ntile / workers), t1 = int(int64_t(g + 1) * ntile / workers), n = t1 - t0;
  auto tile_token = [&](int k) -> int { return vis.row_tile(t0 + k, len) << C::LOG_TILE; };
  auto live_of = [&](int k) -> LiveWindow {
    const int tok0 = tile_token(k), rows = len - tok0, lo = vis.first(len) - tok0, sk = vis.sinks - tok0;
    return LiveWindow{rows, lo, sk, rows >= C::TILE && (lo <= 0 || sk >= C::TILE)};
  };

  // Block ids of the run's copies, 32 at a time: entry e is copy e % nbox of tile e / nbox.
  const int log2_nbox = C::LOG_TILE - p.log2_box, nbox = 1 << log2_nbox;
  const int32_t* trow = p.table + int64_t(b) * p.bt_stride;
  auto window_of = [&](int first) -> int {
    const int e = first + lane, k = e >> log2_nbox;
    if (k >= n) return 0;
    const int tok = tile_token(k) + ((e & (nbox - 1)) << p.log2_box), page = tok >> p.log2_bs;
    return tok < len && page < p.max_blocks ? __ldg(trow + page) : 0;
  };
  int win = window_of(0), win_at = 0;
  const uint64_t kv_policy = l2_policy_evict_first();
  const uint32_t box_bytes = uint32_t(p.box_tokens) * uint32_t(C::ROW_BYTES);
  auto issue = [&](int k, int s) {
    const int tok0 = tile_token(k);
    const int nvalid = min(nbox, (len - tok0 + p.box_tokens - 1) >> p.log2_box);
    const uint32_t full = smem_addr(my_bars + s), kdst = stages_addr + uint32_t(s * C::STAGE_BYTES);
    if ((k << log2_nbox) >= win_at + 32) {
      win_at += 32;
      win = window_of(win_at);
    }
    if (lane == 0) mbar_arrive_expect_tx(full, 2u * uint32_t(nvalid) * box_bytes);
    for (int j = 0; j < nvalid; ++j) {
      const int blk = __shfl_sync(FULL_MASK, win, ((k << log2_nbox) + j) & 31);
      if (lane == 0) {
        const int off = (tok0 + (j << p.log2_box)) & (p.block_size - 1);
        const uint32_t at = kdst + j * box_bytes;
        if constexpr (sizeof(T) == 4) {
          tma_load_4d_hint(at, &kmap, full, 0, h, off, blk, kv_policy);
          tma_load_4d_hint(at + uint32_t(C::TILE_BYTES), &vmap, full, 0, h, off, blk, kv_policy);
        } else {
          tma_load_5d_hint(at, &kmap, full, 0, off, h, 0, blk, kv_policy);
          tma_load_5d_hint(at + uint32_t(C::TILE_BYTES), &vmap, full, 0, off, h, 0, blk, kv_policy);
        }
      }
    }
  };
  int issued = 0;
  for (; issued < min(n, S); ++issued) issue(issued, issued);
  using M = ClusterMath<T, D, GT>;
  typename M::W mw;
  mw.init(lane, p.box_tokens, p.log2_box);
  mw.start(reinterpret_cast<const T*>(p.q) + int64_t(b) * p.q_sb, p.q_sh, hq0, heads);

  bool ok = true;
  if (n > 0) {
    float sc_cur[M::R], sc_nxt[M::R];
    auto wait = [&](int k) -> bool {
      return warp_wait_phase(smem_addr(my_bars + k % S), uint32_t(k / S) & 1u, p.wait_ns);
    };
    ok = wait(0);
    if (ok) mw.scores(stages_addr, live_of(0), p.scale_log2, sc_cur);
    for (int k = 0; ok && k < n; ++k) {
      const int s = k % S;
      if (k + 1 < n && !wait(k + 1)) {
        ok = false;
        break;
      }
      const LiveWindow live = live_of(k);
      mw.max_update(sc_cur);
      // the next tile's scores and this one's P V are independent chains
      if (k + 1 < n)
        mw.scores(stages_addr + uint32_t((k + 1) % S * C::STAGE_BYTES), live_of(k + 1), p.scale_log2, sc_nxt);
      if constexpr (LOG) mw.store_scores(my_scores + k * (C::TILE * GT), GT, GT, live, sc_cur);
      mw.pv(stages_addr + uint32_t(s * C::STAGE_BYTES + C::TILE_BYTES), sc_cur, live, live.full);
      __syncwarp();
      if (issued < n) {
        issue(issued, s);
        ++issued;
      }
#pragma unroll
      for (int j = 0; j < M::R; ++j) sc_cur[j] = sc_nxt[j];
    }
    if (!ok) {
      if (lane == 0) atomicOr(p.err, DEVERR_WAIT_TIMEOUT);
      for (int k = max(issued - S, 0); k < issued; ++k)
        warp_wait_phase(smem_addr(my_bars + k % S), uint32_t(k / S) & 1u, DRAIN_LIMIT_NS);
    }
  }

  // The sums that this warp's tokens have so far, the first ones under way while the pieces meet.
  constexpr int AHEAD = 4;
  float* const sums = LOG ? c.weights + int64_t(b) * c.w_sb + int64_t(h) * c.w_sh : nullptr;
  float old[AHEAD];
  auto load_old = [&](int i0) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (i0 + u * 32 >= n * C::TILE) break;
      const int i = i0 + u * 32 + lane;
      const int j = i < n * C::TILE ? tile_token(i >> C::LOG_TILE) + (i & (C::TILE - 1)) : len;
      old[u] = j < len ? sums[j] : 0.f;
    }
  };
  if constexpr (LOG) load_old(0);

  // ---- the warps' pieces, in their own stages; a warp without tiles has m = -inf and no accumulators
  float* const piece = reinterpret_cast<float*>(my_stages);
  if (n > 0 && ok) {
    float lt[M::L];
    mw.total_l(lt);
    mw.store_ml(s_m[warp], s_l[warp], lt);
    mw.store_acc(piece);
  } else if (lane < GT) {
    s_m[warp][lane] = -INFINITY;
    s_l[warp][lane] = 0.f;
  }
  __syncthreads();
  const unsigned char* pieces = smem + (((base + uint32_t(c.scores_bytes) + 1023u) & ~1023u) - base);
  constexpr int GPH = D / 4, GROUPS = GT * GPH;  // float4 groups of a head, of the item
  for (int i = tid; i < GROUPS; i += W * 32) {
    const int hd = i / GPH;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, s_m[w][hd]);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (s_m[w][hd] == -INFINITY) continue;
      const float f = exp2f(s_m[w][hd] - m);
      const float4 x = reinterpret_cast<const float4*>(pieces + size_t(w) * S * C::STAGE_BYTES)[i];
      l = fmaf(f, s_l[w][hd], l);
      a.x = fmaf(f, x.x, a.x);
      a.y = fmaf(f, x.y, a.y);
      a.z = fmaf(f, x.z, a.z);
      a.w = fmaf(f, x.w, a.w);
    }
    reinterpret_cast<float4*>(s_acc)[i] = a;
    if (i % GPH == 0) {
      s_cta[hd] = m;
      s_cta[GT + hd] = l;
    }
  }
  if (split > 1) {
    cluster_sync();
  } else {
    __syncthreads();
  }
  // ---- the CTAs' pieces: every CTA finishes a share of the item's groups
  const uint32_t cta_addr = smem_addr(s_cta), acc_addr = smem_addr(s_acc);
  for (int i = (tid << c.log2_split) + rank; i < heads * GPH; i += (W * 32) << c.log2_split) {
    const int hd = i / GPH;
    float mr[8], lr[8];
    float4 x[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r < split) {
        mr[r] = ld_cluster_f32(cluster_addr(cta_addr + hd * 4, r));
        lr[r] = ld_cluster_f32(cluster_addr(cta_addr + (GT + hd) * 4, r));
        x[r] = ld_cluster_v4(cluster_addr(acc_addr + i * 16, r));
      }
    }
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < split) m = fmaxf(m, mr[r]);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r < split && mr[r] != -INFINITY) {
        const float f = exp2f(mr[r] - m);
        l = fmaf(f, lr[r], l);
        a.x = fmaf(f, x[r].x, a.x);
        a.y = fmaf(f, x[r].y, a.y);
        a.z = fmaf(f, x[r].z, a.z);
        a.w = fmaf(f, x[r].w, a.w);
      }
    }
    const float inv = normaliser(m, l);
    T* const out = reinterpret_cast<T*>(p.out) + int64_t(b) * p.o_sb + int64_t(hq0 + hd) * p.o_sh + i % GPH * 4;
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(out) = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    } else {
      uint2 o;
      o.x = E::pack2(a.x * inv, a.y * inv);
      o.y = E::pack2(a.z * inv, a.w * inv);
      *reinterpret_cast<uint2*>(out) = o;
    }
  }
  if constexpr (LOG) {
    if (tid < heads) {
      float m = -INFINITY, l = 0.f;
      for (int r = 0; r < split; ++r) m = fmaxf(m, ld_cluster_f32(cluster_addr(cta_addr + tid * 4, r)));
      for (int r = 0; r < split; ++r) {
        const float mr = ld_cluster_f32(cluster_addr(cta_addr + tid * 4, r));
        if (mr != -INFINITY) l = fmaf(exp2f(mr - m), ld_cluster_f32(cluster_addr(cta_addr + (GT + tid) * 4, r)), l);
      }
      s_final[0][tid] = m;
      s_final[1][tid] = 1.f / l;
    }
    __syncthreads();
    float m_of[GT], inv_of[GT];
#pragma unroll
    for (int q = 0; q < GT; ++q) {
      m_of[q] = q < heads ? s_final[0][q] : 0.f;
      inv_of[q] = q < heads ? s_final[1][q] : 0.f;
    }
    for (int i0 = 0; ok && i0 < n * C::TILE; i0 += 32 * AHEAD) {
      if (i0 > 0) load_old(i0);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (i0 + u * 32 >= n * C::TILE) break;
        const int i = i0 + u * 32 + lane;
        const int j = i < n * C::TILE ? tile_token(i >> C::LOG_TILE) + (i & (C::TILE - 1)) : len;
        if (j >= len) continue;
        float s[GT];
        if constexpr (GT >= 4) {
#pragma unroll
          for (int q = 0; q < GT; q += 4) *reinterpret_cast<float4*>(s + q) = *reinterpret_cast<const float4*>(my_scores + i * GT + q);
        } else if constexpr (GT == 2) {
          *reinterpret_cast<float2*>(s) = *reinterpret_cast<const float2*>(my_scores + i * GT);
        } else {
          s[0] = my_scores[i];
        }
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < GT; ++q)
          if (q < heads) sum = fmaf(exp2f(s[q] - m_of[q]), inv_of[q], sum);
        sums[j] = old[u] + sum;
      }
    }
  }
  if (split > 1) cluster_sync();  // nothing of this CTA is read any more
}

template <typename T, int D, int GT, bool LOG, int W>
cudaError_t launch_cluster_w(const DecodeParams& p, const ClusterDecode& c, const CUtensorMap& kmap, const CUtensorMap& vmap,
                             int items, cudaStream_t stream) {
  auto fn = pd_decode_cluster_kernel<T, D, GT, LOG, W>;
  constexpr int MOST = cluster_smem(W, GT, D);
  static SmemRaised raised{};
  const cudaError_t err = raise_smem_limit(fn, MOST, raised);
  if (err != cudaSuccess) return err;
  const size_t smem = size_t(c.scores_bytes) + 1024 + size_t(W) * p.stages * DecodeCfg<T, D, GT>::STAGE_BYTES;
  if (smem > size_t(MOST)) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1u << c.log2_split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(items) << c.log2_split);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = c.log2_split > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, p, c, kmap, vmap);
}

template <typename T, int D, int GT, bool LOG>
cudaError_t launch_cluster(const DecodeParams& p, const ClusterDecode& c, const CUtensorMap& kmap, const CUtensorMap& vmap,
                           int items, cudaStream_t stream) {
  return c.warps == 4 ? launch_cluster_w<T, D, GT, LOG, 4>(p, c, kmap, vmap, items, stream)
                      : launch_cluster_w<T, D, GT, LOG, 8>(p, c, kmap, vmap, items, stream);
}

// Clusters of 2^log2_split CTAs of W warps that the current device runs at once (a cluster stays in one of its
// groups of multiprocessors: of eight CTAs of eight warps, 15 clusters on 148), 0 where it cannot be asked.
template <typename T, int W>
int cluster_room_of(int log2_split) {
  auto fn = pd_decode_cluster_kernel<T, 128, 2, false, W>;
  constexpr int SMEM = cluster_smem(W, 2, 128);
  static SmemRaised raised{};
  if (raise_smem_limit(fn, SMEM, raised) != cudaSuccess) return 0;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1u << log2_split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1u << log2_split);
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = SMEM;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, fn, &cfg) == cudaSuccess ? n : 0;
}

}  // namespace pd
