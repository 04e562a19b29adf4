// pd_evict.cu -- eviction from a paged cache by accumulated attention weight (sm_100a).
//
// Per (layer, row, kv head) with n > keep tokens: the first `sinks` and the last `recent` tokens stay, and of
// the ones between the keep - sinks - recent with the largest sums (a tie keeps the lower index; NaN counts as
// the smallest). The kept tokens' K and V rows close ranks, in their order, and their sums with them.
//
// Two launches. (1) select: one CTA per (layer, row, kv head) finds the threshold -- the largest 32-bit pattern
// that at least as many of the order-preserving keys reach as there are places -- bit by bit, by counting: no
// histogram, so equal sums cost nothing extra. The keys stay in registers. Then the tokens are ranked in order
// (ballots and one scan per CTA-wide stretch), which gives the list of kept tokens, and the sums move.
// (2) move: a CTA takes a column slice of the K or V rows of one (layer, row, kv head) and walks its list in
// order. In place a token only moves down, so a stretch's rows are all in registers before any of them is
// stored, and no later source has been overwritten; slices never meet.
#include "pd_evict.cuh"

#include "pd_block_copy.cuh"

namespace pd {

namespace {

constexpr int SELECT_THREADS = 512;
constexpr int SELECT_WARPS = SELECT_THREADS / 32;

// Keys in the order of the sums: NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// P: keys of a thread in registers, or 0: read again for every count.
template <int P>
__global__ void __launch_bounds__(SELECT_THREADS) pd_evict_select_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int s_count[2][SELECT_WARPS];
  __shared__ int2 s_scan[2][SELECT_WARPS];
  __shared__ int s_first;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int item = blockIdx.x;  // (layer, row, kv head)
  const int h = item % p.n_kv_head, b = item / p.n_kv_head % p.batch, layer = item / p.n_kv_head / p.batch;
  int n = __ldg(p.seqlen + b);
  n = n < 0 ? 0 : (n > p.capacity ? p.capacity : n);
  const float* w = p.weights + layer * p.w_sl + b * p.w_sb + h * p.w_sh;
  float* wo = p.weights_out + layer * p.wo_sl + b * p.wo_sb + h * p.wo_sh;
  const int m = n < p.keep ? n : p.keep;
  if (n <= p.keep) {
    for (int64_t j = tid; j < p.w_len; j += SELECT_THREADS) wo[j] = j < n ? w[j] : 0.f;
    if (tid == 0) p.info[item] = make_int2(n, n);
    return;
  }
  const int lo = p.sinks, hi = n - p.recent, places = p.keep - p.sinks - p.recent;
  if (tid == 0) s_first = n;

  uint32_t key[P ? P : 1];
  if constexpr (P != 0) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int j = i * SELECT_THREADS + tid;
      key[i] = j >= lo && j < hi ? key_of(w[j]) : 0u;
    }
  }
  // CTA-wide count of the middle tokens whose key reaches x (x > 0, so that the zeros elsewhere do not).
  int turn = 0;
  auto reach = [&](uint32_t x) -> int {
    int c = 0;
    if constexpr (P != 0) {
#pragma unroll
      for (int i = 0; i < P; ++i) c += key[i] >= x;
    } else {
      for (int j = lo + tid; j < hi; j += SELECT_THREADS) c += key_of(w[j]) >= x;
    }
    c = __reduce_add_sync(FULL_MASK, c);
    if (lane == 0) s_count[turn][warp] = c;
    __syncthreads();
    c = __reduce_add_sync(FULL_MASK, lane < SELECT_WARPS ? s_count[turn][lane] : 0);
    turn ^= 1;  // the next count's writes do not meet this one's reads
    return c;
  };
  // The largest x that at least `places` keys reach (0: every key does).
  uint32_t x = 0u;
  int got = hi - lo;  // keys that reach x
  if (places > 0) {
    for (int bit = 31; bit >= 0 && got != places; --bit) {
      const int c = reach(x | 1u << bit);
      if (c >= places) {
        x |= 1u << bit;
        got = c;
      }
    }
  }
  // Above the threshold all stay; of those at it, the first. got == places: all that reach it stay.
  int above = got, at = 0;
  if (places == 0) {
    x = 0xffffffffu;  // no key is that large (it would be a NaN's pattern)
    above = 0;
  } else if (got != places) {
    above = x == 0xffffffffu ? 0 : reach(x + 1u);
    at = places - above;
  }
  const bool exact = at == 0;  // keys >= x are the ones (places == 0: none)

  int32_t* order = p.order + int64_t(item) * p.keep;
  int base = 0, ties = 0;  // kept tokens, and tokens at the threshold, before this stretch
  int side = 0;
  __syncthreads();  // s_first
  for (int j0 = 0; j0 < n; j0 += SELECT_THREADS, side ^= 1) {
    const int j = j0 + tid;
    const float value = j < n ? w[j] : 0.f;
    const bool middle = j >= lo && j < hi;
    const uint32_t k = key_of(value);
    const bool tie = middle && !exact && k == x;
    bool stays = j < n && (!middle || (exact ? k >= x : k > x));
    const unsigned tie_mask = __ballot_sync(FULL_MASK, tie), stay_mask = __ballot_sync(FULL_MASK, stays);
    if (lane == 0) s_scan[side][warp] = make_int2(__popc(stay_mask), __popc(tie_mask));
    __syncthreads();  // also: every value of the stretch is read before one is written
    int2 before = make_int2(0, 0), all = make_int2(0, 0);
#pragma unroll
    for (int i = 0; i < SELECT_WARPS; ++i) {
      const int2 c = s_scan[side][i];
      if (i < warp) {
        before.x += c.x;
        before.y += c.y;
      }
      all.x += c.x;
      all.y += c.y;
    }
    const unsigned lower = (1u << lane) - 1u;
    const int tie_rank = ties + before.y + __popc(tie_mask & lower);
    if (tie && tie_rank < at) stays = true;
    // kept before j: those above or outside, and the ties that still had a place
    const int rank = base + before.x + __popc(stay_mask & lower) + min(tie_rank, at) - min(ties, at);
    base += all.x + min(ties + all.y, at) - min(ties, at);
    ties += all.y;
    if (stays) {
      wo[rank] = value;
      order[rank] = j;
    }
    const unsigned gone = __ballot_sync(FULL_MASK, j < n && !stays);
    if (gone && lane == 0) atomicMin(&s_first, j0 + warp * 32 + __ffs(gone) - 1);
  }
  __syncthreads();  // s_first
  for (int64_t j = m + tid; j < p.w_len; j += SELECT_THREADS) wo[j] = 0.f;
  if (tid == 0) p.info[item] = make_int2(s_first, m);
}

constexpr int MOVE_THREADS = 256;
constexpr int AHEAD = 4;  // rows of a thread in flight

__global__ void __launch_bounds__(MOVE_THREADS) pd_evict_move_kernel(const __grid_constant__ EvictParams p, int log2_slice) {
  const int tid = threadIdx.x;
  const int per = 1 << log2_slice;                  // 16-byte units of a slice
  const int slices = (p.chunks + per - 1) >> log2_slice;
  const int slice = blockIdx.x % slices;
  const int rest = blockIdx.x / slices;
  const int is_v = rest & 1, item = rest >> 1;
  const int h = item % p.n_kv_head, b = item / p.n_kv_head % p.batch, layer = item / p.n_kv_head / p.batch;
  griddep_wait();
  const int2 info = p.info[item];
  if (p.seqlen_out != nullptr && layer == 0 && h == 0 && is_v == 0 && slice == 0 && tid == 0) p.seqlen_out[b] = info.y;
  const int32_t* order = p.order + int64_t(item) * p.keep;
  const int32_t* from = p.table + int64_t(b) * p.bt_stride;
  const int32_t* to = p.new_table + int64_t(b) * p.nbt_stride;
  const int64_t sb = is_v ? p.v_sb : p.k_sb, sn = is_v ? p.v_sn : p.k_sn, sh = is_v ? p.v_sh : p.k_sh;
  const int unit = (slice << log2_slice) + (tid & (per - 1));
  uint4* pool = static_cast<uint4*>(is_v ? p.v[layer] : p.k[layer]) + h * sh + unit;
  const bool mine = unit < p.chunks;
  const int mask = (1 << p.log2_bs) - 1;
  const int step = MOVE_THREADS >> log2_slice;
  // The row of token t by a table of `width` blocks, or nullptr (reported).
  auto row = [&](const int32_t* table, int width, int t) -> uint4* {
    const int page = t >> p.log2_bs;
    const int blk = page < width ? __ldg(table + page) : -1;
    if (blk < 0 || blk >= p.n_blocks) {
      atomicOr(p.err, DEVERR_COPY_RANGE);
      return nullptr;
    }
    return pool + int64_t(blk) * sb + int64_t(t & mask) * sn;
  };
  for (int r0 = p.fresh ? 0 : info.x; r0 < info.y; r0 += step * AHEAD) {
    uint4 x[AHEAD];
    uint4* dst[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int r = r0 + i * step + (tid >> log2_slice);
      dst[i] = nullptr;
      if (!mine || r >= info.y) continue;
      const uint4* src = row(from, p.max_blocks, r < info.x ? r : order[r]);
      if (src == nullptr) continue;
      x[i] = *src;
      dst[i] = row(to, p.new_max_blocks, r);
    }
    __syncthreads();  // a stretch's rows are read before one is written
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (dst[i] != nullptr) *dst[i] = x[i];
  }
}

}  // namespace

cudaError_t launch_evict(const EvictParams& p, cudaStream_t stream) {
  const int64_t items = int64_t(p.layers) * p.batch * p.n_kv_head;
  if (items == 0) return cudaSuccess;
  void (*select)(EvictParams) = pd_evict_select_kernel<0>;
  if (p.capacity <= SELECT_THREADS * 4) select = pd_evict_select_kernel<4>;
  else if (p.capacity <= SELECT_THREADS * 16) select = pd_evict_select_kernel<16>;
  else if (p.capacity <= SELECT_THREADS * 64) select = pd_evict_select_kernel<64>;
  select<<<unsigned(items), SELECT_THREADS, 0, stream>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // Slices of at least 32 bytes, until there are eight CTAs for every SM.
  int log2_slice = 0;
  while ((1 << log2_slice) < p.chunks) ++log2_slice;
  while (log2_slice > 1 && 2 * items * ((p.chunks + (1 << log2_slice) - 1) >> log2_slice) < 8 * int64_t(p.sms)) --log2_slice;
  const int64_t ctas = 2 * items * ((p.chunks + (1 << log2_slice) - 1) >> log2_slice);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(MOVE_THREADS);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pd_evict_move_kernel, p, log2_slice);
}

}  // namespace pd
