// pd_evict.cu -- eviction from a paged cache by accumulated attention weight (sm_100a).
//
// Per (layer, row, kv head) with n > keep tokens: the first `sinks` and the last `recent` tokens stay, and of
// the ones between the keep - sinks - recent with the largest sums (a tie keeps the lower index; NaN counts as
// the smallest). The kept tokens' K and V rows close ranks, in their order, and their sums with them.
//
// Two launches. (1) select: one CTA per (layer, row, kv head) finds the threshold -- the largest key that at least as
// many of the order-preserving 32-bit keys reach as there are places -- by histograms of 256 bins over the range that
// is left, at first that of the row's own keys, so that two or three rounds mostly do, over a copy in shared memory.
// Then the tokens are ranked in order (every warp a stretch, after one scan of the stretches' counts), which gives
// the list of kept tokens, and the sums move.
// (2) move: a CTA takes the K or V rows (a column slice of them) of one (layer, row, kv head) and walks its list in
// order, the next stretch's loads under way while it stores. In place a token only moves down, so that a stretch's
// rows need only be read before one of them is written; slices never meet.
//
// Measured (8 kv heads of 128, bf16): 32 rows of 1040 cut to 1024 in 8 layers, where a tenth of the sums are zero and
// tokens move from about the 750th on, 119 us, of which select 19.7 (bound by its instructions, 74 % of the issue
// slots) and move 99 (512 MB of DRAM traffic at 5.2 TB/s); the same without equal sums, so that almost every token moves,
// 352 us (314 would move the bytes); one row of 700 cut to 512 in 28 layers 32.5 us, select 8.5 (its rounds, one after the
// other) and move 20.
#include "pd_evict.cuh"

#include <algorithm>

#include "pd_block_copy.cuh"
#include "pd_smem_limit.cuh"

namespace pd {

namespace {


// Keys in the order of the sums: NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int BINS = 256;

// WARPS of a CTA; COPY: the row's sums are copied into shared memory, else read again from global for every pass.
// (In registers the passes would be unrolled, and a CTA that runs 60 KB of code once waits for its instructions:
// 2048 rows of 1040 took 68 us.)
template <int WARPS, bool COPY>
__global__ void __launch_bounds__(WARPS * 32) pd_evict_select_kernel(const __grid_constant__ EvictParams p) {
  constexpr int THREADS = WARPS * 32;
  extern __shared__ float s_sums[];
  griddep_launch_dependents();
  __shared__ uint2 s_range[WARPS];
  __shared__ __align__(16) int s_bins[BINS];
  __shared__ int4 s_found;  // bin of the threshold, keys above it, keys in it
  __shared__ int2 s_scan[2][WARPS];
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
    for (int64_t j = tid; j < p.w_len; j += THREADS) wo[j] = j < n ? w[j] : 0.f;
    if (tid == 0) p.info[item] = make_int2(n, n);
    return;
  }
  const int lo = p.sinks, hi = n - p.recent, places = p.keep - p.sinks - p.recent;
  if (tid == 0) s_first = n;
  uint32_t* s_keys = reinterpret_cast<uint32_t*>(s_sums + (COPY ? n : 0));
  uint32_t low = 0xffffffffu, high = 0u;  // of the middle tokens' keys
  if constexpr (COPY) {
#pragma unroll 8
    for (int j = tid; j < n; j += THREADS) {
      const float value = w[j];
      const uint32_t k = key_of(value);
      s_sums[j] = value;
      s_keys[j] = k;
      if (j >= lo && j < hi) {
        low = min(low, k);
        high = max(high, k);
      }
    }
  } else {
    for (int j = lo + tid; j < hi; j += THREADS) {
      const uint32_t k = key_of(w[j]);
      low = min(low, k);
      high = max(high, k);
    }
  }
  auto key = [&](int j) -> uint32_t { return COPY ? s_keys[j] : key_of(w[j]); };
  // The threshold x, and how many of the tokens at it stay (the first ones; `exact`: all that reach x stay).
  uint32_t x = 0xffffffffu;  // no token has this key: it is a NaN's pattern
  int at = 0;
  if (places > 0) {
    // Keys low .. high hold the threshold; `need` of them stay.
    int need = places;
    for (bool first = true;; first = false) {
      if (!first) {  // the range of the keys that are left
        uint32_t a = 0xffffffffu, z = 0u;
#pragma unroll 4
        for (int j = lo + tid; j < hi; j += THREADS) {
          const uint32_t k = key(j);
          if (k - low <= high - low) {
            a = min(a, k);
            z = max(z, k);
          }
        }
        low = a;
        high = z;
      }
      low = __reduce_min_sync(FULL_MASK, low);
      high = __reduce_max_sync(FULL_MASK, high);
      if (lane == 0) s_range[warp] = make_uint2(low, high);
      for (int i = tid; i < BINS; i += THREADS) s_bins[i] = 0;
      __syncthreads();
      const uint2 r = s_range[lane < WARPS ? lane : 0];
      low = __reduce_min_sync(FULL_MASK, r.x);
      high = __reduce_max_sync(FULL_MASK, r.y);
      x = low;
      if (low == high) {  // one key: the first of its tokens stay
        at = need;
        break;
      }
      // Bins of 2^shift from `base` on, the last one at `high`. At first an eighth of an octave each, so that the
      // bins are many and few atomics meet; what lies 32 octaves below the largest, zeros above all, is in the lowest.
      const int width = 32 - __clz(high - low);
      const int shift = max((first ? min(width, 28) : width) - 8, 0);
      const uint32_t span = uint32_t(BINS - 1) << shift;
      const uint32_t base = high - low > span ? (high - span) >> shift << shift : low;
#pragma unroll 4
      for (int j = lo + tid; j < hi; j += THREADS) {
        const uint32_t k = key(j);
        if (k - low <= high - low) atomicAdd(&s_bins[min((max(k, base) - base) >> shift, uint32_t(BINS - 1))], 1);
      }
      __syncthreads();
      if (warp == 0) {  // lane l: bins 8 l .. 8 l + 7; the first from above with which `need` are reached
        const int4 c0 = reinterpret_cast<const int4*>(s_bins)[lane * 2], c1 = reinterpret_cast<const int4*>(s_bins)[lane * 2 + 1];
        const int c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
        const int sum = c0.x + c0.y + c0.z + c0.w + c1.x + c1.y + c1.z + c1.w;
        int from = sum;  // keys in this lane's bins and above
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_down_sync(FULL_MASK, from, o);
          if (lane + o < 32) from += y;
        }
        int above = from - sum;
        if (above < need && from >= need) {
#pragma unroll
          for (int i = 7; i >= 0; --i) {
            if (above + c[i] >= need) {
              s_found = make_int4(lane * 8 + i, above, c[i], 0);
              break;
            }
            above += c[i];
          }
        }
      }
      __syncthreads();
      const int4 f = s_found;
      if (f.x < BINS - 1) high = min(high, base + (uint32_t(f.x + 1) << shift) - 1u);
      if (f.x > 0) low = base + (uint32_t(f.x) << shift);
      need -= f.y;
      x = low;
      if (need == f.z) break;  // all of the bin stay
    }
  }
  const bool exact = at == 0;
  if (places == 0) __syncthreads();  // the copy (the rounds above have waited for it)

  int32_t* order = p.order + int64_t(item) * p.keep;
  const unsigned lower = (1u << lane) - 1u;
  const uint32_t enough = exact ? x : x + 1u;  // (x is below the largest number)
  auto kept = [&](int j, uint32_t k) -> bool { return j < lo || j >= hi || k >= enough; };  // but for a tie
  auto is_tie = [&](int j, uint32_t k) -> bool { return !exact && k == x && j >= lo && j < hi; };
  // Token j goes to `rank`, if it stays: `before` kept tokens and `ties` at the threshold lie before its 32.
  bool all_stay = true;  // so far in this warp
  auto place = [&](int j, float value, int before, int ties, unsigned stay_mask, unsigned tie_mask) {
    bool stays = stay_mask >> lane & 1u;
    int rank = before + __popc(stay_mask & lower);
    if (!exact) {
      const int tie_rank = ties + __popc(tie_mask & lower);
      stays = stays || ((tie_mask >> lane & 1u) && tie_rank < at);
      rank += min(tie_rank, at);
    }
    if (stays) {
      wo[rank] = value;
      order[rank] = j;
    }
    if (all_stay) {
      const unsigned gone = __ballot_sync(FULL_MASK, j < n && !stays);
      if (gone) {
        all_stay = false;
        if (lane == 0) atomicMin(&s_first, j + __ffs(gone) - 1);
      }
    }
  };
  if constexpr (COPY) {
    // A warp's stretch of 32-token steps: whether they stay, a bit a step, one scan of the counts, then every
    // warp ranks its own.
    const int per = (n + THREADS - 1) / THREADS, start = warp * per * 32 + lane;
    unsigned stay_bits = 0u, tie_bits = 0u;  // (at most 32 steps: launch_select)
#pragma unroll 4
    for (int i = 0; i < per; ++i) {
      const int j = start + i * 32;
      if (j < n) {
        const uint32_t k = s_keys[j];
        stay_bits |= unsigned(kept(j, k)) << i;
        tie_bits |= unsigned(is_tie(j, k)) << i;
      }
    }
    const int stay = __reduce_add_sync(FULL_MASK, __popc(stay_bits));
    const int tie = __reduce_add_sync(FULL_MASK, __popc(tie_bits));
    if (lane == 0) s_scan[0][warp] = make_int2(stay, tie);
    __syncthreads();
    const int2 c = lane < warp ? s_scan[0][lane] : make_int2(0, 0);
    int before = __reduce_add_sync(FULL_MASK, c.x), ties = __reduce_add_sync(FULL_MASK, c.y);
    for (int i = 0; i < per; ++i) {
      const int j = start + i * 32;
      const unsigned stay_mask = __ballot_sync(FULL_MASK, stay_bits >> i & 1u);
      const unsigned tie_mask = exact ? 0u : __ballot_sync(FULL_MASK, tie_bits >> i & 1u);
      place(j, j < n ? s_sums[j] : 0.f, before, ties, stay_mask, tie_mask);
      before += __popc(stay_mask);
      ties += __popc(tie_mask);
    }
  } else {
    // A CTA-wide stretch at a time: in place, what is written never lies past the stretch at hand.
    int before = 0, ties = 0, side = 0;
    __syncthreads();  // s_first
    for (int j0 = 0; j0 < n; j0 += THREADS, side ^= 1) {
      const int j = j0 + tid;
      const float value = j < n ? w[j] : 0.f;
      const unsigned stay_mask = __ballot_sync(FULL_MASK, j < n && kept(j, key_of(value)));
      const unsigned tie_mask = __ballot_sync(FULL_MASK, j < n && is_tie(j, key_of(value)));
      if (lane == 0) s_scan[side][warp] = make_int2(__popc(stay_mask), __popc(tie_mask));
      __syncthreads();  // also: every sum of the stretch is read before one is written
      const int2 c = lane < WARPS ? s_scan[side][lane] : make_int2(0, 0);
      const int2 mine_before = make_int2(__reduce_add_sync(FULL_MASK, lane < warp ? c.x : 0),
                                         __reduce_add_sync(FULL_MASK, lane < warp ? c.y : 0));
      place(j, value, before + mine_before.x, ties + mine_before.y, stay_mask, tie_mask);
      before += __reduce_add_sync(FULL_MASK, c.x);
      ties += __reduce_add_sync(FULL_MASK, c.y);
    }
  }
  __syncthreads();  // s_first
  for (int64_t j = m + tid; j < p.w_len; j += THREADS) wo[j] = 0.f;
  if (tid == 0) p.info[item] = make_int2(s_first, m);
}

constexpr int MOVE_THREADS = 256;
constexpr int AHEAD = 4;             // rows of a thread in a stretch
constexpr int CHUNK = MOVE_THREADS;  // rows whose places are looked up at a time
static_assert(EVICT_UNITS <= MOVE_THREADS, "every unit of a slice has a thread, so that a step is a row or more");

// `parts` CTAs share the list of one (layer, row, kv head)'s K or V (new pages only: nothing that is written is
// read), each of them in slices of 2^log2_slice 16-byte units, at least 4, so that a stretch is at most a chunk.
__global__ void __launch_bounds__(MOVE_THREADS) pd_evict_move_kernel(const __grid_constant__ EvictParams p, int log2_slice,
                                                                     int parts) {
  __shared__ int64_t s_src[2][CHUNK], s_dst[2][CHUNK];
  const int tid = threadIdx.x;
  const int per = 1 << log2_slice;
  const int slices = (p.chunks + per - 1) >> log2_slice;
  const int slice = blockIdx.x % slices, part = blockIdx.x / slices % parts;
  const int rest = blockIdx.x / slices / parts;
  const int is_v = rest & 1, item = rest >> 1;
  const int h = item % p.n_kv_head, b = item / p.n_kv_head % p.batch, layer = item / p.n_kv_head / p.batch;
  const int32_t* from = p.table + int64_t(b) * p.bt_stride;
  const int32_t* to = p.new_table + int64_t(b) * p.nbt_stride;
  const int64_t sb = is_v ? p.v_sb : p.k_sb, sn = is_v ? p.v_sn : p.k_sn, sh = is_v ? p.v_sh : p.k_sh;
  const int unit = (slice << log2_slice) + (tid & (per - 1));
  uint4* pool = static_cast<uint4*>(is_v ? p.v[layer] : p.k[layer]) + h * sh + unit;
  const bool mine = unit < p.chunks;
  const int mask = (1 << p.log2_bs) - 1;
  const int step = MOVE_THREADS >> log2_slice, my_row = tid >> log2_slice;
  griddep_wait();
  const int2 info = p.info[item];
  if (p.seqlen_out != nullptr && layer == 0 && h == 0 && is_v == 0 && slice == 0 && part == 0 && tid == 0)
    p.seqlen_out[b] = info.y;
  const int32_t* order = p.order + int64_t(item) * p.keep;
  const int all0 = p.fresh ? 0 : info.x, share = ((info.y - all0 + parts - 1) / parts + CHUNK - 1) / CHUNK * CHUNK;
  const int first = all0 + part * share, count = min(share, info.y - first);
  // Offset of token t's row by a table of `width` blocks, or -1 (reported).
  auto row = [&](const int32_t* table, int width, int t) -> int64_t {
    const int page = t >> p.log2_bs;
    const int blk = page < width ? __ldg(table + page) : -1;
    if (blk < 0 || blk >= p.n_blocks) {
      atomicOr(p.err, DEVERR_COPY_RANGE);
      return -1;
    }
    return int64_t(blk) * sb + int64_t(t & mask) * sn;
  };
  auto look_up = [&](int chunk) {  // a thread a row
    const int i = chunk * CHUNK + tid, r = first + i;
    int64_t src = -1, dst = -1;
    if (i < count) {
      dst = row(to, p.new_max_blocks, r);
      src = row(from, p.max_blocks, r < info.x ? r : order[r]);
      if (src < 0) dst = -1;
    }
    s_src[chunk & 1][tid] = src;
    s_dst[chunk & 1][tid] = dst;
  };
  auto load = [&](int i0, uint4 (&x)[AHEAD]) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * step + my_row;
      if (i >= count) continue;
      const int64_t src = s_src[(i / CHUNK) & 1][i % CHUNK];
      if (mine && src >= 0) x[k] = pool[src];
    }
  };
  if (count <= 0) return;
  uint4 x[AHEAD], y[AHEAD];
  look_up(0);
  __syncthreads();
  load(0, x);
  for (int i0 = 0; i0 < count; i0 += step * AHEAD) {
    __syncthreads();  // this stretch's rows are read before one is written; the last chunk's places are done with
    if (i0 % CHUNK == 0 && i0 + CHUNK < count) {
      look_up(i0 / CHUNK + 1);
      __syncthreads();
    }
    load(i0 + step * AHEAD, y);  // in place, what is written now lies before every later source
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * step + my_row;
      if (i >= count) continue;
      const int64_t dst = s_dst[(i / CHUNK) & 1][i % CHUNK];
      if (mine && dst >= 0) pool[dst] = x[k];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) x[k] = y[k];
  }
}

// Rows of up to so many tokens are copied into shared memory.
constexpr int COPY_TOKENS = 24576;  // in keys and sums, 8 bytes a token

template <int WARPS, bool COPY>
cudaError_t select(const EvictParams& p, int64_t items, cudaStream_t stream) {
  auto fn = pd_evict_select_kernel<WARPS, COPY>;
  static SmemRaised raised{};
  const cudaError_t err = raise_smem_limit(fn, COPY ? COPY_TOKENS * 8 : 0, raised);
  if (err != cudaSuccess) return err;
  fn<<<unsigned(items), WARPS * 32, COPY ? size_t(p.capacity) * 8 : 0, stream>>>(p);
  return cudaGetLastError();
}

// Warps by the row's length: eight or so tokens a thread, and half that where there are few rows.
cudaError_t launch_select(const EvictParams& p, int64_t items, cudaStream_t stream) {
  const int64_t tokens = items < 4 * int64_t(p.sms) ? int64_t(p.capacity) * 2 : p.capacity;
  if (p.capacity > COPY_TOKENS) return select<32, false>(p, items, stream);
  if (tokens <= 512) return select<2, true>(p, items, stream);
  if (tokens <= 1280) return select<4, true>(p, items, stream);
  if (tokens <= 2560) return select<8, true>(p, items, stream);
  if (tokens <= 5120) return select<16, true>(p, items, stream);
  return select<32, true>(p, items, stream);
}

}  // namespace

cudaError_t launch_evict(const EvictParams& p, cudaStream_t stream) {
  const int64_t items = int64_t(p.layers) * p.batch * p.n_kv_head;
  if (items == 0) return cudaSuccess;
  if (p.chunks > EVICT_UNITS) return cudaErrorInvalidValue;
  cudaError_t e = launch_select(p, items, stream);
  if (e != cudaSuccess) return e;
  // New pages' lists are shared by CTAs until there are four for every SM, down to a chunk each (9 prompts in 4 layers:
  // one or two 49.4 us, four 43.6). Rows moved in place are cut into slices, down to 64 bytes, until there are two: wider
  // copies are worth more than more of them (one row in 28 layers: whole rows 30.0 us, 128 bytes 31.7, 64 33.3).
  int log2_slice = 2, parts = 1;
  while ((1 << log2_slice) < p.chunks) ++log2_slice;
  int64_t ctas = 2 * items;
  const int64_t enough = (p.fresh ? 4 : 2) * int64_t(p.sms);
  if (p.fresh) {
    parts = int(std::min((enough + ctas - 1) / ctas, int64_t(p.keep + CHUNK - 1) / CHUNK));
    ctas *= parts;
  } else {
    while (log2_slice > 2 && ctas < enough) {
      --log2_slice;
      ctas = 2 * items * ((p.chunks + (1 << log2_slice) - 1) >> log2_slice);
    }
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(MOVE_THREADS);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pd_evict_move_kernel, p, log2_slice, parts);
}

}  // namespace pd
