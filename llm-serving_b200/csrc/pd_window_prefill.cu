// pd_window_prefill.cu -- attention of query chunks over a window of a paged cache on the 5th-generation
// tensor cores (tcgen05 / TMEM) for sm_100a: bf16 / fp16 pools, head_dim 64, 128 or 256, any group.
//
// Query token t of a chunk of S tokens sits at i = seqlen - S + t and sees key j iff j <= i and
// (i - j < window or j < sinks): out = softmax(q K^T scale) V over those, fp32 softmax and accumulation.
// A query row is a (token, q head of the kv head's group) pair, token-major, so a group's heads share every
// K/V tile.
//
// How (one CTA = a block of 128 query rows of one row's chunk and one kv head; two CTAs share an SM, so that one's
// start and end and its softmax hide behind the other's products; at head_dim 256 one, as O takes 256 of TMEM's 512
// columns):
//  * The keys that some query row of the CTA sees -- sinks and window, in whole copies of `box` tokens -- are
//    numbered without the gap between them and cut into steps of 64 keys, so a few sinks cost a copy, not a step.
//  * One warp streams K, another V, by TMA into rings of stages of a step, a lane a copy, block ids one step ahead. No
//    block without a visible token is looked up; where the last step ends early, V is filled with zeros from outside
//    the pool.
//  * One warp issues S = Q K^T (M 128, N 64, K head_dim) into one of two S buffers in TMEM, another O += P V with P read
//    from TMEM, where the softmax wrote it over the S it came from; so the next S is there when the softmax is done with
//    one. Where a step's copies hold tokens that no row of the CTA sees, the warp of the P V first zeroes their V, so
//    that whatever bytes they hold never reach O.
//  * 4 softmax warps, one thread per row (TMEM lane = row): maximum over the row's scores, P = 2^(s - m + 7), and
//    the fp32 sum; no exchange between threads. The maximum moves only when a step passes it by 2^8, so rescaling O
//    in TMEM is rare.
//  * P enters as two 16-bit operands, P = hi + lo: 2^-17 of the weighted mean of |v| in bf16 and 2^-22 in fp16, as
//    the causal chunk kernel (pd_prefill_tc.cu) has it; one bf16 part alone would be off by as much as the result's
//    own rounding. The factor 2^7, which the sums carry too, keeps fp16 weights down to 2^-21 normal numbers.
//  * With few blocks a cluster of `split` CTAs shares one block's steps. Each leaves its O, m and l in shared memory,
//    and every one merges a share of the rows from all of them.
//  * Measured (bf16, 16 heads on 8 of 128, window 1024): 4 prompts of 4096 tokens 175-180 us in a burst, 0.6 of the rate
//    that its three products a step allow (P V twice), and 209 call after call, under the power cap; inside the steps the
//    tensor pipe is busy 0.9 of the time, a CTA's start and end, which its neighbour on the SM covers in part, are a
//    quarter of its clocks. With S of 128 keys at a time, which leaves one CTA an SM, 204 us in a burst. 16 chunks of 1-8
//    tokens 17.9 us, latency: 9.1 would move the bytes.
//  * The grid is the longest chunk's blocks times rows and kv heads: blocks past a shorter chunk start and leave, and what
//    they take of the GPU is not left for clusters. One prompt of 4096 beside 60 rows of one token is 271 us, the
//    prompt alone 49 and the others 54.
//  * Every wait is bounded; a role whose wait runs out records DEVERR_WAIT_TIMEOUT and raises the CTA's abort
//    flag, every role then leaves its loop, copies and MMAs in flight are waited for, and the CTA frees its TMEM. All
//    threads reach the cluster's two barriers on every path.
#include "paged_decode.h"
#include "pd_smem_limit.cuh"
#include "pd_tcgen05.cuh"
#include "pd_tile.cuh"
#include "pd_window.cuh"

#include <algorithm>
#include <type_traits>

namespace pd {

namespace {

constexpr int ROWS = WINDOW_ROWS;
constexpr int KEYS = 64;   // keys of a softmax step (the S MMA's N)
constexpr float P_SHIFT = 7.f, HEADROOM = 8.f;

template <int D>
struct Cfg {
  static constexpr int CTAS = D <= 128 ? 2 : 1;  // per SM
  static constexpr int PIECES = D / 64;
  static constexpr int SOFTMAX_WARPS = 4;
  static constexpr int K_WARP = 4, V_WARP = 5, S_WARP = 6;  // and warp 7: P V
  static constexpr int THREADS = 256;
  // Where two CTAs share the registers they are dealt anew between the groups of four warps, so that a softmax
  // thread holds a row's scores and P; with one, every thread has enough.
  static constexpr bool DEAL = CTAS == 2;
  static constexpr int LAUNCH_REGS = 65536 / CTAS / THREADS / 8 * 8;
  static constexpr int SOFTMAX_REGS = 168;
  static constexpr int OTHER_REGS = 80;
  static_assert(!DEAL || SOFTMAX_REGS + OTHER_REGS <= 2 * LAUNCH_REGS, "a split above the launch's registers would wait for ever");
  static constexpr int STAGES = D == 64 ? 4 : 2;  // steps of K, and of V, in shared memory
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int KV_BYTES = KEYS * D * 2;
  static constexpr int O_COL = 2 * KEYS;  // behind the S/P buffers
  static constexpr int TMEM_COLS = CTAS == 2 ? 256 : 512;
  static_assert(O_COL + D <= TMEM_COLS && CTAS * TMEM_COLS <= 512, "TMEM columns");
  static constexpr int OFF_ML = 512;  // (m, l) of a row for the cluster's merge; barriers and flags before it
  static constexpr int OFF_AGAIN = 1536;  // rows that the merge found not finite
  static constexpr int OFF_Q = 2048;
  static constexpr int OFF_K = OFF_Q + Q_BYTES;
  static constexpr int OFF_V = OFF_K + STAGES * KV_BYTES;
  static constexpr int OFF_O = OFF_K;  // fp32 O for the cluster's merge, over K and V
  static_assert(ROWS * D * 4 <= 2 * STAGES * KV_BYTES, "O fits over K and V");
  static constexpr int SMEM = OFF_V + STAGES * KV_BYTES + 1024;  // + run-time 1 KB alignment
  static_assert(CTAS * (SMEM + 1024) <= 233472, "shared memory per SM");
};

// Barrier slots (8 bytes each) at the front of shared memory.
struct Bars {
  static constexpr int K_FULL = 0;    // [4] K of a step landed (transaction bytes)
  static constexpr int V_FULL = 4;    // [4]
  static constexpr int K_EMPTY = 8;   // [4] the step's S completed (commit)
  static constexpr int V_EMPTY = 12;  // [4] the step's P V completed (commit)
  static constexpr int S_FULL = 16;   // [2] S buffer written (commit)
  static constexpr int P_FULL = 18;   // [2] P written over it, O rescaled: one arrival per softmax warp
  static constexpr int O_DONE = 20;   // [2] P V that read the buffer completed (commit)
  static constexpr int Q_FULL = 22;   // Q stored: one arrival per softmax warp
  static constexpr int DRAIN = 23;    // [2]
  static constexpr int TMEM_SLOT = 240;  // byte offsets
  static constexpr int ABORT = 248;
};

// The keys that a CTA's query rows see, numbered without the gap between sinks and window: key u of the
// CTA is token u + (u >= head ? gap : 0).
struct Keys {
  int head;   // tokens of the sinks' copies (0 where the window reaches them: gap 0)
  int gap;    // a multiple of the copies' tokens
  int first;  // first token of the window (u - gap)
  int count;  // keys
  __device__ __forceinline__ int token(int u) const { return u >= head ? u + gap : u; }
};

// Bits [lo, hi) of 32, bounds outside 0..32 cut.
__device__ __forceinline__ uint32_t bits(int lo, int hi) {
  const uint32_t below_hi = hi <= 0 ? 0u : hi >= 32 ? 0xffffffffu : (1u << hi) - 1u;
  const uint32_t below_lo = lo <= 0 ? 0u : lo >= 32 ? 0xffffffffu : (1u << lo) - 1u;
  return below_hi & ~below_lo;
}

// One query row by one warp, over the keys it sees and no others. The tiles multiply every V of a step with some weight,
// 0 for a key that a row does not see, and 0 times an infinity or a NaN is a NaN: a row whose result is not finite is
// computed again here. (A row that sees such a value is not finite again.)
template <typename T, int D>
__device__ __noinline__ void row_again(const WindowPrefillParams& p, int b, int h, int lk, int token, int head, int at) {
  using E = Elem<T>;
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31;
  const T* q = reinterpret_cast<const T*>(p.q) + int64_t(token) * p.q_st + int64_t(head) * p.q_sh;
  const int32_t* trow = p.table + int64_t(b) * p.bt_stride;
  const int first = max(at - p.window + 1, 0), sinks = min(p.sinks, first), count = sinks + max(at + 1 - first, 0);
  float m = MAX_START, l = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  for (int i0 = 0; i0 < count; i0 += 32) {
    // a lane a key
    const int i = i0 + lane, j = i < sinks ? i : first + i - sinks, page = j >> p.log2_bs;
    const int blk = i < count && j < lk && page < p.max_blocks ? __ldg(trow + page) : -1;
    const bool known = blk >= 0 && blk < p.n_blocks;  // a block outside the pool reads zeros
    const int in_block = j & ((1 << p.log2_bs) - 1);
    float s = 0.f;
    if (known) {
      const T* k = reinterpret_cast<const T*>(p.k) + int64_t(blk) * p.k_sb + int64_t(in_block) * p.k_sn + int64_t(h) * p.k_sh;
#pragma unroll 1
      for (int d = 0; d < D; d += 8) {
        float x[8], y[8];
        E::unpack(__ldg(reinterpret_cast<const uint4*>(q + d)), x);
        E::unpack(__ldg(reinterpret_cast<const uint4*>(k + d)), y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
      }
    }
    s = i < count ? s * p.scale_log2 : -INFINITY;
    float top = s;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, o));
    const float m_new = fmaxf(m, top), alpha = m == m_new ? 1.f : exp2f(m - m_new);
    const float w = i < count ? exp2f(s - m_new) : 0.f;  // (m_new is never -inf: scores of -inf have weight 0)
    m = m_new;
    l = fmaf(l, alpha, w);  // a lane's own sum
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] *= alpha;
    const int64_t v_at = int64_t(blk) * p.v_sb + int64_t(in_block) * p.v_sn + int64_t(h) * p.v_sh;
    for (int t = 0; t < min(32, count - i0); ++t) {  // every lane PER elements of each key
      const float wt = __shfl_sync(FULL_MASK, w, t);
      const int64_t row = __shfl_sync(FULL_MASK, (long long)v_at, t);
      if (!__shfl_sync(FULL_MASK, known, t)) continue;
      const T* v = reinterpret_cast<const T*>(p.v) + row + lane * PER;
#pragma unroll
      for (int e = 0; e < PER; ++e) acc[e] = fmaf(wt, E::to_float(v[e]), acc[e]);
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(FULL_MASK, l, o);
  T* out = reinterpret_cast<T*>(p.out) + int64_t(token) * p.o_st + int64_t(head) * p.o_sh + lane * PER;
  const float inv = count > 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) out[e] = E::from_float(acc[e] * inv);
}

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::THREADS, Cfg<D>::CTAS)
    pd_window_prefill_kernel(const __grid_constant__ WindowPrefillParams p, const __grid_constant__ CUtensorMap kmap,
                             const __grid_constant__ CUtensorMap vmap, int blocks, int log2_split) {
  using C = Cfg<D>;
  using E = Elem<T>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t raw = smem_addr(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t sbase = smem_addr(smem);
  auto bar = [&](int slot) -> uint32_t { return sbase + uint32_t(slot) * 8u; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Bars::ABORT);
  // Query blocks slowest and last ones first: a prompt's first blocks have the fewest keys.
  const int split = 1 << log2_split, rank = int(blockIdx.x) & (split - 1), work = int(blockIdx.x) >> log2_split;
  const int b = work % p.batch, pair = work / p.batch;
  const int h = pair % p.n_kv_head;
  const int qblock = blocks - 1 - pair / p.n_kv_head;
  // n / group, 0 <= n < 2^31 (launch_t: group_mul is 2^group_shift / group rounded up)
  auto tokens_of = [&](int n) -> int { return int((uint64_t(uint32_t(n)) * p.group_mul) >> p.group_shift); };

  if (warp == C::S_WARP) {
    if (lane == 0) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
      for (int i = 0; i < C::STAGES; ++i) {
        mbar_init(bar(Bars::K_FULL + i), 1);
        mbar_init(bar(Bars::V_FULL + i), 1);
        mbar_init(bar(Bars::K_EMPTY + i), 1);
        mbar_init(bar(Bars::V_EMPTY + i), 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar(Bars::S_FULL + i), 1);
        mbar_init(bar(Bars::P_FULL + i), C::SOFTMAX_WARPS);
        mbar_init(bar(Bars::O_DONE + i), 1);
        mbar_init(bar(Bars::DRAIN + i), 1);
      }
      mbar_init(bar(Bars::Q_FULL), C::SOFTMAX_WARPS);
      *abort_flag = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tc::tmem_alloc(sbase + Bars::TMEM_SLOT, C::TMEM_COLS);
    tc::tmem_relinquish();
  }
  // The roles meet once, before any load: from here on each goes at its own pace (K is under way while Q is copied).
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + Bars::TMEM_SLOT);
  griddep_wait();  // everything that is read may be the preceding kernel's
  // The stream's next kernel may be launched now, not before: a CTA of it that held TMEM while it waits for this grid
  // must not be in the way of this one's, and what it reads early must not be an earlier kernel's (pd_decode_kernel.cuh).
  griddep_launch_dependents();

  const int q_begin = min(max(__ldg(p.cu_q + b), 0), p.total_q);
  const int chunk = max(min(max(__ldg(p.cu_q + b + 1), 0), p.total_q) - q_begin, 0);
  const int sq = min(chunk, p.max_seqlen_q);
  int lk = __ldg(p.seqlen + b);
  lk = lk < 0 ? 0 : (lk > p.capacity ? p.capacity : lk);
  const int rows = sq * p.group;
  const int row0 = qblock * ROWS;  // first query row of the CTA
  const int ctx = lk - chunk;      // position of the chunk's first token
  const int box = 1 << p.log2_box;
  // What the CTA's rows see: up to its last token, from its first token's window on, and the sinks.
  Keys keys;
  {
    const int last = min(row0 + ROWS, rows) - 1;
    const int end = row0 < rows ? max(ctx + tokens_of(last) + 1, 0) : 0;  // <= lk
    keys.first = max(ctx + tokens_of(row0) - p.window + 1, 0);
    const int head = (min(p.sinks, end) + box - 1) >> p.log2_box << p.log2_box;
    keys.gap = max((keys.first >> p.log2_box << p.log2_box) - head, 0);
    keys.head = keys.gap > 0 ? head : 0;
    keys.count = end - keys.gap;
  }
  // Keys that no row of the CTA sees: [blind0, blind1), and from keys.count on.
  const int blind0 = min(p.sinks, keys.count), blind1 = keys.first - keys.gap;
  // This CTA's steps: step0 .. step0 + steps - 1. Step i uses S/P buffer i % 2 for the i / 2-th time.
  const int all_steps = (keys.count + KEYS - 1) / KEYS;
  const int step0 = (rank * all_steps) >> log2_split, steps = (((rank + 1) * all_steps) >> log2_split) - step0;

  auto k_addr = [&](int s) -> uint32_t { return sbase + uint32_t(C::OFF_K + s * C::KV_BYTES); };
  auto v_addr = [&](int s) -> uint32_t { return sbase + uint32_t(C::OFF_V + s * C::KV_BYTES); };
  // Where row r (a key) of 128-byte piece pc of a stage sits: 8-row groups `gstride` bytes apart, pieces
  // `pstride` apart. Grouped copies land [group][piece][8 rows], one-piece copies [piece][row].
  const uint32_t gstride = p.grouped ? uint32_t(C::PIECES * 1024) : 1024u;
  const uint32_t pstride = p.grouped ? 1024u : uint32_t(KEYS * 128);
  auto stage = [](int i) -> int { return i % C::STAGES; };
  auto turn = [](int i) -> uint32_t { return uint32_t(i / C::STAGES) & 1u; };  // parity of the stage's use
  auto fail = [&]() {
    *abort_flag = 1;
    atomicOr(p.err, DEVERR_WAIT_TIMEOUT);
  };
  const uint32_t q_base = sbase + uint32_t(C::OFF_Q);

  if (row0 >= rows) {
    // no query row (of any CTA of the cluster)
  } else if (warp >= C::SOFTMAX_WARPS) {
    if constexpr (C::DEAL) regs_down<C::OTHER_REGS>();
    if (warp == C::K_WARP || warp == C::V_WARP) {
      // ---------------------------------------------------------------- copies
      // Lane c makes copy c of a step: a box of all pieces, or one piece of a box.
      const bool is_k = warp == C::K_WARP;
      const CUtensorMap* map = is_k ? &kmap : &vmap;
      const uint32_t full = bar(is_k ? Bars::K_FULL : Bars::V_FULL), empty = bar(is_k ? Bars::K_EMPTY : Bars::V_EMPTY);
      const uint32_t ring = is_k ? k_addr(0) : v_addr(0);
      const int per_box = p.grouped ? 1 : C::PIECES;
      const int my_box = lane / per_box, my_piece = lane - my_box * per_box;
      const int boxes = KEYS >> p.log2_box;
      const int32_t* trow = p.table + int64_t(b) * p.bt_stride;
      const int bs_mask = (1 << p.log2_bs) - 1;
      // Token of box `box_i` of step i, or -1 where it holds no key of the CTA.
      auto token_of = [&](int i, int box_i) -> int {
        const int u = (step0 + i) * KEYS + (box_i << p.log2_box);
        return i < steps && box_i < boxes && u < keys.count ? keys.token(u) : -1;
      };
      // Block ids, a window of 32 boxes at a time, the next window's under way: a load a step would be a load's
      // latency a step.
      const int log2_boxes = 6 - p.log2_box, span = 5 - log2_boxes;  // 2^span steps a window
      auto window_of = [&](int first) -> int {
        const int token = token_of(first + (lane >> log2_boxes), lane & (boxes - 1)), page = token >> p.log2_bs;
        return token >= 0 && page < p.max_blocks ? __ldg(trow + page) : -1;
      };
      int win = window_of(0), win_next = window_of(1 << span);
      bool ok = true;
      int done = 0;  // steps whose copies were issued
      const uint32_t bytes = uint32_t(C::PIECES / per_box) * 128u << p.log2_box;  // of a copy
      for (int i = 0; i < steps; ++i) {
        if (__any_sync(FULL_MASK, *abort_flag != 0)) break;
        const int s = stage(i);
        if (i > 0 && (i & ((1 << span) - 1)) == 0) {
          win = win_next;
          win_next = window_of(i + (1 << span));
        }
        const int tok = token_of(i, my_box);
        const int blk = __shfl_sync(FULL_MASK, win, ((i << log2_boxes) + my_box) & 31);
        // V's copies past the last key fill with zeros
        const bool copy = is_k ? tok >= 0 : my_box < boxes;
        const int copies = __popc(__ballot_sync(FULL_MASK, copy));
        const int in_block = tok >= 0 ? tok & bs_mask : 0;
        // a block outside the pool reads zeros: a coordinate past the last block's
        const int64_t known = blk >= 0 && blk < p.n_blocks ? blk : p.n_blocks;
        if (i >= C::STAGES && !warp_wait_phase(empty + uint32_t(s) * 8u, turn(i) ^ 1u, p.wait_ns)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(full + uint32_t(s) * 8u, uint32_t(copies) * bytes);
        if (copy) {
          const uint32_t dst = ring + uint32_t(s * C::KV_BYTES);
          if (p.grouped)
            tma_load_5d(dst + uint32_t(my_box << p.log2_box) * uint32_t(C::PIECES * 128), map, full + uint32_t(s) * 8u, 0, 0, 0,
                        h, int(known << (p.log2_bs - 3)) + (in_block >> 3));
          else
            tma_load_5d(dst + uint32_t(my_piece * KEYS + (my_box << p.log2_box)) * 128u, map, full + uint32_t(s) * 8u, 0,
                        in_block, h, my_piece, int(known));
        }
        ++done;
      }
      if (!ok && lane == 0) fail();
      // never leave with a copy in flight
      for (int i = max(done - C::STAGES, 0); i < done; ++i)
        warp_wait_phase(full + uint32_t(stage(i)) * 8u, turn(i), DRAIN_LIMIT_NS);
    } else if (warp == C::S_WARP) {
      // ---------------------------------------------------------------- S = Q K^T
      // The whole warp runs this loop and one elected lane issues, so descriptors and addresses stay
      // uniform over the warp and no operand of an MMA is moved on its own.
      constexpr uint32_t IDESC_S = tc::instr_desc_f16(BF16, ROWS, KEYS, false, false);
      bool ok = lane_wait(bar(Bars::Q_FULL), 0u, p.wait_ns);
      const uint64_t q_desc = tc::smem_desc(q_base, 16u, 1024u);
      const uint64_t k_desc = tc::smem_desc(k_addr(0), 16u, gstride);
      for (int i = 0; i < steps; ++i) {
        if (!__all_sync(FULL_MASK, ok && *abort_flag == 0)) break;
        const int s = stage(i), sb = i & 1;
        ok = ok && lane_wait(bar(Bars::K_FULL + s), turn(i), p.wait_ns);
        // once P V of the buffer's previous use has read its P
        if (i > 1) ok = ok && lane_wait(bar(Bars::O_DONE + sb), uint32_t(((i >> 1) - 1) & 1), p.wait_ns);
        __syncwarp();
        tc::fence_after_sync();
        const uint64_t b0 = k_desc + uint64_t((s * C::KV_BYTES) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks)
            tc::mma_f16_ss(tmem + uint32_t(sb * KEYS), q_desc + uint64_t(((ks >> 2) * (ROWS * 128) + (ks & 3) * 32) >> 4),
                           b0 + uint64_t((uint32_t(ks >> 2) * pstride + uint32_t((ks & 3) * 32)) >> 4), IDESC_S, ks > 0);
          tc::commit(bar(Bars::S_FULL + sb));
          tc::commit(bar(Bars::K_EMPTY + s));
        }
        __syncwarp();
      }
      if (!__all_sync(FULL_MASK, ok) && lane == 0) fail();
      if (elect_one()) tc::commit(bar(Bars::DRAIN));  // never leave with an MMA in flight
      __syncwarp();
      warp_wait_phase(bar(Bars::DRAIN), 0u, DRAIN_LIMIT_NS);
    } else {
      // ---------------------------------------------------------------- O += P V
      constexpr uint32_t IDESC_PV = tc::instr_desc_f16(BF16, ROWS, D, false, true);
      const uint64_t v_desc = tc::smem_desc(v_addr(0), pstride, gstride);
      bool ok = true;
      for (int i = 0; i < steps; ++i) {
        if (!__all_sync(FULL_MASK, ok && *abort_flag == 0)) break;
        const int s = stage(i), sb = i & 1;
        ok = ok && lane_wait(bar(Bars::V_FULL + s), turn(i), p.wait_ns);
        const int u0 = (step0 + i) * KEYS;
        if (__any_sync(FULL_MASK, (blind0 < blind1 && u0 < blind1 && u0 + KEYS > blind0) || u0 + KEYS > keys.count)) {
          auto clear = [&](int lo, int hi) {  // fewer than two copies' tokens
            lo = max(lo, u0) - u0;
            hi = min(hi, u0 + KEYS) - u0;
#pragma unroll 1
            for (int e = lane; e < (hi - lo) * (D / 8); e += 32) {
              const int r = lo + e / (D / 8), u = e % (D / 8);
              sts128(v_addr(s) + uint32_t(r >> 3) * gstride + uint32_t((r & 7) * 128) + uint32_t(u >> 3) * pstride +
                         uint32_t((u & 7) << 4),
                     0u, 0u, 0u, 0u);
            }
          };
          if (__all_sync(FULL_MASK, ok)) {  // (else copies may still be under way)
            clear(blind0, blind1);
            clear(keys.count, (keys.count + box - 1) >> p.log2_box << p.log2_box);
            fence_proxy_async_smem();
          }
          __syncwarp();
        }
        ok = ok && lane_wait(bar(Bars::P_FULL + sb), uint32_t((i >> 1) & 1), p.wait_ns);
        __syncwarp();
        tc::fence_after_sync();
        const uint64_t b0 = v_desc + uint64_t((s * C::KV_BYTES) >> 4);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < KEYS / 16; ++kk)
#pragma unroll
            for (int part = 0; part < 2; ++part)  // hi in the upper half of the buffer's columns, lo in the lower
              tc::mma_f16_ts(tmem + uint32_t(C::O_COL), tmem + uint32_t(sb * KEYS + (1 - part) * (KEYS / 2) + kk * 8),
                             b0 + uint64_t((uint32_t(kk) * 2u * gstride) >> 4), IDESC_PV, i > 0 || kk > 0 || part > 0);
          tc::commit(bar(Bars::O_DONE + sb));
          tc::commit(bar(Bars::V_EMPTY + s));
        }
        __syncwarp();
      }
      if (!__all_sync(FULL_MASK, ok) && lane == 0) fail();
      if (elect_one()) tc::commit(bar(Bars::DRAIN + 1));
      __syncwarp();
      warp_wait_phase(bar(Bars::DRAIN + 1), 0u, DRAIN_LIMIT_NS);
    }
  } else {
    // ---------------------------------------------------------------- softmax warps
    if constexpr (C::DEAL) regs_up<C::SOFTMAX_REGS>();
    const int r = tid;  // row of the block = TMEM lane
    const int n = row0 + r;
    const bool live = n < rows;
    // Q into its place: 16-byte units of 8 elements, all copies in flight at once.
    constexpr int LANES = D / 8, STEP = 128 / LANES;
    {
      const int u = tid % LANES;
      const int m0 = row0 + tid / LANES;
      int mt = tokens_of(m0), mh = m0 - mt * p.group;
      const int dt = tokens_of(STEP), dh = STEP - dt * p.group;
      const T* base = reinterpret_cast<const T*>(p.q) + int64_t(q_begin) * p.q_st + int64_t(h) * p.group * p.q_sh + u * 8;
#pragma unroll 4
      for (int rr = tid / LANES; rr < ROWS; rr += STEP) {
        const bool in = row0 + rr < rows;
        cp_async16(q_base + uint32_t((u >> 3) * (ROWS * 128)) + sw128(rr, u & 7),
                   base + (in ? int64_t(mt) * p.q_st + int64_t(mh) * p.q_sh : 0), in);
        mt += dt;
        mh += dh;
        if (mh >= p.group) {
          mh -= p.group;
          ++mt;
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (p.scale_log2 < 0.f) {  // a negative scale's sign goes into Q, so that the multiplier is never negative
      asm volatile("bar.sync 1, 128;" ::: "memory");  // the block's rows are in
      for (int u = 0; u < LANES; ++u) {
        const uint32_t at = q_base + uint32_t((u >> 3) * (ROWS * 128)) + sw128(r, u & 7);
        const uint4 w = lds128(at);
        sts128(at, w.x ^ 0x80008000u, w.y ^ 0x80008000u, w.z ^ 0x80008000u, w.w ^ 0x80008000u);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(Bars::Q_FULL));
    // never zero (a scale of 0 gives scores below 2^-80 instead), so that a hidden key's -inf stays one
    const float mul = fmaxf(fabsf(p.scale_log2), 1.2e-38f);
    // Keys of the CTA that this row sees: below `own_sinks`, and first_key .. last_key. Rows past the chunk's
    // end take the last row's, so that they ask for no mask of their own.
    const int at = ctx + tokens_of(min(n, rows - 1));  // position
    const int last_key = at - keys.gap;
    const int first_key = max(at - p.window + 1 - keys.gap, keys.head);
    const int own_sinks = min(p.sinks, last_key + 1);
    const uint32_t lane_base = tmem + (uint32_t(warp * 32) << 16);
    const uint32_t o_tmem = lane_base + uint32_t(C::O_COL);
    float m_run = -3.0e38f, l_run = 0.f;
    bool ok = true;
    const bool idle = row0 + warp * 32 >= rows;  // no row of this warp is one of the chunk's: whatever P is there serves
    for (int i = 0; i < steps; ++i) {
      const int sb = i & 1;
      // (where another role has failed no further S comes, and this wait ends by its limit)
      if (!warp_wait_phase(bar(Bars::S_FULL + sb), uint32_t(i >> 1) & 1u, p.wait_ns)) {
        ok = false;
        break;
      }
      if (idle) {
        if (lane == 0) mbar_arrive(bar(Bars::P_FULL + sb));
        continue;
      }
      tc::fence_after_sync();
      const uint32_t s_tmem = lane_base + uint32_t(sb * KEYS);
      // The row's scores stay in registers from the maximum to P, which is stored over the upper half of
      // their columns, its second part over the lower.
      float x[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS; c += 32)
        tc::ld_32x32b_x32(s_tmem + uint32_t(c), *reinterpret_cast<uint32_t(*)[32]>(x + c));
      tc::wait_ld();
      const int u0 = (step0 + i) * KEYS;
      // unless no key of the step is hidden from a row of the warp
      if (!__all_sync(FULL_MASK, u0 + KEYS - 1 <= last_key && (u0 >= first_key || u0 + KEYS <= own_sinks))) {
#pragma unroll
        for (int c = 0; c < KEYS; c += 32) {
          const int v0 = u0 + c;
          const uint32_t mask = bits(first_key - v0, last_key + 1 - v0) | bits(0, own_sinks - v0);
          if (__all_sync(FULL_MASK, mask == 0xffffffffu)) continue;
#pragma unroll
          for (int k = 0; k < 32; ++k) x[c + k] = mask & (1u << k) ? x[c + k] : -INFINITY;
        }
      }
      float t[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int k = 4; k < KEYS; k += 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fmaxf(fmaxf(t[e], x[k + e]), k + 4 + e < KEYS ? x[k + 4 + e] : t[e]);
      }
      const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      // mul >= 0: the maximum of the products is the product of the maximum
      const float tmax = top * mul;
      const bool move = tmax > m_run + (P_SHIFT + HEADROOM) || (m_run < -1.0e38f && tmax > m_run);
      if (__any_sync(FULL_MASK, move)) {
        const float ref = tmax - P_SHIFT;
        const float alpha = move ? ex2(m_run - ref) : 1.f;
        if (move) m_run = ref;
        l_run *= alpha;
        if (i > 0) {  // O *= alpha once P V of step i - 1 has landed
          if (!warp_wait_phase(bar(Bars::O_DONE + ((i - 1) & 1)), uint32_t((i - 1) >> 1) & 1u, p.wait_ns)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tc::ld_32x32b_x32(o_tmem + uint32_t(c), o);
            tc::wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tc::st_32x32b_x32(o_tmem + uint32_t(c), o);
          }
        }
      }
      const float2 mul2 = make_float2(mul, mul), neg_m2 = make_float2(-m_run, -m_run);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < KEYS; c += 32) {  // two keys to a column
        uint32_t w[16], rest[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          float2 e = fma2(make_float2(x[c + k], x[c + k + 1]), mul2, neg_m2);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], e);
          w[k >> 1] = E::pack2(e.x, e.y);
          float f[2];
          E::unpack2(w[k >> 1], f);
          rest[k >> 1] = E::pack2(e.x - f[0], e.y - f[1]);
        }
        st_32x32b_x16(s_tmem + uint32_t(KEYS / 2 + c / 2), w);
        st_32x32b_x16(s_tmem + uint32_t(c / 2), rest);
      }
      const float2 total = add2(sum[0], sum[1]);
      l_run += total.x + total.y;
      tc::wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Bars::P_FULL + sb));
    }
    if (ok && steps > 0)
      ok = warp_wait_phase(bar(Bars::O_DONE + ((steps - 1) & 1)), uint32_t((steps - 1) >> 1) & 1u, p.wait_ns);
    tc::fence_after_sync();
    const bool merge = ok && split > 1;
    if (!ok) {
      if (lane == 0) fail();
    } else if (split > 1) {
      // For the merge: m and l, and O over K and V, which no copy or MMA uses any more; 16-byte units of a row
      // permuted by the row, so that a quarter-warp's stores meet different banks.
      *reinterpret_cast<float2*>(smem + C::OFF_ML + r * 8) = make_float2(m_run, l_run);
      reinterpret_cast<float*>(smem + C::OFF_AGAIN)[r] = 0.f;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (steps > 0) {
          tc::ld_32x32b_x32(o_tmem + uint32_t(c), o);
          tc::wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (live) {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            sts128(sbase + uint32_t(C::OFF_O + r * (D * 4)) + uint32_t(((c / 4 + u) ^ (r & 7)) << 4), o[4 * u], o[4 * u + 1],
                   o[4 * u + 2], o[4 * u + 3]);
        }
      }
    } else {
      // a row that sees no key gives zeros
      const bool blind = last_key < 0 || !live;
      float whole = 0.f;  // stays 0 while the row's results are finite
      const float inv = blind ? 0.f : 1.f / l_run;
      // Through the warp's own 32 rows of the Q tile, which no MMA reads any more, so that a store
      // instruction writes whole rows instead of 16 bytes of 32 of them. The block's other warps copied Q
      // there: the first S says that their copies have landed, and without one a barrier has to.
      if (steps == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (steps > 0) {
          tc::ld_32x32b_x32(o_tmem + uint32_t(c), o);
          tc::wait_ld();
        }
        if (steps == 0 || blind) {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) whole = fmaf(__uint_as_float(o[k]), 0.f, whole);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = E::pack2(__uint_as_float(o[8 * u + 2 * k]) * inv, __uint_as_float(o[8 * u + 2 * k + 1]) * inv);
          const int at16 = c / 8 + u;
          sts128(q_base + uint32_t((at16 >> 3) * (ROWS * 128)) + sw128(r, at16 & 7), w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      constexpr int AT_ONCE = 32 / LANES;  // rows of a store
      const int u = lane % LANES, r0 = warp * 32 + lane / LANES, m0 = row0 + r0;
      int mt = tokens_of(m0), mh = m0 - mt * p.group;
      const int dt = tokens_of(AT_ONCE), dh = AT_ONCE - dt * p.group;
      T* base = reinterpret_cast<T*>(p.out) + int64_t(q_begin) * p.o_st + int64_t(h) * p.group * p.o_sh + u * 8;
#pragma unroll 4
      for (int i = 0; i < 32; i += AT_ONCE) {
        const uint4 w = lds128(q_base + uint32_t((u >> 3) * (ROWS * 128)) + sw128(r0 + i, u & 7));
        if (m0 + i < rows) *reinterpret_cast<uint4*>(base + int64_t(mt) * p.o_st + int64_t(mh) * p.o_sh) = w;
        mt += dt;
        mh += dh;
        if (mh >= p.group) {
          mh -= p.group;
          ++mt;
        }
      }
      unsigned again = __ballot_sync(FULL_MASK, whole != 0.f);  // (a NaN is not 0)
      while (again != 0u) {
        const int m = row0 + warp * 32 + __ffs(again) - 1, t = tokens_of(m);
        again &= again - 1u;
        __syncwarp();  // this warp has stored the row
        row_again<T, D>(p, b, h, lk, q_begin + t, h * p.group + m - t * p.group, ctx + t);
      }
    }
    // The cluster's merge, in the branch of the warps that have registers for it.
    if (split > 1) {
      __syncwarp();
      cluster_sync();
      const int live_rows = min(ROWS, rows - row0);
      const int mine = merge ? (live_rows - rank + split - 1) >> log2_split : 0;  // (0: its waits ran out)
      // Row by row, the CTAs' rows dealt in turn: a row's 16-byte units over the lanes.
      constexpr int UNITS = D / 4;
      // (all threads of a row's warp take every turn, so that they can vote on it)
      for (int e0 = 0; e0 < mine * UNITS; e0 += 128) {
        const int e = e0 + tid;
        const bool in = e < mine * UNITS;
        const int r = in ? (e / UNITS << log2_split) + rank : rank, u = e % UNITS;
        const uint32_t ml = sbase + uint32_t(C::OFF_ML + r * 8);
        const uint32_t o = sbase + uint32_t(C::OFF_O + r * (D * 4)) + uint32_t((u ^ (r & 7)) << 4);
        float2 part[8];
        float4 v[8];
        float M = -3.0e38f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k < split) {
            part[k] = ld_cluster_v2(cluster_addr(ml, k));
            v[k] = ld_cluster_v4(cluster_addr(o, k));
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < split) M = fmaxf(M, part[k].x);
        float L = 0.f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k < split) {
            const float f = ex2(part[k].x - M);
            L = fmaf(f, part[k].y, L);
            sum.x = fmaf(f, v[k].x, sum.x);
            sum.y = fmaf(f, v[k].y, sum.y);
            sum.z = fmaf(f, v[k].z, sum.z);
            sum.w = fmaf(f, v[k].w, sum.w);
          }
        }
        const int n = row0 + r, t = tokens_of(n);
        const float inv = ctx + t < 0 ? 0.f : 1.f / L;  // a row that sees no key gives zeros
        uint2 w;
        w.x = E::pack2(sum.x * inv, sum.y * inv);
        w.y = E::pack2(sum.z * inv, sum.w * inv);
        if (in)
          *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + int64_t(q_begin + t) * p.o_st +
                                    int64_t(h * p.group + n - t * p.group) * p.o_sh + u * 4) = w;
        // A row that is not finite is noted, and computed again once every thread has stored its part.
        const float whole = sum.x * 0.f + sum.y * 0.f + (sum.z * 0.f + sum.w * 0.f) + inv * 0.f;
        if (in && whole != 0.f) reinterpret_cast<float*>(smem + C::OFF_AGAIN)[r] = 1.f;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      for (int i = warp; i < mine; i += C::SOFTMAX_WARPS) {
        const int r = (i << log2_split) + rank, m = row0 + r, t = tokens_of(m);
        if (reinterpret_cast<const float*>(smem + C::OFF_AGAIN)[r] != 0.f)
          row_again<T, D>(p, b, h, lk, q_begin + t, h * p.group + m - t * p.group, ctx + t);
      }
      __syncwarp();
      cluster_sync();  // nothing of this CTA is read any more
    }
  }
  if (split > 1 && (warp >= C::SOFTMAX_WARPS || row0 >= rows)) {  // the other warps at the cluster's barriers
    __syncwarp();
    cluster_sync();
    cluster_sync();
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == C::S_WARP) {
    __syncwarp();
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <typename T, int D>
cudaError_t launch_t(const WindowPrefillParams& p0, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
  using C = Cfg<D>;
  auto fn = pd_window_prefill_kernel<T, D>;
  static SmemRaised raised{};
  const cudaError_t err = raise_smem_limit(fn, C::SMEM, raised);
  if (err != cudaSuccess) return err;
  WindowPrefillParams p = p0;
  // With 2^(31 + l) / group rounded up, group <= 2^l, the product's excess stays below one part in n < 2^31.
  int l = 0;
  while ((int64_t(1) << l) < p.group) ++l;
  p.group_shift = 31 + l;
  p.group_mul = uint32_t(((uint64_t(1) << p.group_shift) + p.group - 1) / p.group);
  const int64_t rows = int64_t(p.max_seqlen_q) * p.group;
  const int64_t blocks = (rows + ROWS - 1) / ROWS;
  const int64_t ctas = blocks * p.batch * p.n_kv_head;
  // A block's steps are shared while the GPU has room for the CTAs and each keeps two steps or more (at most: the
  // lengths are on the device).
  const int64_t most_keys = std::min<int64_t>(p.capacity, int64_t(p.window) + p.sinks + ROWS / p.group + 1);
  int log2_split = 0;
  while (log2_split < 3 && (ctas << (log2_split + 1)) <= C::CTAS * int64_t(p.sms) &&
         most_keys >= int64_t(2 * KEYS) << (log2_split + 1))
    ++log2_split;
  if ((ctas << log2_split) > 0x7fffffff) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1u << log2_split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas << log2_split));
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = log2_split > 0 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, p, kmap, vmap, int(blocks), log2_split);
}

template <typename T>
cudaError_t launch_d(const WindowPrefillParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap, int head_dim,
                     cudaStream_t stream) {
  switch (head_dim) {
    case 64: return launch_t<T, 64>(p, kmap, vmap, stream);
    case 128: return launch_t<T, 128>(p, kmap, vmap, stream);
    case 256: return launch_t<T, 256>(p, kmap, vmap, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_window_prefill(const WindowPrefillParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap,
                                  int dtype, int head_dim, cudaStream_t stream) {
  return dtype == PD_BF16 ? launch_d<__nv_bfloat16>(p, kmap, vmap, head_dim, stream)
                          : launch_d<__half>(p, kmap, vmap, head_dim, stream);
}

}  // namespace pd
