// pd_window_prefill.cu -- attention of query chunks over a window of a paged cache on the 5th-generation
// tensor cores (tcgen05 / TMEM) for sm_100a: bf16 / fp16 pools, head_dim 64, 128 or 256, any group.
//
// Query token t of a chunk of S tokens sits at i = seqlen - S + t and sees key j iff j <= i and
// (i - j < window or j < sinks): out = softmax(q K^T scale) V over those, fp32 softmax and accumulation.
// A query row is a (token, q head of the kv head's group) pair, token-major, so a group's heads share every
// K/V tile.
//
// How (one CTA = NQ blocks of 128 query rows of one row's chunk and one kv head):
//  * The keys that some query row of the CTA sees -- sinks and window, in whole copies of `box` tokens -- are
//    numbered without the gap between them and cut into tiles of KT keys, so a few sinks cost a copy, not a tile.
//  * One warp streams K and V tiles by TMA into two rings of stages, a lane a copy, block ids one tile ahead. No block
//    without a visible token is looked up; where the last tile ends early, V is filled with zeros from outside the pool.
//  * One warp issues S = Q K^T (M 128, N 64 keys, K head_dim) into one of a block's two S buffers in TMEM, another O += P V
//    with P read from TMEM, where the softmax wrote it over the S it came from; so a block's next S is there when its
//    softmax is done with one. A third warp zeroes the V of tokens that a tile's copies hold but no row of the CTA sees,
//    so that whatever bytes they hold never reach O.
//  * 4 softmax warps per block of query rows, one thread per row (TMEM lane = row): maximum over the row's
//    scores, P = 2^(s - m + 7), and the fp32 sum; no exchange between threads. The maximum moves only when a tile
//    passes it by 2^8, so rescaling O in TMEM is rare.
//  With NQ = 2 a tile serves 256 rows; at head_dim 256 TMEM holds one block (O takes 256 of its 512 columns).
//  * P enters as two 16-bit operands, P = hi + lo: 2^-17 of the weighted mean of |v| in bf16 and 2^-22 in fp16, as
//    the causal chunk kernel (pd_prefill_tc.cu) has it; one bf16 part alone would be off by as much as the result's
//    own rounding. The factor 2^7, which the sums carry too, keeps fp16 weights down to 2^-21 normal numbers.
//  * Every wait is bounded; a role whose wait runs out records DEVERR_WAIT_TIMEOUT and raises the CTA's abort
//    flag, every role then leaves its loop, copies and MMAs in flight are waited for, and the CTA frees its TMEM.
#include "paged_decode.h"
#include "pd_smem_limit.cuh"
#include "pd_tcgen05.cuh"
#include "pd_tile.cuh"
#include "pd_window.cuh"

#include <type_traits>

namespace pd {

namespace {

constexpr int ROWS = 128;  // query rows of a block (the MMA's M)
constexpr int KEYS = 64;   // keys of a softmax step (the S MMA's N)
constexpr float P_SHIFT = 7.f, HEADROOM = 8.f;

template <int D>
struct Cfg {
  static constexpr int NQ = D <= 128 ? 2 : 1;     // blocks of query rows per CTA
  static constexpr int KT = D <= 128 ? 128 : 64;  // keys of a tile of K or V in shared memory
  static constexpr int STEPS = KT / KEYS;         // softmax steps of a tile
  static constexpr int PIECES = D / 64;
  static constexpr int SOFTMAX_WARPS = 4 * NQ;
  static constexpr int TMA_WARP = SOFTMAX_WARPS;
  static constexpr int CLEAR_WARP = SOFTMAX_WARPS + 1;
  static constexpr int S_WARP = SOFTMAX_WARPS + 2;
  static constexpr int THREADS = (SOFTMAX_WARPS + 4) * 32;  // and a warp for P V
  // With two blocks, registers are dealt anew between the groups, so that a softmax thread holds a row's KT
  // scores and P; with one, every thread has enough.
  static constexpr bool SPLIT = NQ == 2;
  static constexpr int LAUNCH_REGS = 65536 / THREADS / 8 * 8;
  static constexpr int SOFTMAX_REGS = 208;
  static constexpr int OTHER_REGS = 80;
  static_assert(!SPLIT || SOFTMAX_WARPS * SOFTMAX_REGS + 4 * OTHER_REGS <= THREADS / 32 * LAUNCH_REGS,
                "a split above the launch's registers would wait for ever");
  static constexpr int STAGES = 2;  // tiles of K, and of V
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int KV_BYTES = KT * D * 2;
  static constexpr int O_COL = NQ * 2 * KEYS;  // behind two S/P buffers a block
  static constexpr int TMEM_COLS = 512;
  static_assert(O_COL + NQ * D <= TMEM_COLS, "TMEM columns");
  static constexpr int OFF_Q = 1024;  // barriers and flags before it
  static constexpr int OFF_K = OFF_Q + NQ * Q_BYTES;
  static constexpr int OFF_V = OFF_K + STAGES * KV_BYTES;
  static constexpr int SMEM = OFF_V + STAGES * KV_BYTES + 1024;  // + run-time 1 KB alignment
  static_assert(SMEM <= 232448, "shared memory per CTA");
};

// Barrier slots (8 bytes each) at the front of shared memory.
struct Bars {
  static constexpr int K_FULL = 0;    // [2] K tile landed (transaction bytes)
  static constexpr int V_FULL = 2;    // [2]
  static constexpr int K_EMPTY = 4;   // [2] every S of the tile completed (commit)
  static constexpr int V_EMPTY = 6;   // [2] every P V of the tile completed (commit)
  static constexpr int V_READY = 8;   // [2] V tile's unseen tokens are zeros
  static constexpr int Q_FULL = 10;   // Q stored: one arrival per softmax warp
  static constexpr int DRAIN = 11;    // [2]
  static constexpr int S_FULL = 13;   // [4] S buffer written (commit)
  static constexpr int P_FULL = 17;   // [4] P written over it, O rescaled: one arrival per softmax warp
  static constexpr int O_DONE = 21;   // [4] P V that read the buffer completed (commit)
  static constexpr int TMEM_SLOT = 200;  // byte offsets
  static constexpr int ABORT = 208;
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

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::THREADS, 1)
    pd_window_prefill_kernel(const __grid_constant__ WindowPrefillParams p, const __grid_constant__ CUtensorMap kmap,
                             const __grid_constant__ CUtensorMap vmap, int blocks) {
  using C = Cfg<D>;
  using E = Elem<T>;
  constexpr int NQ = C::NQ, KT = C::KT;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t raw = smem_addr(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t sbase = smem_addr(smem);
  auto bar = [&](int slot) -> uint32_t { return sbase + uint32_t(slot) * 8u; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Bars::ABORT);

  if (warp == C::S_WARP) {
    if (lane == 0) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar(Bars::K_FULL + i), 1);
        mbar_init(bar(Bars::V_FULL + i), 1);
        mbar_init(bar(Bars::K_EMPTY + i), 1);
        mbar_init(bar(Bars::V_EMPTY + i), 1);
        mbar_init(bar(Bars::V_READY + i), 1);
        mbar_init(bar(Bars::DRAIN + i), 1);
      }
      for (int i = 0; i < 2 * NQ; ++i) {
        mbar_init(bar(Bars::S_FULL + i), 1);
        mbar_init(bar(Bars::P_FULL + i), 4);
        mbar_init(bar(Bars::O_DONE + i), 1);
      }
      mbar_init(bar(Bars::Q_FULL), C::SOFTMAX_WARPS);
      *abort_flag = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tc::tmem_alloc(sbase + Bars::TMEM_SLOT, C::TMEM_COLS);
    tc::tmem_relinquish();
  }

  // Query blocks slowest and last ones first: a prompt's first blocks have the fewest keys.
  const int pairs = p.batch * p.n_kv_head;
  const int b = int(blockIdx.x) % p.batch;
  const int h = (int(blockIdx.x) / p.batch) % p.n_kv_head;
  const int qblock = blocks - 1 - int(blockIdx.x) / pairs;
  const int q_begin = min(max(__ldg(p.cu_q + b), 0), p.total_q);
  const int chunk = max(min(max(__ldg(p.cu_q + b + 1), 0), p.total_q) - q_begin, 0);
  const int sq = min(chunk, p.max_seqlen_q);
  int lk = __ldg(p.seqlen + b);
  lk = lk < 0 ? 0 : (lk > p.capacity ? p.capacity : lk);
  const int rows = sq * p.group;
  const int row0 = qblock * NQ * ROWS;  // first query row of the CTA
  const int ctx = lk - chunk;           // position of the chunk's first token
  const int box = 1 << p.log2_box;
  // What the CTA's rows see: up to its last token, from its first token's window on, and the sinks.
  Keys keys;
  int steps[NQ], most = 0;  // softmax steps of a block, tiles of the CTA
  {
    const int last = min(row0 + NQ * ROWS, rows) - 1;
    const int end = row0 < rows ? max(ctx + last / p.group + 1, 0) : 0;  // <= lk
    keys.first = max(ctx + row0 / p.group - p.window + 1, 0);
    const int head = (min(p.sinks, end) + box - 1) >> p.log2_box << p.log2_box;
    keys.gap = max((keys.first >> p.log2_box << p.log2_box) - head, 0);
    keys.head = keys.gap > 0 ? head : 0;
    keys.count = end - keys.gap;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int r0 = row0 + q * ROWS;
      const int kend = r0 < rows ? max(ctx + (min(r0 + ROWS, rows) - 1) / p.group + 1, 0) - keys.gap : 0;
      steps[q] = max((kend + KEYS - 1) / KEYS, 0);
      most = max(most, (steps[q] + C::STEPS - 1) / C::STEPS);
    }
  }
  // Keys that no row of the CTA sees: [blind0, blind1), and from keys.count on.
  const int blind0 = min(p.sinks, keys.count), blind1 = keys.first - keys.gap;

  // Every role meets here once, with its first loads already in flight; returns the TMEM address.
  auto meet = [&]() -> uint32_t {
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    return *reinterpret_cast<volatile uint32_t*>(smem + Bars::TMEM_SLOT);
  };
  uint32_t tmem;
  auto k_addr = [&](int s) -> uint32_t { return sbase + uint32_t(C::OFF_K + s * C::KV_BYTES); };
  auto v_addr = [&](int s) -> uint32_t { return sbase + uint32_t(C::OFF_V + s * C::KV_BYTES); };
  // Where row r (a key) of 128-byte piece pc of a K/V tile sits: 8-row groups `gstride` bytes apart, pieces
  // `pstride` apart. Grouped copies land [group][piece][8 rows], one-piece copies [piece][row].
  const uint32_t gstride = p.grouped ? uint32_t(C::PIECES * 1024) : 1024u;
  const uint32_t pstride = p.grouped ? 1024u : uint32_t(KT * 128);
  auto fail = [&]() {
    *abort_flag = 1;
    atomicOr(p.err, DEVERR_WAIT_TIMEOUT);
  };

  // Step u of block q uses S/P buffer 2 q + u % 2 for the u / 2-th time.
  const int all_steps = NQ == 2 ? max(steps[0], steps[NQ - 1]) : steps[0];

  if (row0 >= rows) {  // no query row
    tmem = meet();
  } else if (warp >= C::SOFTMAX_WARPS) {
    if constexpr (C::SPLIT) regs_down<C::OTHER_REGS>();
    if (warp == C::TMA_WARP) {
      // ---------------------------------------------------------------- copies
      // Lane c makes copy c of a tile: a box of all pieces, or one piece of a box.
      const int per_box = p.grouped ? 1 : C::PIECES;
      const int my_box = lane / per_box, my_piece = lane - my_box * per_box;
      const int boxes = KT >> p.log2_box;
      const int32_t* trow = p.table + int64_t(b) * p.bt_stride;
      const int bs_mask = (1 << p.log2_bs) - 1;
      // Token of this lane's copy of tile j, or -1 where the copy holds no key of the CTA.
      auto token_of = [&](int j) -> int {
        const int u = j * KT + (my_box << p.log2_box);
        return j < most && my_box < boxes && u < keys.count ? keys.token(u) : -1;
      };
      auto block_of = [&](int token) -> int {
        const int page = token >> p.log2_bs;
        return token >= 0 && page < p.max_blocks ? __ldg(trow + page) : -1;
      };
      int tok = token_of(0);
      int blk = block_of(tok), tok_next = token_of(1);
      int blk_next = block_of(tok_next);
      tmem = meet();
      bool ok = true;
      int k_done = 0, v_done = 0;  // tiles whose copies were issued
      const uint32_t bytes = uint32_t(C::PIECES / per_box) * 128u << p.log2_box;  // of a copy
      for (int j = 0; ok && j < most; ++j) {
        if (__any_sync(FULL_MASK, *abort_flag != 0)) break;
        const int s = j % C::STAGES;
        const uint32_t freed = uint32_t((j / C::STAGES - 1) & 1);  // phase of the stage's previous use
        const int k_copies = __popc(__ballot_sync(FULL_MASK, tok >= 0));
        const int in_block = tok >= 0 ? tok & bs_mask : 0;
        // a block outside the pool reads zeros: a coordinate past the last block's
        const int64_t known = blk >= 0 && blk < p.n_blocks ? blk : p.n_blocks;
        auto copy = [&](const CUtensorMap* map, uint32_t full, uint32_t dst, bool mine, int copies) {
          if (lane == 0) mbar_arrive_expect_tx(full, uint32_t(copies) * bytes);
          if (mine) {
            if (p.grouped)
              tma_load_5d(dst + uint32_t(my_box << p.log2_box) * uint32_t(C::PIECES * 128), map, full, 0, 0, 0, h,
                          int(known << (p.log2_bs - 3)) + (in_block >> 3));
            else
              tma_load_5d(dst + uint32_t(my_piece * KT + (my_box << p.log2_box)) * 128u, map, full, 0, in_block, h,
                          my_piece, int(known));
          }
        };
        if (j >= C::STAGES && !warp_wait_phase(bar(Bars::K_EMPTY + s), freed, p.wait_ns)) {
          ok = false;
          break;
        }
        copy(&kmap, bar(Bars::K_FULL + s), k_addr(s), tok >= 0, k_copies);
        ++k_done;
        if (j >= C::STAGES && !warp_wait_phase(bar(Bars::V_EMPTY + s), freed, p.wait_ns)) {
          ok = false;
          break;
        }
        copy(&vmap, bar(Bars::V_FULL + s), v_addr(s), my_box < boxes, boxes * per_box);
        ++v_done;
        tok = tok_next;
        blk = blk_next;
        tok_next = token_of(j + 2);
        blk_next = block_of(tok_next);
      }
      if (!ok && lane == 0) fail();
      // never leave with a copy in flight
      for (int j = max(k_done - C::STAGES, 0); j < k_done; ++j)
        warp_wait_phase(bar(Bars::K_FULL + j % C::STAGES), uint32_t((j / C::STAGES) & 1), DRAIN_LIMIT_NS);
      for (int j = max(v_done - C::STAGES, 0); j < v_done; ++j)
        warp_wait_phase(bar(Bars::V_FULL + j % C::STAGES), uint32_t((j / C::STAGES) & 1), DRAIN_LIMIT_NS);
    } else if (warp == C::CLEAR_WARP) {
      // ---------------------------------------------------------------- V of tokens that no row sees
      tmem = meet();
      bool ok = true;
      for (int j = 0; j < most; ++j) {
        const int s = j & 1;
        if (__any_sync(FULL_MASK, *abort_flag != 0)) break;
        if (!warp_wait_phase(bar(Bars::V_FULL + s), uint32_t((j >> 1) & 1), p.wait_ns)) {
          ok = false;
          break;
        }
        const int u0 = j * KT;
        auto clear = [&](int lo, int hi) {  // fewer than two copies' tokens
          lo = max(lo, u0) - u0;
          hi = min(hi, u0 + KT) - u0;
          if (lo >= hi) return;
          for (int i = lane; i < (hi - lo) * (D / 8); i += 32) {
            const int r = lo + i / (D / 8), u = i % (D / 8);
            sts128(v_addr(s) + uint32_t(r >> 3) * gstride + uint32_t((r & 7) * 128) + uint32_t(u >> 3) * pstride +
                       uint32_t((u & 7) << 4),
                   0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        };
        clear(blind0, blind1);
        clear(keys.count, (keys.count + box - 1) >> p.log2_box << p.log2_box);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(Bars::V_READY + s));
      }
      if (!ok && lane == 0) fail();
    } else if (warp == C::S_WARP) {
      // ---------------------------------------------------------------- S = Q K^T
      // The whole warp runs this loop and one elected lane issues, so descriptors and addresses stay
      // uniform over the warp and no operand of an MMA is moved on its own.
      tmem = meet();
      if (most > 0) {
        constexpr uint32_t IDESC_S = tc::instr_desc_f16(BF16, ROWS, KEYS, false, false);
        bool ok = lane_wait(bar(Bars::Q_FULL), 0u, p.wait_ns);
        const uint64_t q_desc = tc::smem_desc(sbase + C::OFF_Q, 16u, 1024u);
        const uint64_t k_desc = tc::smem_desc(k_addr(0), 16u, gstride);
        for (int u = 0; u < all_steps; ++u) {
          if (!__all_sync(FULL_MASK, ok && *abort_flag == 0)) break;
          const int j = u / C::STEPS, s = j & 1, part = u % C::STEPS;
          if (part == 0) ok = ok && lane_wait(bar(Bars::K_FULL + s), uint32_t((j >> 1) & 1), p.wait_ns);
          const uint64_t b0 = k_desc + uint64_t((s * C::KV_BYTES) >> 4) + uint64_t((uint32_t(part * (KEYS / 8)) * gstride) >> 4);
          const bool last = part == C::STEPS - 1 || u == all_steps - 1;  // of the tile
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if (u >= steps[q]) continue;
            const int sb = 2 * q + (u & 1);
            // once P V of the buffer's previous use has read its P
            if (u > 1) ok = ok && lane_wait(bar(Bars::O_DONE + sb), uint32_t(((u >> 1) - 1) & 1), p.wait_ns);
            __syncwarp();
            tc::fence_after_sync();
            const bool frees = last && (q == NQ - 1 || u >= steps[NQ - 1]);  // the last S of this K tile
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < D / 16; ++ks)
                tc::mma_f16_ss(tmem + uint32_t(sb * KEYS),
                               q_desc + uint64_t((q * C::Q_BYTES + (ks >> 2) * (ROWS * 128) + (ks & 3) * 32) >> 4),
                               b0 + uint64_t((uint32_t(ks >> 2) * pstride + uint32_t((ks & 3) * 32)) >> 4), IDESC_S, ks > 0);
              tc::commit(bar(Bars::S_FULL + sb));
              if (frees) tc::commit(bar(Bars::K_EMPTY + s));
            }
            __syncwarp();
          }
        }
        if (!__all_sync(FULL_MASK, ok) && lane == 0) fail();
        if (elect_one()) tc::commit(bar(Bars::DRAIN));  // never leave with an MMA in flight
        __syncwarp();
        warp_wait_phase(bar(Bars::DRAIN), 0u, DRAIN_LIMIT_NS);
      }
    } else {
      // ---------------------------------------------------------------- O += P V
      tmem = meet();
      if (most > 0) {
        constexpr uint32_t IDESC_PV = tc::instr_desc_f16(BF16, ROWS, D, false, true);
        const uint64_t v_desc = tc::smem_desc(v_addr(0), pstride, gstride);
        bool ok = true;
        for (int u = 0; u < all_steps; ++u) {
          if (!__all_sync(FULL_MASK, ok && *abort_flag == 0)) break;
          const int j = u / C::STEPS, s = j & 1, part = u % C::STEPS;
          const uint32_t landed = uint32_t((j >> 1) & 1);
          if (part == 0)
            ok = ok && lane_wait(bar(Bars::V_FULL + s), landed, p.wait_ns) &&
                 lane_wait(bar(Bars::V_READY + s), landed, p.wait_ns);
          const uint64_t b0 = v_desc + uint64_t((s * C::KV_BYTES) >> 4) + uint64_t((uint32_t(part * (KEYS / 8)) * gstride) >> 4);
          const bool last = part == C::STEPS - 1 || u == all_steps - 1;
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if (u >= steps[q]) continue;
            const int sb = 2 * q + (u & 1);
            const bool frees = last && (q == NQ - 1 || u >= steps[NQ - 1]);
            ok = ok && lane_wait(bar(Bars::P_FULL + sb), uint32_t((u >> 1) & 1), p.wait_ns);
            __syncwarp();
            tc::fence_after_sync();
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < KEYS / 16; ++kk)
#pragma unroll
                for (int i = 0; i < 2; ++i)  // hi in the upper half of the buffer's columns, lo in the lower
                  tc::mma_f16_ts(tmem + uint32_t(C::O_COL + q * D), tmem + uint32_t(sb * KEYS + (1 - i) * (KEYS / 2) + kk * 8),
                                 b0 + uint64_t((uint32_t(kk) * 2u * gstride) >> 4), IDESC_PV, u > 0 || kk > 0 || i > 0);
              tc::commit(bar(Bars::O_DONE + sb));
              if (frees) tc::commit(bar(Bars::V_EMPTY + s));
            }
            __syncwarp();
          }
        }
        if (!__all_sync(FULL_MASK, ok) && lane == 0) fail();
        if (elect_one()) tc::commit(bar(Bars::DRAIN + 1));
        __syncwarp();
        warp_wait_phase(bar(Bars::DRAIN + 1), 0u, DRAIN_LIMIT_NS);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax warps
    if constexpr (C::SPLIT) regs_up<C::SOFTMAX_REGS>();
    const int q = warp >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the block = TMEM lane
    const int n = row0 + q * ROWS + r;
    const bool live = n < rows;
    // Q into its place: 16-byte units of 8 elements, all copies in flight at once.
    constexpr int LANES = D / 8, STEP = 128 / LANES;
    const uint32_t q_base = sbase + uint32_t(C::OFF_Q + q * C::Q_BYTES);
    {
      const int t = tid - q * 128, u = t % LANES;
      const int m0 = row0 + q * ROWS + t / LANES;
      int mt = m0 / p.group, mh = m0 - mt * p.group;
      const int dt = STEP / p.group, dh = STEP - dt * p.group;
      const T* base = reinterpret_cast<const T*>(p.q) + int64_t(q_begin) * p.q_st + int64_t(h) * p.group * p.q_sh + u * 8;
#pragma unroll 4
      for (int rr = t / LANES; rr < ROWS; rr += STEP) {
        const bool in = row0 + q * ROWS + rr < rows;
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
    tmem = meet();
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (p.scale_log2 < 0.f) {  // a negative scale's sign goes into Q, so that the multiplier is never negative
      asm volatile("bar.sync %0, 128;" ::"r"(1 + q) : "memory");  // the block's rows are in
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
    const int at = ctx + min(n, rows - 1) / p.group;  // position
    const int last_key = at - keys.gap;
    const int first_key = max(at - p.window + 1 - keys.gap, keys.head);
    const int own_sinks = min(p.sinks, last_key + 1);
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t o_tmem = lane_base + uint32_t(C::O_COL + q * D);
    float m_run = -3.0e38f, l_run = 0.f;
    bool ok = true;
    const int mine = q == 0 ? steps[0] : steps[NQ - 1];
    for (int j = 0; j < mine; ++j) {
      const int sb = 2 * q + (j & 1);
      const uint32_t ph = uint32_t(j >> 1) & 1u;
      if (__any_sync(FULL_MASK, *abort_flag != 0) || !warp_wait_phase(bar(Bars::S_FULL + sb), ph, p.wait_ns)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      const uint32_t s_tmem = lane_base + uint32_t(sb * KEYS);
      // no key of the step is hidden from a row of the warp
      const int u0 = j * KEYS;
      const bool open = __all_sync(FULL_MASK, u0 + KEYS - 1 <= last_key && (u0 >= first_key || u0 + KEYS <= own_sinks));
      // The row's scores stay in registers from the maximum to P, which is stored over the upper half of
      // their columns, its second part over the lower.
      float x[KEYS];
#pragma unroll
      for (int c = 0; c < KEYS; c += 32)
        tc::ld_32x32b_x32(s_tmem + uint32_t(c), *reinterpret_cast<uint32_t(*)[32]>(x + c));
      tc::wait_ld();
      if (!open) {
#pragma unroll
        for (int c = 0; c < KEYS; c += 32) {
          const int v0 = u0 + c;
          const uint32_t mask = bits(first_key - v0, last_key + 1 - v0) | bits(0, own_sinks - v0);
          if (__all_sync(FULL_MASK, mask == 0xffffffffu)) continue;
#pragma unroll
          for (int i = 0; i < 32; ++i) x[c + i] = mask & (1u << i) ? x[c + i] : -INFINITY;
        }
      }
      float t[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < KEYS; i += 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = fmaxf(fmaxf(t[k], x[i + k]), i + 4 + k < KEYS ? x[i + 4 + k] : t[k]);
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
        if (j > 0) {  // O *= alpha once P V of step j - 1 has landed
          if (!warp_wait_phase(bar(Bars::O_DONE + 2 * q + ((j - 1) & 1)), uint32_t((j - 1) >> 1) & 1u, p.wait_ns)) {
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
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
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
        for (int i = 0; i < 32; i += 2) {
          float2 e = fma2(make_float2(x[c + i], x[c + i + 1]), mul2, neg_m2);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
          w[i >> 1] = E::pack2(e.x, e.y);
          float f[2];
          E::unpack2(w[i >> 1], f);
          rest[i >> 1] = E::pack2(e.x - f[0], e.y - f[1]);
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
    if (ok && mine > 0) {
      ok = warp_wait_phase(bar(Bars::O_DONE + 2 * q + ((mine - 1) & 1)), uint32_t((mine - 1) >> 1) & 1u, p.wait_ns);
    }
    if (!ok) {
      if (lane == 0) fail();
    } else {
      tc::fence_after_sync();
      // l is 0 or NaN-free of the hidden: a row that sees no key gives zeros
      const float inv = last_key < 0 ? 0.f : 1.f / l_run;
      const bool blind = last_key < 0 || !live;
      // Through the warp's own 32 rows of the Q tile, which no MMA reads any more, so that a store
      // instruction writes whole rows instead of 16 bytes of 32 of them. The block's other warps copied Q
      // there: the first S says that their copies have landed, and without one a barrier has to.
      if (mine == 0) asm volatile("bar.sync %0, 128;" ::"r"(1 + q) : "memory");
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (mine > 0) {
          tc::ld_32x32b_x32(o_tmem + uint32_t(c), o);
          tc::wait_ld();
        }
        if (mine == 0 || blind) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = E::pack2(__uint_as_float(o[8 * u + 2 * i]) * inv, __uint_as_float(o[8 * u + 2 * i + 1]) * inv);
          const int at16 = c / 8 + u;
          sts128(q_base + uint32_t((at16 >> 3) * (ROWS * 128)) + sw128(r, at16 & 7), w[0], w[1], w[2], w[3]);
        }
      }
      __syncwarp();
      constexpr int AT_ONCE = 32 / LANES;  // rows of a store
      const int u = lane % LANES, r0 = (warp & 3) * 32 + lane / LANES, m0 = row0 + q * ROWS + r0;
      int mt = m0 / p.group, mh = m0 - mt * p.group;
      const int dt = AT_ONCE / p.group, dh = AT_ONCE - dt * p.group;
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
    }
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
cudaError_t launch_t(const WindowPrefillParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap, cudaStream_t stream) {
  using C = Cfg<D>;
  auto fn = pd_window_prefill_kernel<T, D>;
  static SmemRaised raised{};
  const cudaError_t err = raise_smem_limit(fn, C::SMEM, raised);
  if (err != cudaSuccess) return err;
  const int64_t rows = int64_t(p.max_seqlen_q) * p.group;
  const int64_t blocks = (rows + C::NQ * ROWS - 1) / (C::NQ * ROWS);
  const int64_t ctas = blocks * p.batch * p.n_kv_head;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  fn<<<dim3(unsigned(ctas)), C::THREADS, C::SMEM, stream>>>(p, kmap, vmap, int(blocks));
  return cudaGetLastError();
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
