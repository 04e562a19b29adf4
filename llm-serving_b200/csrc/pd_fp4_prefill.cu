// pd_fp4_prefill.cu -- causal attention of query chunks over 4-bit pages on the 5th-generation
// tensor cores (tcgen05 / TMEM) for sm_100a: fp16 / bf16 queries, head_dim 64, 128 or 256, any group.
//
// The same function as pd_fp4_attend.cuh (out = softmax(q K^T scale) V over each query's visible
// keys, fp32 softmax and accumulation) for chunks whose products outweigh the cache's bytes. A query
// row is a (token, q head of the kv head's group) pair, token-major, so a group's heads share
// every decoded K/V tile.
//
// How (one CTA = NQ blocks of 128 query rows of one row's chunk and one kv head):
//  * 4 decoding warps turn the next KT keys of the 4-bit pages into fp16 tiles in shared memory:
//    codes by the hardware conversion, times their scale by one packed multiply (exact: 2 by 4
//    significant bits), stored in the 128-byte-swizzled layout the MMA reads (rows = keys, so K is
//    K-major and V MN-major). Raw records are loaded into registers one tile ahead and block
//    ids two, so no conversion waits on memory; units are dealt to lanes so that every 16-byte
//    store of a quarter-warp meets eight different banks.
//  * one warp issues the MMAs: S = Q K^T (M 128, N KT, K head_dim) into TMEM, and O += P V with P read
//    from TMEM, where the softmax wrote it over the S it came from, a tile's first half as soon as it is
//    there (two halves 91.6 us, one whole 94.1 on the chunks below);
//  * 4 softmax warps per block of query rows, one thread per row (TMEM lane = row): maximum over the
//    row's scores, P = 2^(s - m + 7) as fp16, and the fp32 sum; no exchange between threads. The maximum
//    moves only when a tile passes it by 2^8, so rescaling O in TMEM is rare.
//  With NQ = 2 the blocks alternate: while the softmax of one runs, the tensor cores do the other's
//  P V and next S, and each decoded tile serves 256 rows. At head_dim 256 TMEM holds one block
//  (O takes 256 of its 512 columns), which alternates between two S buffers instead.
//  * fp16 q enters as it is, bf16 q as fp16 with a power of two per row that puts its largest element
//    near 2^13 (exact for every element within 2^-27 of the largest).
//  * P enters as fp16, weights whose sum is kept unrounded in fp32. For bf16 results one fp16 is enough: a
//    result is off by at most 2^-11 of the weighted mean of |v|, an eighth of a bf16 half ulp of that mean.
//    fp16 results are no coarser than that, so they get a second MMA with what the first fp16 left, kept
//    in the scores' lower columns: 2^-22, as the warp kernel does
//    (the chunks below in fp16: 117.6 us, 90.5 with one part).
//  * Tokens past the row have P = 0, and their V is stored as zeros, so whatever bytes a page holds
//    there never reach O.
//  * Every wait is bounded; a role whose wait runs out records DEVERR_WAIT_TIMEOUT and raises the
//    CTA's abort flag, every role then leaves its loop, the MMA thread waits for its MMAs and the CTA
//    frees its TMEM and returns.
//
// Measured: 4 chunks of 1001-1024 tokens behind some 2000, bf16, 16 heads on 8 of 128, 91.6 us: 897 TFLOP/s of
// visible pairs, 0.54 of the measured bf16 rate. A tile of 128 keys takes a CTA some 3500 clocks, of which
// its MMAs (hidden pairs included) are 2048 and its exponentials 2048 on their own unit: what bounds it is
// each block's chain S -> softmax -> P V -> next S with four hand-overs of 100-200 clocks; a CTA's
// first S is there after 7000 clocks (three dependent loads and Q's conversion), its rows go out in 4000.
#include "paged_decode.h"
#include "pd_fp4.cuh"
#include "pd_tcgen05.cuh"
#include "pd_tile.cuh"

#include <type_traits>

namespace pd {

namespace {

constexpr int ROWS = 128;  // query rows of a block (the MMA's M)

template <int D>
struct Cfg {
  static constexpr int NQ = D <= 128 ? 2 : 1;     // blocks of query rows per CTA
  static constexpr int KT = D <= 128 ? 128 : 64;  // keys per tile (the S MMA's N)
  static constexpr int PART = KT / 2;             // keys of a tile whose P V may start before the others' P
  static constexpr int NSB = 2;                   // S/P buffers: one per block, or two of the one block
  static constexpr int SOFTMAX_WARPS = 4 * NQ;
  static constexpr int DECODE_WARPS = 4;
  static constexpr int DECODERS = DECODE_WARPS * 32;
  static constexpr int MMA_WARP = SOFTMAX_WARPS + DECODE_WARPS;
  static constexpr int THREADS = (MMA_WARP + 4) * 32;  // the MMA warp's group of four: three are idle
  // Registers are dealt anew between the groups, so that a softmax thread holds a row's KT scores: with
  // 128 for everyone it had to read half of them twice, 99 us against 94 on the 1001-token chunks.
  static constexpr int LAUNCH_REGS = 65536 / THREADS / 8 * 8;
  static constexpr int SOFTMAX_REGS = NQ == 2 ? 184 : 208;
  static constexpr int DECODE_REGS = NQ == 2 ? 96 : 112;
  static constexpr int MMA_REGS = 48;
  static_assert(SOFTMAX_WARPS * SOFTMAX_REGS + DECODE_WARPS * DECODE_REGS + 4 * MMA_REGS <= THREADS / 32 * LAUNCH_REGS,
                "a split above the launch's registers would wait for ever");
  static constexpr int STAGES = 2;  // decoded tiles of K, and of V
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int KV_BYTES = KT * D * 2;
  static constexpr int O_COL = NSB * KT;
  static constexpr int TMEM_COLS = 512;
  static_assert(O_COL + NQ * D <= TMEM_COLS, "TMEM columns");
  static constexpr int OFF_Q = 1024;  // barriers and flags before it
  static constexpr int OFF_K = OFF_Q + NQ * Q_BYTES;
  static constexpr int OFF_V = OFF_K + STAGES * KV_BYTES;
  static constexpr int SMEM = OFF_V + STAGES * KV_BYTES + 1024;  // + run-time 1 KB alignment
  static_assert(SMEM <= 232448, "shared memory per CTA");
  // Units of 16 code bytes (32 elements): of K a token's 32 elements, of V 16 elements of two tokens.
  static constexpr int UNITS = KT * D / 32;
  static constexpr int PER_THREAD = UNITS / (DECODE_WARPS * 32);
  static constexpr int PER_RECORD = D / 2;
};

// Barrier slots (8 bytes each) at the front of shared memory.
struct Bars {
  static constexpr int K_FULL = 0;   // [2] K tile stored: one arrival per decoding warp
  static constexpr int V_FULL = 2;   // [2]
  static constexpr int K_EMPTY = 4;  // [2] every S of the tile completed (commit)
  static constexpr int V_EMPTY = 6;  // [2] every P V of the tile completed (commit)
  static constexpr int S_FULL = 8;   // [2] S buffer written (commit)
  static constexpr int P_FULL = 10;  // [2] P written over it, O rescaled: one arrival per softmax warp
  static constexpr int O_DONE = 12;  // [2] P V that read the buffer completed (commit)
  static constexpr int Q_FULL = 14;  // Q stored: one arrival per softmax warp
  static constexpr int DRAIN = 15;
  static constexpr int P_PART = 16;  // [2] P of the tile's first PART keys written
  static constexpr int TMEM_SLOT = 160;  // byte offsets
  static constexpr int ABORT = 168;
};

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::THREADS, 1) pd_fp4_prefill_kernel(const __grid_constant__ Fp4AttendParams p,
                                                                           int blocks) {
  using C = Cfg<D>;
  using E = Elem<T>;
  constexpr int REC = fp4_record_bytes(D);
  constexpr int NQ = C::NQ, KT = C::KT;
  constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value ? 1 : 2;  // fp16 operands that P is the sum of
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t raw = smem_addr(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const uint32_t sbase = smem_addr(smem);
  auto bar = [&](int slot) -> uint32_t { return sbase + uint32_t(slot) * 8u; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + Bars::ABORT);

  if (warp == C::MMA_WARP) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar(Bars::K_FULL + i), C::DECODE_WARPS);
        mbar_init(bar(Bars::V_FULL + i), C::DECODE_WARPS);
        mbar_init(bar(Bars::K_EMPTY + i), 1);
        mbar_init(bar(Bars::V_EMPTY + i), 1);
        mbar_init(bar(Bars::S_FULL + i), 1);
        mbar_init(bar(Bars::P_FULL + i), 4);
        mbar_init(bar(Bars::P_PART + i), 4);
        mbar_init(bar(Bars::O_DONE + i), 1);
      }
      mbar_init(bar(Bars::Q_FULL), C::SOFTMAX_WARPS);
      mbar_init(bar(Bars::DRAIN), 1);
      *abort_flag = 0;
      fence_barrier_init();
    }
    __syncwarp();
    tc::tmem_alloc(sbase + Bars::TMEM_SLOT, C::TMEM_COLS);
    tc::tmem_relinquish();
  }

  // Query blocks slowest and last ones first: the causal tail has the most keys.
  const int pairs = p.batch * p.n_kv_head;
  const int b = int(blockIdx.x) % p.batch;
  const int h = (int(blockIdx.x) / p.batch) % p.n_kv_head;
  const int qblock = blocks - 1 - int(blockIdx.x) / pairs;
  // Unit i of decoding thread t is unit u of record first_rec + i * REC_STEP of the tile. The first
  // tile's block ids are loaded beside the lengths; whether a record is the row's is asked later.
  constexpr int N = C::PER_THREAD;
  constexpr int REC_STEP = C::DECODERS / C::PER_RECORD;
  const int t = tid - C::SOFTMAX_WARPS * 32, u = t % C::PER_RECORD, first_rec = t / C::PER_RECORD;
  const int32_t* trow = p.table + int64_t(b) * p.bt_stride;
  auto block_of = [&](int tile, int i) -> int {
    const int page = (tile * (KT / 16) + first_rec + i * REC_STEP) >> p.log2_tpb;
    return page < p.max_blocks ? __ldg(trow + page) : -1;
  };
  int blk[N];
  if (warp >= C::SOFTMAX_WARPS && warp < C::MMA_WARP) {
#pragma unroll
    for (int i = 0; i < N; ++i) blk[i] = block_of(0, i);
  }
  const int q_begin = min(max(__ldg(p.cu_q + b), 0), p.total_q);
  const int chunk = max(min(max(__ldg(p.cu_q + b + 1), 0), p.total_q) - q_begin, 0);
  const int sq = min(chunk, p.max_seqlen_q);
  int lk = __ldg(p.seqlen + b);
  lk = lk < 0 ? 0 : (lk > p.capacity ? p.capacity : lk);
  const int rows = sq * p.group;
  const int row0 = qblock * NQ * ROWS;  // first query row of the CTA
  // keys that block q of the CTA needs: up to its last row's token
  int kend[NQ], tiles[NQ], most = 0;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int r0 = row0 + q * ROWS;
    const int last = min(r0 + ROWS, rows) - 1;
    kend[q] = r0 < rows ? min(max(lk - chunk + last / p.group + 1, 0), lk) : 0;
    tiles[q] = (kend[q] + KT - 1) / KT;
    most = max(most, tiles[q]);
  }

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
  auto fail = [&]() {
    *abort_flag = 1;
    atomicOr(p.err, DEVERR_WAIT_TIMEOUT);
  };

  if (row0 >= rows) {  // no query row
    tmem = meet();
  } else if (warp >= C::SOFTMAX_WARPS && warp < C::MMA_WARP) {
    // ---------------------------------------------------------------- decoding warps
    regs_down<C::DECODE_REGS>();
    const int tpb_mask = (1 << p.log2_tpb) - 1;
    const int records = (lk + FP4_TILE - 1) / FP4_TILE;
    const unsigned char* head = p.pages + (int64_t(h) << p.log2_tpb) * REC;
    const uint32_t block_stride = uint32_t(p.n_kv_head << p.log2_tpb) * REC;
    // K unit: 32 elements of token k_tok, 16 tokens side by side, so that a quarter-warp's stores go
    // to eight rows and, swizzled, to eight banks.
    constexpr int W = D < 128 ? D : 128, CH = W / 32;  // 16-byte chunks of a token in a block
    const int k_tok = u % 16, k_blk = u / 16 / CH, k_ch = u / 16 % CH;
    const int k_el = k_blk * W + k_ch * 32;  // first element
    const int k_code_off = k_blk * 8 * W + k_tok * (W / 2) + k_ch * 16;
    const int k_scale_off = 8 * D + k_blk * W + k_tok * (W / 16) + k_ch * 2;
    const uint32_t k_row = uint32_t((k_el >> 6) * (KT * 128) + k_tok * 128);  // in the tile, of record 0
    const uint32_t k_x = uint32_t((((k_el & 63) >> 3) ^ (k_tok & 7)) << 4);   // swizzled unit of word 0
    // V unit: 16 elements of tokens v_tok, v_tok + 1. Even rows of two groups meet the same four banks,
    // so lanes of odd groups store their two 8-element units in the other order.
    const int v_half = u / (D / 4), v_gr = (u / 4) % (D / 16), v_tok = v_half * 8 + (u % 4) * 2;
    const bool v_odd = v_gr & 1;
    const int v_code_off = 9 * D + 16 * u;
    const int v_scale_off = 17 * D + v_half * (D / 2) + v_gr * 8 + (u % 4) * 2;
    const uint32_t v_row = uint32_t((v_gr >> 2) * (KT * 128) + v_tok * 128);
    const uint32_t v_x = uint32_t((((v_gr & 3) * 2 + (v_odd ? 1 : 0)) ^ (v_tok & 7)) << 4);

    // a negative scale's sign goes into K, so that the score multiplier is never negative
    const uint32_t k_sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;
    uint4 kraw[N], vraw[N];
    uint32_t ksc[N], vsc[N];
    int blk_next[N];
    const unsigned char* ptr[N];  // the records being loaded, or nullptr
    auto aim = [&](int tile) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int rec = tile * (KT / 16) + first_rec + i * REC_STEP;
        ptr[i] = rec < records && blk[i] >= 0 && blk[i] < p.n_blocks ? head + uint64_t(blk[i]) * block_stride + (rec & tpb_mask) * REC
                                                    : nullptr;
      }
    };
    auto load = [&](uint4 (&code)[N], uint32_t (&scale)[N], int code_off, int scale_off) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        code[i] = make_uint4(0u, 0u, 0u, 0u);
        scale[i] = 0u;
        if (ptr[i] != nullptr) {
          code[i] = __ldg(reinterpret_cast<const uint4*>(ptr[i] + code_off));
          scale[i] = __ldg(reinterpret_cast<const uint16_t*>(ptr[i] + scale_off));
        }
      }
    };
    aim(0);
    load(kraw, ksc, k_code_off, k_scale_off);
    load(vraw, vsc, v_code_off, v_scale_off);
#pragma unroll
    for (int i = 0; i < N; ++i) blk[i] = block_of(1, i);
#pragma unroll
    for (int i = 0; i < N; ++i) blk_next[i] = block_of(2, i);
    tmem = meet();
    bool ok = true;
    for (int j = 0; ok && j < most; ++j) {
      if (__any_sync(FULL_MASK, *abort_flag != 0)) break;
      const int s = j % C::STAGES;
      const uint32_t freed = uint32_t((j / C::STAGES - 1) & 1);  // phase of the stage's previous use
      if (j >= C::STAGES && !warp_wait_phase(bar(Bars::K_EMPTY + s), freed, p.wait_ns)) {
        ok = false;
        break;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t pair = e4m3x2_to_half2(ksc[i]) ^ k_sign;
        const uint32_t sc[2] = {__byte_perm(pair, 0, 0x1010), __byte_perm(pair, 0, 0x3232)};
        const uint32_t w[4] = {kraw[i].x, kraw[i].y, kraw[i].z, kraw[i].w};
        const uint32_t row = k_addr(s) + k_row + uint32_t((first_rec + i * REC_STEP) * 2048);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t x[4];
          e2m1x8_to_half2x4(w[e], x);
          sts128(row + (k_x ^ uint32_t(e << 4)), hmul2_bits(x[0], sc[e >> 1]), hmul2_bits(x[1], sc[e >> 1]),
                 hmul2_bits(x[2], sc[e >> 1]), hmul2_bits(x[3], sc[e >> 1]));
        }
      }
      aim(j + 1);
      load(kraw, ksc, k_code_off, k_scale_off);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        blk[i] = blk_next[i];
        blk_next[i] = block_of(j + 3, i);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Bars::K_FULL + s));
      if (j >= C::STAGES && !warp_wait_phase(bar(Bars::V_EMPTY + s), freed, p.wait_ns)) {
        ok = false;
        break;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int key = j * KT + (first_rec + i * REC_STEP) * 16 + v_tok;
        uint32_t pair = e4m3x2_to_half2(vsc[i]);
        if (key + 1 >= lk) pair &= key < lk ? 0x0000ffffu : 0u;  // zeros past the row
        const uint32_t sc[2] = {__byte_perm(pair, 0, 0x1010), __byte_perm(pair, 0, 0x3232)};
        const uint32_t w[4] = {v_odd ? vraw[i].y : vraw[i].x, v_odd ? vraw[i].x : vraw[i].y,
                               v_odd ? vraw[i].w : vraw[i].z, v_odd ? vraw[i].z : vraw[i].w};
        const uint32_t row = v_addr(s) + v_row + uint32_t((first_rec + i * REC_STEP) * 2048);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // token v_tok + e / 2: its row is the next one, its swizzle one bit off
          uint32_t x[4];
          e2m1x8_to_half2x4(w[e], x);
          sts128(row + uint32_t((e >> 1) * 128) + (v_x ^ uint32_t(((e & 1) ^ (e >> 1)) << 4)),
                 hmul2_bits(x[0], sc[e >> 1]), hmul2_bits(x[1], sc[e >> 1]), hmul2_bits(x[2], sc[e >> 1]),
                 hmul2_bits(x[3], sc[e >> 1]));
        }
      }
      load(vraw, vsc, v_code_off, v_scale_off);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Bars::V_FULL + s));
    }
    if (!ok && lane == 0) fail();
  } else if (warp >= C::MMA_WARP) {
    regs_down<C::MMA_REGS>();
    if (warp > C::MMA_WARP) {
      tmem = meet();
    } else {  // (one meeting before the branch costs the compiler 150 bytes of spills)
      // ---------------------------------------------------------------- MMA issuer
      // The whole warp runs this loop and one elected lane issues, so descriptors and addresses stay
      // uniform over the warp and no operand of an MMA is moved on its own.
      tmem = meet();
      if (most > 0) {
        constexpr uint32_t IDESC_S = tc::instr_desc_f16(false, ROWS, KT, false, false);
        constexpr uint32_t IDESC_PV = tc::instr_desc_f16(false, ROWS, D, false, true);
        bool ok = lane_wait(bar(Bars::Q_FULL), 0u, p.wait_ns);
        const uint64_t q_desc = tc::smem_desc(sbase + C::OFF_Q, 16u, 1024u);
        const uint64_t k_desc = tc::smem_desc(k_addr(0), 16u, 1024u);
        const uint64_t v_desc = tc::smem_desc(v_addr(0), uint32_t(KT * 128), 1024u);
        // (block q, tile j) uses S/P buffer q for the j-th time or, with one block, buffer j % 2 for
        // the j / 2-th.
        auto buf = [&](int q, int j) -> int { return NQ == 2 ? q : j & 1; };
        auto use = [&](int j) -> uint32_t { return NQ == 2 ? uint32_t(j) : uint32_t(j >> 1); };
        // S of (q, j), once P V of the buffer's previous use has read its P
        auto issue_s = [&](int q, int j) {
          const int s = j & 1, sb = buf(q, j);
          if (q == 0 || j >= tiles[0])  // else the first block has waited for this K tile
            ok = ok && lane_wait(bar(Bars::K_FULL + s), uint32_t((j >> 1) & 1), p.wait_ns);
          if (use(j) > 0) ok = ok && lane_wait(bar(Bars::O_DONE + sb), (use(j) - 1) & 1u, p.wait_ns);
          __syncwarp();
          tc::fence_after_sync();
          const uint64_t a0 = q_desc + uint64_t((q * C::Q_BYTES) >> 4), b0 = k_desc + uint64_t((s * C::KV_BYTES) >> 4);
          const bool frees = q == NQ - 1 || j >= tiles[NQ - 1];  // the last block that uses this K tile
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              tc::mma_f16_ss(tmem + uint32_t(sb * KT), a0 + uint64_t(((ks >> 2) * (ROWS * 128) + (ks & 3) * 32) >> 4),
                             b0 + uint64_t(((ks >> 2) * (KT * 128) + (ks & 3) * 32) >> 4), IDESC_S, ks > 0);
            tc::commit(bar(Bars::S_FULL + sb));
            if (frees) tc::commit(bar(Bars::K_EMPTY + s));
          }
          __syncwarp();
        };
        auto issue_pv = [&](int q, int j) {
          const int s = j & 1, sb = buf(q, j);
          if (q == 0 || j >= tiles[0])
            ok = ok && lane_wait(bar(Bars::V_FULL + s), uint32_t((j >> 1) & 1), p.wait_ns);
          const uint64_t b0 = v_desc + uint64_t((s * C::KV_BYTES) >> 4);
          const bool frees = q == NQ - 1 || j >= tiles[NQ - 1];
          auto part = [&](int k0, int k1) {
#pragma unroll
            for (int kk = k0; kk < k1; ++kk)
#pragma unroll
              for (int i = 0; i < PARTS; ++i)  // the first part in the upper half of the buffer's columns
                tc::mma_f16_ts(tmem + uint32_t(C::O_COL + q * D), tmem + uint32_t(sb * KT + (1 - i) * (KT / 2) + kk * 8),
                               b0 + uint64_t((kk * 2048) >> 4), IDESC_PV, j > 0 || kk > 0 || i > 0);
          };
          // the first PART keys while the softmax is at the others
          ok = ok && lane_wait(bar(Bars::P_PART + sb), use(j) & 1u, p.wait_ns);
          __syncwarp();
          tc::fence_after_sync();
          if (elect_one()) part(0, C::PART / 16);
          __syncwarp();
          ok = ok && lane_wait(bar(Bars::P_FULL + sb), use(j) & 1u, p.wait_ns);
          __syncwarp();
          tc::fence_after_sync();
          if (elect_one()) {
            part(C::PART / 16, KT / 16);
            tc::commit(bar(Bars::O_DONE + sb));
            if (frees) tc::commit(bar(Bars::V_EMPTY + s));
          }
          __syncwarp();
        };
        if (__all_sync(FULL_MASK, ok)) {
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            if (tiles[q] > 0) issue_s(q, 0);
        }
        for (int j = 0; j < most; ++j) {
          if (!__all_sync(FULL_MASK, ok && *abort_flag == 0)) break;
          if (NQ == 1 && j + 1 < most) issue_s(0, j + 1);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if (j < tiles[q]) issue_pv(q, j);
            if (NQ == 2 && j + 1 < tiles[q]) issue_s(q, j + 1);
          }
        }
        if (!__all_sync(FULL_MASK, ok) && lane == 0) fail();
        if (elect_one()) tc::commit(bar(Bars::DRAIN));  // never leave with an MMA in flight
        __syncwarp();
        warp_wait_phase(bar(Bars::DRAIN), 0u, DRAIN_LIMIT_NS);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax warps
    regs_up<C::SOFTMAX_REGS>();
    const int q = warp >> 2;
    const int r = (warp & 3) * 32 + lane;  // row of the block = TMEM lane
    const int n = row0 + q * ROWS + r;
    const bool live = n < rows;
    const int tok = live ? n / p.group : 0;
    float down = 1.f;  // 1 / the row's power of two
    // Q as it is into its place (16-byte units of 8 elements, all copies in flight at once); bf16 rows are
    // then turned into fp16 where they stand, a thread its own row.
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
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      asm volatile("bar.sync %0, 128;" ::"r"(1 + q) : "memory");  // the block's rows are in
      constexpr int KEEP = LANES < 16 ? LANES : 16;  // units of a row in registers at a time
      auto unit = [&](int u) -> uint32_t { return q_base + uint32_t((u >> 3) * (ROWS * 128)) + sw128(r, u & 7); };
      uint4 w[KEEP];
      __nv_bfloat162 top2 = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll 1
      for (int u0 = LANES - KEEP; u0 >= 0; u0 -= KEEP) {
#pragma unroll
        for (int i = 0; i < KEEP; ++i) w[i] = lds128(unit(u0 + i));
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
          const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&w[i]);
          const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(v[0]), __habs2(v[1])), __hmax2(__habs2(v[2]), __habs2(v[3])));
          top2 = __hmax2(top2, m);
        }
      }
      const float top = fmaxf(__low2float(top2), __high2float(top2));
      int e = int(__float_as_uint(top) >> 23);
      e = e == 0 || e == 255 ? 140 : e;
      const int shift = min(126, 140 - e);  // at least -114; its inverse is a normal number
      const float up = __uint_as_float(uint32_t(127 + shift) << 23);
      down = __uint_as_float(uint32_t(127 - shift) << 23);
#pragma unroll 1
      for (int u0 = 0; u0 < LANES; u0 += KEEP) {
        if (u0 > 0) {
#pragma unroll
          for (int i = 0; i < KEEP; ++i) w[i] = lds128(unit(u0 + i));
        }
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
          float x[8];
          E::unpack(w[i], x);
          sts128(unit(u0 + i), Elem<__half>::pack2(x[0] * up, x[1] * up), Elem<__half>::pack2(x[2] * up, x[3] * up),
                 Elem<__half>::pack2(x[4] * up, x[5] * up), Elem<__half>::pack2(x[6] * up, x[7] * up));
        }
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(Bars::Q_FULL));
    // never zero (a scale of 0 gives scores below 2^-80 instead), so that a hidden key's -inf stays one
    const float mul = fmaxf(fabsf(p.scale_log2) * (p.units != nullptr ? __ldg(p.units + h) : 1.f) * down, 1.2e-38f);
    const float v_unit = p.units != nullptr ? __ldg(p.units + p.n_kv_head + h) : 1.f;
    const int lim = live ? lk - chunk + tok : lk - 1;  // last visible key; padding rows see any
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t o_tmem = lane_base + uint32_t(C::O_COL + q * D);
    float m_run = -3.0e38f, l_run = 0.f;
    bool ok = true;
    int mine = tiles[0];
#pragma unroll
    for (int i = 1; i < NQ; ++i) mine = q == i ? tiles[i] : mine;
    for (int j = 0; j < mine; ++j) {
      const int sb = NQ == 2 ? q : j & 1;
      const uint32_t ph = (NQ == 2 ? uint32_t(j) : uint32_t(j >> 1)) & 1u;
      if (__any_sync(FULL_MASK, *abort_flag != 0) || !warp_wait_phase(bar(Bars::S_FULL + sb), ph, p.wait_ns)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      const uint32_t s_tmem = lane_base + uint32_t(sb * KT);
      const bool open = __all_sync(FULL_MASK, j * KT + KT - 1 <= lim);  // no key of the tile is hidden
      // The row's scores stay in registers from the maximum to P, which is stored over the upper half of
      // their columns, its second part over the lower.
      float x[KT];
#pragma unroll
      for (int c = 0; c < KT; c += 32)
        tc::ld_32x32b_x32(s_tmem + uint32_t(c), *reinterpret_cast<uint32_t(*)[32]>(x + c));
      tc::wait_ld();
      if (!open) {
#pragma unroll
        for (int c = 0; c < KT; c += 32) {
          const int seen = lim - (j * KT + c);  // the last visible of these columns
          if (__all_sync(FULL_MASK, seen >= 31)) continue;
#pragma unroll
          for (int i = 0; i < 32; ++i) x[c + i] = i <= seen ? x[c + i] : -INFINITY;
        }
      }
      float t[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < KT; i += 8) {
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = fmaxf(fmaxf(t[k], x[i + k]), i + 4 + k < KT ? x[i + 4 + k] : t[k]);
      }
      const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      // mul >= 0: the maximum of the products is the product of the maximum
      const float tmax = top * mul;
      const bool move = tmax > m_run + (FP4_P_SHIFT + FP4_HEADROOM) || (m_run < -1.0e38f && tmax > m_run);
      if (__any_sync(FULL_MASK, move)) {
        const float ref = tmax - FP4_P_SHIFT;
        const float alpha = move ? ex2(m_run - ref) : 1.f;
        if (move) m_run = ref;
        l_run *= alpha;
        if (j > 0) {  // O *= alpha once P V of tile j - 1 has landed
          const int pb = NQ == 2 ? q : (j - 1) & 1;
          const uint32_t pp = (NQ == 2 ? uint32_t(j - 1) : uint32_t((j - 1) >> 1)) & 1u;
          if (!warp_wait_phase(bar(Bars::O_DONE + pb), pp, p.wait_ns)) {
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
      for (int c = 0; c < KT; c += 32) {  // two keys to a column
        uint32_t w[16], rest[PARTS == 2 ? 16 : 1];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float2 e = fma2(make_float2(x[c + i], x[c + i + 1]), mul2, neg_m2);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
          w[i >> 1] = Elem<__half>::pack2(e.x, e.y);
          if constexpr (PARTS == 2) {
            float f[2];
            Elem<__half>::unpack2(w[i >> 1], f);
            rest[i >> 1] = Elem<__half>::pack2(e.x - f[0], e.y - f[1]);
          }
        }
        st_32x32b_x16(s_tmem + uint32_t(KT / 2 + c / 2), w);
        if constexpr (PARTS == 2) st_32x32b_x16(s_tmem + uint32_t(c / 2), rest);
        if (c + 32 == C::PART) {
          tc::wait_st();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(Bars::P_PART + sb));
        }
      }
      const float2 total = add2(sum[0], sum[1]);
      l_run += total.x + total.y;
      tc::wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Bars::P_FULL + sb));
    }
    if (ok && mine > 0) {
      const int lb = NQ == 2 ? q : (mine - 1) & 1;
      const uint32_t lp = (NQ == 2 ? uint32_t(mine - 1) : uint32_t((mine - 1) >> 1)) & 1u;
      ok = warp_wait_phase(bar(Bars::O_DONE + lb), lp, p.wait_ns);
    }
    if (!ok) {
      if (lane == 0) fail();
    } else {
      tc::fence_after_sync();
      const float inv = l_run > 0.f ? v_unit / l_run : 0.f;
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
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = E::pack2(__uint_as_float(o[8 * u + 2 * i]) * inv, __uint_as_float(o[8 * u + 2 * i + 1]) * inv);
          const int at = c / 8 + u;
          sts128(q_base + uint32_t((at >> 3) * (ROWS * 128)) + sw128(r, at & 7), w[0], w[1], w[2], w[3]);
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
  if (warp == C::MMA_WARP) {
    __syncwarp();
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <typename T, int D>
cudaError_t launch_t(const Fp4AttendParams& p, cudaStream_t stream) {
  using C = Cfg<D>;
  auto fn = pd_fp4_prefill_kernel<T, D>;
  static SmemRaised raised{};
  const cudaError_t err = raise_smem_limit(fn, C::SMEM, raised);
  if (err != cudaSuccess) return err;
  const int64_t rows = int64_t(p.max_seqlen_q) * p.group;
  const int64_t blocks = (rows + C::NQ * ROWS - 1) / (C::NQ * ROWS);
  const int64_t ctas = blocks * p.batch * p.n_kv_head;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  fn<<<dim3(unsigned(ctas)), C::THREADS, C::SMEM, stream>>>(p, int(blocks));
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_d(const Fp4AttendParams& p, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 64: return launch_t<T, 64>(p, stream);
    case 128: return launch_t<T, 128>(p, stream);
    case 256: return launch_t<T, 256>(p, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_fp4_prefill(const Fp4AttendParams& p, int dtype, int head_dim, cudaStream_t stream) {
  return dtype == PD_BF16 ? launch_d<__nv_bfloat16>(p, head_dim, stream) : launch_d<__half>(p, head_dim, stream);
}

}  // namespace pd
