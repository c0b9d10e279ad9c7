// Attention over the pages, 128 rows at a time (tcgen05): chunks of prompts, several drafted tokens with
// many heads, and a whole batch against its shared prefix.
//
// The mathematics and the rows are paged_attn_kernel's (paged.cuh): the rows of a Q tile are `tokens`
// consecutive new tokens times the G query heads of one K/V head, token-major, so that each K/V tile is
// read once for up to 128 (or, with two Q tiles, 256) rows. 4 * 128 FLOP per row and key against 512
// bytes per key: from about 130 rows on the tensor cores and the exponentials bound it, not HBM.
//
// A block is the warp-specialised pipeline of the contiguous kernel (attn_fwd_sm100.cuh; the TMEM
// layout, the order of the MMAs, the softmax and its lazy rescaling are described there):
//
//   warps 0-3 / 4-7  softmax, correction and epilogue, one row per thread: of Q tile 0 / 1, or of the even /
//                    odd steps of the only Q tile
//   warps 8 and 10   TMA: Q tiles and K, and V; the lanes hold the page numbers of a tile's groups of box_rows
//                    keys (a power of two that divides the page size) and each issues its own boxes
//   warp 9           one thread issues every tcgen05.mma
//   warp 11          the schedule: pieces of work into a small ring that the other warps read
//
// Schedule. A unit is (sequence, K/V head, Q tiles of `block_tokens` tokens) and has as many steps as
// 128-key tiles up to its last visible key. All units lie on one line of steps, with room before each for
// what it costs beside them, and every block takes an equal stretch of it, so ragged batches, causal chunks
// and few rows against many keys are balanced alike; the prefix sums of the steps have a closed form, so the
// line needs no plan and no host. A unit that a boundary cuts leaves (m, l, O) per piece in the workspace, in FP32,
// and paged_join_kernel adds them up in key order.
//
// Measured with the join: 4096 tokens behind 28672 keys, 8 heads on 2, 489 us (1055 TFLOP/s at the power limit,
// 1310 in the kernel alone at 1965 MHz), where neither the tensor pipe (54 %) nor MUFU (57 %) is full and the
// round trip softmax -> P V -> S -> softmax bounds; 16 sequences of 3 to 7 tokens, 71 MB of keys, 25 us, 10 of them
// at HBM speed between a start of 6, an epilogue and the join.
#pragma once
#include "attn_fwd_sm100.cuh"
#include "paged.cuh"

namespace fav4 {

constexpr int kPieceSlots = 4;
constexpr uint32_t kTileSoftmaxRegs = 208;  // 128 * (2 * 208 + 88) = 384 * 168
constexpr uint32_t kTileOtherRegs = 88;

struct PagedTileParams {
  PagedParams p;        // part_o / part_ml: [2 grid][QTiles] tiles, see below; arrived: unused
  int4* cut;            // [grid]: the unit that block c opens and does not finish: first token, tokens, K/V head, last block (-1: none)
  int tile_tokens;      // tokens per Q tile: 128 / group
  int box_rows;         // keys per TMA box
  uint32_t* status;
  uint64_t wait_limit_ns;
};

// The waits of sm100.cuh with the part that does wait out of line, for the warps that can afford the call: a
// kernel of a few microseconds notices the code that it fetches. The MMA and softmax warps, whose waits are
// on the way of every step, keep theirs in line (out of line in the MMA warp: 2 % slower on long chunks).
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, WaitCtl ctl, uint32_t code) {
  return mbar_wait(bar, parity, ctl, code);
}
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, const WaitCtl& ctl, uint32_t code) {
  return mbar_test(bar, parity) || wait_long(bar, parity, ctl, code);
}
__device__ __forceinline__ bool warp_wait_phase(uint32_t bar, uint32_t parity, const WaitCtl& ctl, uint32_t code) {
  return __all_sync(0xffffffffu, wait_phase(bar, parity, ctl, code));
}

// A stretch of one unit.
struct Piece {
  int token0, tokens;   // the unit's first row of Q, and how many tokens it has
  int past;             // keys before that first token (its own position in the sequence)
  int len, h, b;        // keys of the sequence, K/V head, sequence
  int tile0, cnt, n;    // steps [tile0, tile0 + cnt) of n
  int pad[7];
};
static_assert(sizeof(Piece) == 64, "four 16-byte words");

template <int QTiles>
struct PagedTileLayout {
  static constexpr int kSlots = QTiles == 1 ? 3 : 2;
  static constexpr int kSlotBytes = 2 * kTileBytes;
  static constexpr int kQ = 0;
  static constexpr int kKV = QTiles * kTileBytes;
  static constexpr int kBar = kKV + kSlots * kSlotBytes;
  static constexpr int kQFull = 0, kQEmpty = 1, kKVFull = 2, kKVEmpty = kKVFull + kSlots, kVFix = kKVEmpty + kSlots;
  static constexpr int kSFull = kVFix + kSlots, kPFull = kSFull + 2, kOFull = kPFull + 2, kOEmpty = kOFull + 2;
  static constexpr int kPieceFull = kOEmpty + 2, kPieceEmpty = kPieceFull + kPieceSlots;
  static constexpr int kXFull = kPieceEmpty + kPieceSlots, kXEmpty = kXFull + 1;  // one Q tile: the streams' (m, l)
  static constexpr int kTeardown = kXEmpty + 1;
  static constexpr int kNumBars = kTeardown + 1;
  static constexpr int kPieces = (kBar + kNumBars * 8 + 15) & ~15;
  static constexpr int kMisc = kPieces + kPieceSlots * 64;  // TMEM base, abort flag, schedule scan
  static constexpr int kScan = (kMisc + 8 + 15) & ~15;      // 12 warps' sums, then base, sequence
  static constexpr int kMl = kScan + 20 * 8;  // one Q tile: (m, l) of the two key streams
  static constexpr int kBytes = kMl + (QTiles == 1 ? 2 * 128 * 8 : 0);
  static constexpr int kAlloc = kBytes;  // the kernel checks that its base is 1 KiB aligned
  static_assert(kAlloc <= 227 * 1024, "shared memory budget");
};

// Transposes 8 x 8 16-byte pieces over each eight lanes: lane i's piece k becomes piece i of lane k's.
__device__ __forceinline__ void transpose_pieces(uint4 (&v)[8], int lane) {
#pragma unroll
  for (int s = 4; s > 0; s /= 2) {
    const bool high = lane & s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j & s) continue;
      const uint4 out = high ? v[j] : v[j | s];
      uint4 in;
      in.x = __shfl_xor_sync(0xffffffffu, out.x, s);
      in.y = __shfl_xor_sync(0xffffffffu, out.y, s);
      in.z = __shfl_xor_sync(0xffffffffu, out.z, s);
      in.w = __shfl_xor_sync(0xffffffffu, out.w, s);
      if (high) v[j] = in;
      else v[j | s] = in;
    }
  }
}

// Rows of one tile in the workspace, as the softmax threads (one row each) write them: 4-column piece c of
// row r at float4 index c * 128 + r, so that a warp's stores and loads are whole lines.
__device__ __forceinline__ int64_t part_tile(int slot, int qtiles, int i) { return static_cast<int64_t>(slot) * qtiles + i; }

template <int QTiles>
__global__ void __launch_bounds__(384, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedTileParams tp) {
  using L = PagedTileLayout<QTiles>;
  constexpr int Slots = L::kSlots;
  constexpr int KA = QTiles == 1 ? 2 : 1;  // S runs this many steps ahead of P V
  const PagedParams& p = tp.p;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_addr(smem);
  if (sbase & 1023) {  // the swizzled tiles need it; there is no room to round up
    wait_for_predecessor();
    if (threadIdx.x == 0) {
      atomicOr(tp.status, kStatusSmemAlign);
      tp.cut[blockIdx.x] = make_int4(0, 0, 0, -1);
    }
    return;
  }
  const uint32_t bar0 = sbase + L::kBar;
  auto bar = [&](int slot) -> uint32_t { return bar0 + 8u * slot; };
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMisc);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kMisc + 4);
  int64_t* scan = reinterpret_cast<int64_t*>(smem + L::kScan);
  Piece* pieces = reinterpret_cast<Piece*>(smem + L::kPieces);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  WaitCtl ctl{abort_flag, tp.status, tp.wait_limit_ns};

  if (threadIdx.x == 0) {
    *abort_flag = 0u;
    mbar_init(bar(L::kQFull), 1);
    mbar_init(bar(L::kQEmpty), 1);
    for (int s = 0; s < Slots; ++s) {
      mbar_init(bar(L::kKVFull + s), 2);  // the K side and the V side
      mbar_init(bar(L::kKVEmpty + s), 1);
      mbar_init(bar(L::kVFix + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(L::kSFull + i), 1);
      mbar_init(bar(L::kPFull + i), 4);
      mbar_init(bar(L::kOFull + i), 1);
      mbar_init(bar(L::kOEmpty + i), QTiles == 1 ? 8 : 4);  // the warps that read O_i
    }
    for (int s = 0; s < kPieceSlots; ++s) {
      mbar_init(bar(L::kPieceFull + s), 1);
      mbar_init(bar(L::kPieceEmpty + s), 3 + 8);  // load, MMA and V warps, softmax warps
    }
    mbar_init(bar(L::kXFull), 8);
    mbar_init(bar(L::kXEmpty), 8);
    mbar_init(bar(L::kTeardown), 1);
    fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 9) {
    tmem_alloc(smem_addr(tmem_holder), 512);
    tmem_relinquish();
  }
  wait_for_predecessor();

  // ---- this block's stretch of the line of steps, and the sequence that it begins in ----
  const int bt = tp.tile_tokens * QTiles;
  int64_t total = 0, per = 1, begin = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t base = 0;
    for (int b0 = 0; b0 < p.c.batch; b0 += 384) {
      const int b = b0 + threadIdx.x;
      SeqView view = {0, 0, 0};
      if (b < p.c.batch) view = seq_view(p.c, p.cu, p.total_q, p.max_sq, p.causal, b);
      const int64_t head_work = tile_seq_work(view, p.causal, bt), mine = head_work * p.c.kv_heads;
      int64_t v = mine;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const int64_t up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
      }
      if (lane == 31) scan[warp] = v;
      __syncthreads();
      int64_t sum = 0;
      for (int w = 0; w < 12; ++w) {
        if (w < warp) v += scan[w];
        sum += scan[w];
      }
      if (p.c.batch <= 384) {  // one step sees the whole batch
        total = sum;
        per = max(quotient(total + gridDim.x - 1, gridDim.x), int64_t(1));
        begin = blockIdx.x * per;
        pass = 1;
      }
      if (pass == 1 && base + v - mine <= begin && begin < base + v) {
        scan[12] = base + v - mine;
        scan[13] = b;
        scan[14] = head_work;
        scan[15] = view.q0;
        scan[16] = view.sq;
        scan[17] = view.len;
      }
      base += sum;
      __syncthreads();
    }
    if (pass == 0) {
      total = base;
      per = max(quotient(total + gridDim.x - 1, gridDim.x), int64_t(1));
      begin = blockIdx.x * per;
    }
  }
  const int64_t end = min(total, begin + per);

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  // Reads the next piece; every warp that calls it does so converged and releases the slot at once.
  int piece_at = 0;
  auto next_piece = [&](Piece* out, bool in_line = false) -> bool {
    const int s = piece_at % kPieceSlots;
    if (in_line ? !warp_wait(bar(L::kPieceFull + s), (piece_at / kPieceSlots) & 1u, ctl, kStatusTimeoutLoad)
                : !warp_wait_phase(bar(L::kPieceFull + s), (piece_at / kPieceSlots) & 1u, ctl, kStatusTimeoutLoad)) return false;
    const int4* src = reinterpret_cast<const int4*>(pieces + s);
    int4 w0 = src[0], w1 = src[1], w2 = src[2];
    out->token0 = w0.x; out->tokens = w0.y; out->past = w0.z; out->len = w0.w;
    out->h = w1.x; out->b = w1.y; out->tile0 = w1.z; out->cnt = w1.w;
    out->n = w2.x;
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(L::kPieceEmpty + s));
    ++piece_at;
    return out->cnt > 0;
  };
  // Steps of Q tile i within the piece (0: none of its rows sees a key there).
  auto tile_steps = [&](const Piece& w, int i) -> int {
    const int t0 = i * tp.tile_tokens;
    if (t0 >= w.tokens) return 0;
    int64_t keys = w.len;
    if (p.causal) keys = min(keys, static_cast<int64_t>(w.past) + min(w.tokens, t0 + tp.tile_tokens));
    if (keys <= 0) return 0;
    const int n = static_cast<int>((keys + kTileKeys - 1) / kTileKeys);
    return max(min(n - w.tile0, w.cnt), 0);
  };

  static_assert(128 * (2 * kTileSoftmaxRegs + kTileOtherRegs) <= 384 * kLaunchRegs, "register split exceeds the launch");

  if (warp >= 8) {
    regs_release<kTileOtherRegs>();
    if (warp == 8 || warp == 10) {
      // ============================ TMA producers ===========================
      // Warp 8 loads Q and K, warp 10 loads V: issuing a box costs some tens of ns, and a tile of small pages has
      // sixteen. The ring's groups are {K_0}, .., {V_g, K_(g+KA)}, .., {V_(N-1)}; both warps arrive at each. Warp 10
      // then zeroes the V rows past the end of a sequence.
      const bool side_v = warp == 10;
      const CUtensorMap* map = side_v ? &tm_v : &tm_k;
      const int lead = side_v ? 0 : KA;  // the tile of group g: g + lead
      const uint64_t pol_kv = policy_evict_last();
      const uint64_t pol_q = policy_evict_first();
      Ring ring;
      LoadState<true> st;
      bool ok = true;
      Piece w;
      const int R = tp.box_rows, groups = kTileKeys / R;
      const uint32_t q_box = static_cast<uint32_t>(tp.tile_tokens) * p.group * 128u;
      while (ok && next_piece(&w)) {
        const int n0 = tile_steps(w, 0), n1 = QTiles > 1 ? tile_steps(w, 1) : 0;
        const int N = max(n0, n1);
        if (N == 0) continue;
        if (!side_v) {
          if (!warp_wait_phase(bar(L::kQEmpty), st.q_empty(), ctl, kStatusTimeoutLoad)) { ok = false; break; }
          st.flip_q_empty();
          if (lane == 0) {
            mbar_arrive_expect_tx(bar(L::kQFull), ((n0 > 0 ? 1 : 0) + (n1 > 0 ? 1 : 0)) * 2 * q_box);
            for (int i = 0; i < QTiles; ++i) {
              if ((i == 0 ? n0 : n1) == 0) continue;
              const uint32_t dst = sbase + L::kQ + i * kTileBytes;
              const int row = w.token0 + i * tp.tile_tokens;
              tma_load_3d(dst, &tm_q, bar(L::kQFull), 0, w.h * p.group, row, pol_q);
              tma_load_3d(dst + kBoxBytes, &tm_q, bar(L::kQFull), 64, w.h * p.group, row, pol_q);
            }
          }
          __syncwarp();
        }
        // lane x < groups has the page of keys [128 j + x R, + R) of the next tile j
        const int* table = p.c.table + w.b * p.c.table_stride;
        auto page_of = [&](int j) -> int {
          const int key = (w.tile0 + j) * kTileKeys + lane * R;  // lengths stay well below INT_MAX
          if (lane >= groups || j >= N || key >= w.len) return 0;
          return min(max(load<false>(table + key / p.c.page_size), 0), p.c.num_pages - 1);
        };
        int page = page_of(0);
        for (int g = -KA; g < N && ok; ++g) {
          if (KA > 1 && g < 0 && g + KA >= N) continue;  // neither K nor V
          const int j = g + lead;
          const bool mine = j >= 0 && j < N;
          if (!warp_wait_phase(bar(L::kKVEmpty + ring.stage), ring.phase ^ 1u, ctl, kStatusTimeoutLoad)) { ok = false; break; }
          const uint32_t fb = bar(L::kKVFull + ring.stage);
          if (mine) {
            const int left = w.len - (w.tile0 + j) * kTileKeys;  // whole boxes up to the last key
            if (lane == 0) mbar_arrive_expect_tx(fb, left >= kTileKeys ? kTileBytes : ((left + R - 1) & -R) * 256u);
            st.arm(ring.stage, ring.phase);
            __syncwarp();
            if (lane < groups && lane * R < left) {
              const uint32_t dst = sbase + L::kKV + ring.stage * L::kSlotBytes + (side_v ? 0 : kTileBytes) + lane * R * 128;
              const int slot = ((w.tile0 + j) * kTileKeys + lane * R) % p.c.page_size;
              tma_load_4d(dst, map, fb, 0, w.h, slot, page, pol_kv);
              tma_load_4d(dst + kBoxBytes, map, fb, 64, w.h, slot, page, pol_kv);
            }
            __syncwarp();
            page = page_of(j + 1);
            if (side_v && j + 1 == N && left < kTileKeys) {
              // slots past the end may hold NaN, and 0 * NaN in P V would reach the result
              if (!warp_wait_phase(fb, ring.phase, ctl, kStatusTimeoutLoad)) { ok = false; break; }
              uint8_t* v = smem + L::kKV + ring.stage * L::kSlotBytes;
              for (int x = left * 8 + lane; x < kTileKeys * 8; x += 32) {
                reinterpret_cast<uint4*>(v)[x] = make_uint4(0u, 0u, 0u, 0u);
                reinterpret_cast<uint4*>(v + kBoxBytes)[x] = make_uint4(0u, 0u, 0u, 0u);
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(L::kVFix + ring.stage));
            }
          } else if (lane == 0) {
            mbar_arrive(fb);
          }
          ring.advance<Slots>();
        }
      }
      if (*abort_flag) {
        // Let every copy this warp issued land before the block exits.
        volatile uint32_t no_abort = 0;
        WaitCtl drain{&no_abort, tp.status, tp.wait_limit_ns};
        for (int s = 0; s < Slots; ++s)
          if (st.was_armed(s)) wait_phase(bar(L::kKVFull + s), st.armed_parity(s), drain, kStatusTimeoutDrain);
        // the parity of the last Q load's phase; with none it is the one that a new barrier has behind it
        if (!side_v) wait_phase(bar(L::kQFull), st.q_empty(), drain, kStatusTimeoutDrain);
      }
      __syncwarp();
    } else if (warp == 9) {
      // ============================= MMA issuer =============================
      constexpr uint32_t idesc_qk = make_idesc_bf16(kBlockM, kTileKeys, false);
      constexpr uint32_t idesc_pv = make_idesc_bf16(kBlockM, kHeadDim, true);
      Ring ring;
      MmaParities<true> par;
      uint32_t fix_par = 0;  // bit s: parity of the V fix barrier of slot s
      bool ok = true;
      const uint64_t dk = make_sdesc_sw128(sbase, 16, 1024);
      const uint64_t dv = make_sdesc_sw128(sbase, kBoxBytes, 1024);
      const uint32_t k_lo = static_cast<uint32_t>(dk), k_hi = static_cast<uint32_t>(dk >> 32);
      const uint32_t v_lo = static_cast<uint32_t>(dv), v_hi = static_cast<uint32_t>(dv >> 32);
      // S = Q_i K^T into TMEM columns 128 s; O_o += P V, P at columns 128 s
      auto issue_s = [&](int i, int s, int slot) {
        const uint32_t qa = k_lo + ((L::kQ + i * kTileBytes) >> 4);
        const uint32_t ka = k_lo + ((L::kKV + slot * L::kSlotBytes + kTileBytes) >> 4);
        const uint32_t d = tmem + s * 128;
#pragma unroll
        for (int k = 0; k < kHeadDim / 16; ++k) {
          const uint32_t off = ((k / 4) * kBoxBytes + (k % 4) * 32) >> 4;
          umma_ss_w(d, qa + off, k_hi, ka + off, k_hi, idesc_qk, k > 0 ? 1u : 0u);
        }
        tc_commit(bar(L::kSFull + s));
      };
      auto issue_pv = [&](int o, int s, int slot, bool acc) {
        const uint32_t va = v_lo + ((L::kKV + slot * L::kSlotBytes) >> 4);
        const uint32_t d = tmem + 256 + o * 128, pa = tmem + s * 128;
        umma_ts_w(d, pa, va, v_hi, idesc_pv, acc ? 1u : 0u);
#pragma unroll
        for (int k = 1; k < kTileKeys / 16; ++k) umma_ts_w(d, pa + k * 8, va + ((k * 2048) >> 4), v_hi, idesc_pv, 1u);
      };
      Piece w;
      while (ok && next_piece(&w)) {
        const int n0 = tile_steps(w, 0), n1 = QTiles > 1 ? tile_steps(w, 1) : 0;
        const int N = max(n0, n1);
        if (N == 0) continue;
        if (lane == 0) {
          // the last V tile has rows past the end of the sequence
          const bool ragged = static_cast<int64_t>(w.tile0 + N) * kTileKeys > w.len;
          auto wait_fix = [&](int slot) -> bool {
            if (!mbar_wait(bar(L::kVFix + slot), (fix_par >> slot) & 1u, ctl, kStatusTimeoutMma)) return false;
            fix_par ^= 1u << slot;
            return true;
          };
          if (!mbar_wait(bar(L::kQFull), par.q_full(), ctl, kStatusTimeoutMma)) ok = false;
          par.flip_q_full();
          if constexpr (QTiles == 1) {
            // two key streams: step j goes through S buffer j % 2 into O_(j % 2)
            for (int pb = 0; pb < 2 && pb < N && ok; ++pb) {
              if (!mbar_wait(bar(L::kKVFull + ring.stage), ring.phase, ctl, kStatusTimeoutMma)) { ok = false; break; }
              tc_fence_after();
              issue_s(0, pb, ring.stage);
              tc_commit(bar(L::kKVEmpty + ring.stage));
              ring.advance<Slots>();
            }
            if (N <= 2 && ok) tc_commit(bar(L::kQEmpty));
            if (ok && !mbar_wait(bar(L::kKVFull + ring.stage), ring.phase, ctl, kStatusTimeoutMma)) ok = false;
            for (int j = 0; j < N && ok; ++j) {
              const int b = j & 1, cur = ring.stage;
              if (!mbar_wait(bar(L::kPFull + b), par.p_full(b), ctl, kStatusTimeoutMma)) { ok = false; break; }
              par.flip_p_full(b);
              if (j < 2) {
                if (!mbar_wait(bar(L::kOEmpty + b), par.o_empty(b), ctl, kStatusTimeoutMma)) { ok = false; break; }
                par.flip_o_empty(b);
              }
              if (ragged && j + 1 == N && !wait_fix(cur)) { ok = false; break; }
              tc_fence_after();
              issue_pv(b, b, cur, j > 1);
              if (j + 2 >= N) tc_commit(bar(L::kOFull + b));
              if (j + 2 < N) issue_s(0, b, cur);
              tc_commit(bar(L::kKVEmpty + cur));
              if (j + 3 == N) tc_commit(bar(L::kQEmpty));
              ring.advance<Slots>();
              if (j + 1 < N && !mbar_wait(bar(L::kKVFull + ring.stage), ring.phase, ctl, kStatusTimeoutMma)) {
                ok = false;
                break;
              }
            }
          } else {
            if (ok && !mbar_wait(bar(L::kKVFull + ring.stage), ring.phase, ctl, kStatusTimeoutMma)) ok = false;
            if (ok) {
              tc_fence_after();
              if (n0 > 0) issue_s(0, 0, ring.stage);
              if (n1 > 0) issue_s(1, 1, ring.stage);
              tc_commit(bar(L::kKVEmpty + ring.stage));
              if (N == 1) tc_commit(bar(L::kQEmpty));
              ring.advance<Slots>();
              if (!mbar_wait(bar(L::kKVFull + ring.stage), ring.phase, ctl, kStatusTimeoutMma)) ok = false;
            }
            for (int j = 0; j < N && ok; ++j) {
              const int cur = ring.stage;
              Ring nxt = ring;
              nxt.advance<Slots>();
              if (ragged && j + 1 == N && !wait_fix(cur)) { ok = false; break; }
#pragma unroll
              for (int i = 0; i < QTiles; ++i) {
                const int ni = i == 0 ? n0 : n1;
                if (j < ni && ok) {
                  if (!mbar_wait(bar(L::kPFull + i), par.p_full(i), ctl, kStatusTimeoutMma)) { ok = false; continue; }
                  par.flip_p_full(i);
                  if (j == 0) {
                    if (!mbar_wait(bar(L::kOEmpty + i), par.o_empty(i), ctl, kStatusTimeoutMma)) { ok = false; continue; }
                    par.flip_o_empty(i);
                  }
                  tc_fence_after();
                  issue_pv(i, i, cur, j > 0);
                  if (j + 1 == ni) tc_commit(bar(L::kOFull + i));
                }
                if (i == QTiles - 1 && j + 1 < N && ok) {
                  if (!mbar_wait(bar(L::kKVFull + nxt.stage), nxt.phase, ctl, kStatusTimeoutMma)) { ok = false; continue; }
                }
                if (j + 1 < ni && ok) issue_s(i, i, cur);
              }
              if (!ok) break;
              tc_commit(bar(L::kKVEmpty + cur));
              if (j + 2 == N) tc_commit(bar(L::kQEmpty));
              ring = nxt;
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
      }
      if (lane == 0) {
        // Every MMA this thread issued has finished once this barrier flips.
        tc_commit(bar(L::kTeardown));
        volatile uint32_t no_abort = 0;
        WaitCtl drain{&no_abort, tp.status, tp.wait_limit_ns};
        mbar_wait(bar(L::kTeardown), 0, drain, kStatusTimeoutDrain);
      }
      __syncwarp();
    } else {
      // ============================== schedule ==============================
      int4 cut = make_int4(0, 0, 0, -1);
      int out = 0;
      bool ok = true;
      auto put = [&](const Piece& w) {  // lane 0
        const int s = out % kPieceSlots;
        if (!wait_phase(bar(L::kPieceEmpty + s), ((out / kPieceSlots) & 1u) ^ 1u, ctl, kStatusTimeoutLoad)) {
          ok = false;
          return;
        }
        int4* dst = reinterpret_cast<int4*>(pieces + s);
        dst[0] = make_int4(w.token0, w.tokens, w.past, w.len);
        dst[1] = make_int4(w.h, w.b, w.tile0, w.cnt);
        dst[2] = make_int4(w.n, 0, 0, 0);
        mbar_arrive(bar(L::kPieceFull + s));  // releases the writes above
        ++out;
      };
      if (begin < end) {
        int64_t base = scan[12], pos = begin;
        int b = static_cast<int>(scan[13]);
        SeqView s = {static_cast<int>(scan[15]), static_cast<int>(scan[16]), static_cast<int>(scan[17])};
        int64_t head_work = scan[14];
        while (true) {
          const int64_t stop = min(end, base + head_work * p.c.kv_heads);
          if (pos < stop) {
            const int units = (s.sq + bt - 1) / bt;
            int h = static_cast<int>(quotient(pos - base, head_work));
            // the unit that holds `pos`: the last r whose earlier units end at or before it, 32 probes a round
            const int64_t x = pos - base - h * head_work;
            int r = 0, hi = units;  // r fits, hi does not
            int64_t before = 0;     // cost of the units before r
            while (hi - r > 1) {
              const int step = (hi - r + 31) / 32;
              const int64_t probe = r + static_cast<int64_t>(lane) * step;
              const int64_t sum = probe < hi ? units_cost(s, p.causal, bt, probe) : 0;
              const int n = __popc(__ballot_sync(0xffffffffu, probe < hi && sum <= x));  // lane 0 always fits
              before = __shfl_sync(0xffffffffu, sum, n - 1);
              r += (n - 1) * step;
              hi = min(hi, r + step);
            }
            if (lane == 0) {
              int64_t first = base + h * head_work + before;  // the unit's place on the line
              while (first < stop && ok) {
                Piece w;
                w.n = unit_steps(s, p.causal, bt, r);
                const int64_t step0 = first + kUnitExtra;  // the place of its first step
                w.tile0 = steps_before(begin - step0, w.n);
                w.cnt = steps_before(end - step0, w.n) - w.tile0;
                w.token0 = s.q0 + r * bt;
                w.tokens = min(bt, s.sq - r * bt);
                w.past = s.len - s.sq + r * bt;
                w.len = s.len;
                w.h = h;
                w.b = b;
                if (w.cnt > 0) put(w);
                if (w.tile0 == 0 && w.cnt > 0 && w.cnt < w.n)
                  cut = make_int4(w.token0, w.tokens, h, static_cast<int>(quotient(step0 + w.n - 1, per)));
                first = step0 + w.n;
                if (++r == units) {
                  r = 0;
                  ++h;
                }
              }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            pos = stop;
          }
          if (pos >= end) break;
          base += head_work * p.c.kv_heads;
          ++b;
          s = seq_view(p.c, p.cu, p.total_q, p.max_sq, p.causal, b);
          head_work = tile_seq_work(s, p.causal, bt);
        }
      }
      if (lane == 0) {
        tp.cut[blockIdx.x] = cut;
        if (ok) {
          Piece w = {};
          put(w);  // cnt = 0: no more
        }
      }
    }
  } else {
    // ============================== softmax ===============================
    // Two Q tiles: warpgroup i has tile i. One Q tile: warpgroup i has the tile's steps i, i + 2, ... with an
    // m, l and O of its own, which both warpgroups join at the end of the piece, 64 columns each.
    regs_claim<kTileSoftmaxRegs>();
    constexpr int kStreams = QTiles == 1 ? 2 : 1;
    constexpr int kCols = 128 / kStreams;  // columns of O that this thread finishes
    const int i = warp / 4;
    const int tile = QTiles == 1 ? 0 : i;
    const int row = (warp % 4) * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>((warp % 4) * 32) << 16;
    const uint32_t t_s = tmem + lane_off + i * 128;
    const uint32_t t_o = tmem + lane_off + 256 + i * 128;
    const int col0 = QTiles == 1 ? i * kCols : 0;
    float2* ml_shared = reinterpret_cast<float2*>(smem + L::kMl);  // [stream][row]
    uint32_t s_par = 0, o_full_par = 0, x_par = 0;  // o_full: bit x for O_x
    const float scale_log2 = p.scale_log2;
    const int row_token = row / p.group;  // token of this row within the Q tile
    const int row_head = row - row_token * p.group;
    bool ok = true;
    Piece w;
    while (ok && next_piece(&w, true)) {
      const int t0 = tile * tp.tile_tokens;
      if (t0 >= w.tokens) continue;  // no rows in this Q tile
      const int ni = tile_steps(w, tile);
      const bool live = row_token < tp.tile_tokens && t0 + row_token < w.tokens;
      const int first_lim = p.causal ? w.past + t0 : w.len - 1;            // last visible key of the tile's first row
      const int lim_row = p.causal ? w.past + t0 + row_token : w.len - 1;  // and of this one
      const int j0 = QTiles == 1 ? i : 0;
      float m = -INFINITY, l = 0.f;
      for (int j = j0; j < ni; j += kStreams) {
        if (!warp_wait(bar(L::kSFull + i), s_par, ctl, kStatusTimeoutSoftmax)) { ok = false; break; }
        s_par ^= 1u;
        tc_fence_after();
        uint32_t sr[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, sr[c]);
        tmem_ld_wait();
        float s[128];
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] = __uint_as_float(sr[c / 32][c % 32]);
        const int key0 = (w.tile0 + j) * kTileKeys;
        if (key0 + kTileKeys - 1 > min(first_lim, w.len - 1)) {
          const int lim = min(lim_row, w.len - 1) - key0;
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c > lim ? -INFINITY : s[c];
        }
        float mx0 = fmax3(s[0], s[1], s[2]), mx1 = fmax3(s[3], s[4], s[5]);
        float mx2 = fmax3(s[6], s[7], s[8]), mx3 = fmax3(s[9], s[10], s[11]);
#pragma unroll
        for (int c = 12; c < 124; c += 8) {
          mx0 = fmax3(mx0, s[c], s[c + 1]);
          mx1 = fmax3(mx1, s[c + 2], s[c + 3]);
          mx2 = fmax3(mx2, s[c + 4], s[c + 5]);
          mx3 = fmax3(mx3, s[c + 6], s[c + 7]);
        }
        mx0 = fmax3(mx0, s[124], s[125]);
        mx1 = fmax3(mx1, s[126], s[127]);
        const float mx = fmax3(fmaxf(mx0, mx1), mx2, mx3) * scale_log2;
        const float cand = fmaxf(m, mx);
        const bool update = (j == j0) || (cand > m + kRescaleThreshold);
        const float m_new = update ? cand : m;
        const bool rescale = (j > j0) && __any_sync(0xffffffffu, update);
        const float alpha = rescale ? ((m_new == -INFINITY) ? 1.f : ex2_mufu(m - m_new)) : 1.f;
        m = m_new;
        const float mb = (m == -INFINITY) ? 0.f : m;
        const float rowsum = exp_pack_store<0, true>(s, scale_log2, mb, t_s);
        l = l * alpha + rowsum;
        if (rescale) {
          // O_i holds every earlier step of this stream: the commit that released S covers them
          const float2 a2 = make_float2(alpha, alpha);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t orow[32];
            tmem_ld32(t_o + c * 32, orow);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 v = __fmul2_rn(make_float2(__uint_as_float(orow[e]), __uint_as_float(orow[e + 1])), a2);
              orow[e] = __float_as_uint(v.x);
              orow[e + 1] = __float_as_uint(v.y);
            }
            tmem_st32(t_o + c * 32, orow);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::kPFull + i));
      }
      // ------------------------------ epilogue ------------------------------
      float ov[kCols];
      if constexpr (QTiles == 1) {
        // both streams' (m, l), exchanged with bounded waits like every other: a hardware barrier would wait for
        // good for a warp that gave up
        if (!ok || !warp_wait(bar(L::kXEmpty), x_par ^ 1u, ctl, kStatusTimeoutSoftmax)) { ok = false; break; }
        ml_shared[i * 128 + row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::kXFull));
        if (!warp_wait(bar(L::kXFull), x_par, ctl, kStatusTimeoutSoftmax)) { ok = false; break; }
        const float2 x0 = ml_shared[row], x1 = ml_shared[128 + row];
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::kXEmpty));
        x_par ^= 1u;
        const float top = fmaxf(x0.x, x1.x), zero = top == -INFINITY ? 0.f : top;
        const float a0 = exp2f(x0.x - zero), a1 = exp2f(x1.x - zero);
        m = top;
        l = x0.y * a0 + x1.y * a1;
#pragma unroll
        for (int c = 0; c < kCols; ++c) ov[c] = 0.f;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (ni > x && ok) {
            ok = warp_wait(bar(L::kOFull + x), (o_full_par >> x) & 1u, ctl, kStatusTimeoutSoftmax);
            o_full_par ^= 1u << x;
            if (ok) {
              tc_fence_after();
              uint32_t part[kCols / 32][32];
#pragma unroll
              for (int c = 0; c < kCols / 32; ++c) tmem_ld32(tmem + lane_off + 256 + x * 128 + col0 + c * 32, part[c]);
              tmem_ld_wait();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(L::kOEmpty + x));
              const float a = x == 0 ? a0 : a1;
#pragma unroll
              for (int c = 0; c < kCols; ++c) ov[c] = fmaf(__uint_as_float(part[c / 32][c % 32]), a, ov[c]);
            }
          }
        }
        if (!ok) break;
      } else {
        if (!ok) break;
        if (ni > 0) {
          if (!warp_wait(bar(L::kOFull + i), o_full_par, ctl, kStatusTimeoutSoftmax)) { ok = false; break; }
          o_full_par ^= 1u;
          tc_fence_after();
          uint32_t part[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(t_o + c * 32, part[c]);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(L::kOEmpty + i));
#pragma unroll
          for (int c = 0; c < kCols; ++c) ov[c] = __uint_as_float(part[c / 32][c % 32]);
        } else {
#pragma unroll
          for (int c = 0; c < kCols; ++c) ov[c] = 0.f;
        }
      }
      if (w.cnt < w.n) {  // a piece: (m, l, O) to the workspace
        if (!live) continue;
        const int64_t at = part_tile(2 * blockIdx.x + (w.tile0 == 0 ? 1 : 0), QTiles, tile);
        float4* dst = reinterpret_cast<float4*>(p.part_o) + at * 4096 + (col0 / 4) * 128 + row;
#pragma unroll
        for (int c = 0; c < kCols / 4; ++c)
          dst[c * 128] = make_float4(ov[4 * c], ov[4 * c + 1], ov[4 * c + 2], ov[4 * c + 3]);
        if (col0 == 0) reinterpret_cast<float2*>(p.part_ml)[at * 128 + row] = make_float2(m, l);
        continue;
      }
      const int64_t token = w.token0 + t0 + row_token;
      const int head = w.h * p.group + row_head;
      const int64_t orow = token * p.heads + head, lse_at = static_cast<int64_t>(head) * p.total_q + token;
      float a = 1.f, x = 0.f;
      if (live && p.add_o != nullptr) {  // the other result of this row, joined in
        const float other = __ldcg(p.add_lse + lse_at) * 1.4426950408889634f;
        // relative to 0 where neither saw a key: a NaN of either still goes through
        const float top = fmaxf(m, other), zero = top == -INFINITY ? 0.f : top;
        a = exp2f(m - zero);
        x = exp2f(other - zero);
        l = l * a + x;
        m = top;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      a *= inv;
      x *= inv;
      if (live && p.lse != nullptr && col0 == 0) p.lse[lse_at] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
      const int place = live ? static_cast<int>(orow) : -1;
#pragma unroll
      for (int half = 0; half < kCols / 64; ++half) {
        const float4* add = reinterpret_cast<const float4*>(p.add_o + orow * 128 + col0 + half * 64);
        uint4 pieces16[8];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const float* q = ov + half * 64 + 4 * c;
          float4 u = make_float4(q[0] * a, q[1] * a, q[2] * a, q[3] * a);
          float4 v = make_float4(q[4] * a, q[5] * a, q[6] * a, q[7] * a);
          if (live && p.add_o != nullptr) {
            const float4 e = __ldcg(add + c), f = __ldcg(add + c + 1);
            u = make_float4(fmaf(e.x, x, u.x), fmaf(e.y, x, u.y), fmaf(e.z, x, u.z), fmaf(e.w, x, u.w));
            v = make_float4(fmaf(f.x, x, v.x), fmaf(f.y, x, v.y), fmaf(f.z, x, v.z), fmaf(f.w, x, v.w));
          }
          if (p.o == nullptr && live) {
            reinterpret_cast<float4*>(p.o32 + orow * 128 + col0 + half * 64)[c] = u;
            reinterpret_cast<float4*>(p.o32 + orow * 128 + col0 + half * 64)[c + 1] = v;
          }
          pieces16[c / 2] =
              make_uint4(pack_bf16x2(u.x, u.y), pack_bf16x2(u.z, u.w), pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        }
        if (p.o == nullptr) continue;
        if constexpr (QTiles == 1) {
          // eight lanes write 128 bytes of one row, instead of 32 lanes 16 bytes of as many: 4 prompts of 4096
          // tokens 173 -> 167 us with one Q tile per block; with two, whose other tile hides the stores, 155 -> 157
          transpose_pieces(pieces16, lane);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int at = __shfl_sync(0xffffffffu, place, (lane & 24) + k);
            if (at >= 0)
              reinterpret_cast<uint4*>(p.o + static_cast<int64_t>(at) * 128 + col0)[lane & 7] = pieces16[k];
          }
        } else if (live) {
#pragma unroll
          for (int k = 0; k < 8; ++k) reinterpret_cast<uint4*>(p.o + orow * 128 + half * 64)[k] = pieces16[k];
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds up the pieces of the units that paged_tile_kernel cut, in key order: O = sum 2^(m_c - M) O_c / L,
// M = max m_c, L = sum 2^(m_c - M) l_c. Reads each piece once and writes each row once: L2 traffic, and at
// small sizes its latency. 128 threads take C of the 32 column pieces of a unit's Q tile, one row each.
// Halves = 1: the two halves of a block work on their own (many units, few pieces each). Halves = 2: they
// share one item's pieces (two units of 64 pieces still have work for every SM). 148 units of two or three pieces,
// 39 MB: 14-17 us with cold caches; a few units: 6-9, most of it launch and latency.
template <int QTiles, int C, int Halves>
__device__ __forceinline__ void join_items(const PagedTileParams& tp, const int4* cuts, const int* first_block,
                                           int count, float4* half_o, float2* half_ml) {
  static_assert(Halves == 1 || C == 1, "the halves meet in one piece per row");
  constexpr int kBatch = 8 / C;  // pieces whose loads are in flight together
  const PagedParams& p = tp.p;
  const int row = threadIdx.x % 128, half = threadIdx.x / 128;
  const int row_token = row / p.group, row_head = row - row_token * p.group;
  const float4* part_o = reinterpret_cast<const float4*>(p.part_o);
  const float2* part_ml = reinterpret_cast<const float2*>(p.part_ml);
  const int items = count * QTiles * (32 / C);
  const int first = Halves == 1 ? blockIdx.x * 2 + half : blockIdx.x, stride = Halves == 1 ? gridDim.x * 2 : gridDim.x;
  for (int item = first; item < items; item += stride) {
    const int u = item / (QTiles * (32 / C)), i = item / (32 / C) % QTiles, col = item % (32 / C) * C;
    const int4 c = cuts[u];
    const int t0 = i * tp.tile_tokens;
    if (t0 >= c.y) continue;  // the same for all threads that share the item
    const bool live = row_token < tp.tile_tokens && t0 + row_token < c.y;
    if (Halves == 1 && !live) continue;
    const int64_t token = c.x + t0 + row_token;
    const int head = c.z * p.group + row_head;
    const int64_t orow = token * p.heads + head, lse_at = static_cast<int64_t>(head) * p.total_q + token;
    const int c0 = first_block[u], parts = c.w - c0 + 1, mid = (parts + 1) / 2;
    const int from = Halves == 2 && half ? mid : 0, to = Halves == 2 && !half ? mid : parts;
    auto tile = [&](int x) { return part_tile(2 * (c0 + x) + (x == 0 ? 1 : 0), QTiles, i); };
    float m = -INFINITY, l = 0.f;
    float4 acc[C];
#pragma unroll
    for (int e = 0; e < C; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x0 = from; x0 < to && live; x0 += kBatch) {
      float2 ml[kBatch];
      float4 o[kBatch][C];
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        ml[x] = make_float2(-INFINITY, 0.f);
        if (x0 + x < to) ml[x] = __ldcg(part_ml + tile(x0 + x) * 128 + row);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          o[x][e] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (x0 + x < to) o[x][e] = __ldcg(part_o + tile(x0 + x) * 4096 + (col + e) * 128 + row);
        }
      }
      float top = m;
#pragma unroll
      for (int x = 0; x < kBatch; ++x) top = fmaxf(top, ml[x].x);
      // relative to 0 while no piece has seen a key: NaN sums still go through
      const float zero = top == -INFINITY ? 0.f : top, a = exp2f(m - zero);
      l *= a;
      m = top;
#pragma unroll
      for (int e = 0; e < C; ++e) acc[e] = make_float4(acc[e].x * a, acc[e].y * a, acc[e].z * a, acc[e].w * a);
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        const float b = exp2f(ml[x].x - zero);
        l = fmaf(ml[x].y, b, l);
#pragma unroll
        for (int e = 0; e < C; ++e)
          acc[e] = make_float4(fmaf(o[x][e].x, b, acc[e].x), fmaf(o[x][e].y, b, acc[e].y),
                               fmaf(o[x][e].z, b, acc[e].z), fmaf(o[x][e].w, b, acc[e].w));
      }
    }
    if (Halves == 2) {
      if (half) {
        half_o[row] = acc[0];
        half_ml[row] = make_float2(m, l);
      }
      __syncthreads();
    }
    if (live && (Halves == 1 || !half)) {
      const float2 ml = Halves == 2 ? half_ml[row] : make_float2(-INFINITY, 0.f);
      const float other = p.add_o != nullptr ? __ldcg(p.add_lse + lse_at) * 1.4426950408889634f : -INFINITY;
      const float top = fmax3(m, ml.x, other), zero = top == -INFINITY ? 0.f : top;
      float a = exp2f(m - zero), b = exp2f(ml.x - zero), x = exp2f(other - zero);
      l = l * a + ml.y * b + x;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      a *= inv;
      b *= inv;
      x *= inv;
#pragma unroll
      for (int e = 0; e < C; ++e) {
        float4 v = make_float4(acc[e].x * a, acc[e].y * a, acc[e].z * a, acc[e].w * a);
        if (Halves == 2) {
          const float4 o = half_o[row];
          v = make_float4(fmaf(o.x, b, v.x), fmaf(o.y, b, v.y), fmaf(o.z, b, v.z), fmaf(o.w, b, v.w));
        }
        if (p.add_o != nullptr) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(p.add_o + orow * 128) + col + e);
          v = make_float4(fmaf(f.x, x, v.x), fmaf(f.y, x, v.y), fmaf(f.z, x, v.z), fmaf(f.w, x, v.w));
        }
        if (p.o != nullptr)
          *reinterpret_cast<uint2*>(p.o + orow * 128 + (col + e) * 4) =
              make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        else
          reinterpret_cast<float4*>(p.o32 + orow * 128)[col + e] = v;
      }
      if (p.lse != nullptr && col == 0) p.lse[lse_at] = l == 0.f ? -INFINITY : top * kLn2 + logf(l);
    }
    if (Halves == 2) __syncthreads();
  }
}

constexpr int kJoinPerSm = 4;

template <int QTiles>
__global__ void __launch_bounds__(256, kJoinPerSm) paged_join_kernel(const __grid_constant__ PagedTileParams tp, int blocks) {
  constexpr int kMaxCuts = 256;
  __shared__ int4 cuts[kMaxCuts];
  __shared__ int first_block[kMaxCuts];
  __shared__ int warp_cuts[kMaxCuts / 32];
  __shared__ float4 half_o[128];
  __shared__ float2 half_ml[128];
  wait_for_predecessor();
  // the cut units, numbered alike in every block: by the block that opens them (blocks <= kMaxCuts threads)
  const int warp = threadIdx.x / 32;
  const int4 mine = static_cast<int>(threadIdx.x) < blocks ? __ldcg(tp.cut + threadIdx.x) : make_int4(0, 0, 0, -1);
  const uint32_t opens = __ballot_sync(0xffffffffu, mine.w >= 0);
  if (threadIdx.x % 32 == 0) warp_cuts[warp] = __popc(opens);
  __syncthreads();
  int at = __popc(opens & ((1u << (threadIdx.x % 32)) - 1)), count = 0;
#pragma unroll
  for (int w = 0; w < kMaxCuts / 32; ++w) {
    if (w < warp) at += warp_cuts[w];
    count += warp_cuts[w];
  }
  if (mine.w >= 0) {
    cuts[at] = mine;
    first_block[at] = threadIdx.x;
  }
  __syncthreads();
  if (count * QTiles * 32 > 2 * static_cast<int>(gridDim.x))
    join_items<QTiles, 4, 1>(tp, cuts, first_block, count, half_o, half_ml);
  else
    join_items<QTiles, 1, 2>(tp, cuts, first_block, count, half_o, half_ml);
}

}  // namespace fav4
