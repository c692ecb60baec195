// paged_tiles.cuh - attention over a paged cache for many rows per key head:
// prompts and chunks of them (tcgen05, sm_100a).
//
// Bound by the tensor cores and, equally, by exp: a pair of 128-row tiles costs
// 2048 cycles of tensor work per 128-key tile at head width 128, and their 2 x
// 128 x 128 exponentials cost the same at 16 a cycle. So a block works on two
// 128-row tiles (A, B) that share every key tile: while the tensor cores form
// P.V and the next S of one, a warpgroup takes the softmax of the other. Rows are
// the G heads of consecutive tokens, so a key tile is fetched once for the group.
// Long runs are under the power cap: a quarter of the exponentials formed on the
// FMA pipe instead took as many cycles and 3% more time, at a lower clock.
//   warps 0-3, 4-7   softmax of A and of B: thread r owns row r (TMEM lane r),
//                    reads its 128 scores, writes P back over them as 16-bit
//                    pairs (the A operand of P.V), rescales O in TMEM when the
//                    row's maximum moved by more than 2^8 (P stays below 2^8 and
//                    the sums share the stale maximum, so the quotient is
//                    exact), and writes the output.
//   warps 8-11       in tiles that some row masks: clear value rows that no row
//                    sees and take values that are not finite out of the others.
//   warp 12          TMA: Q, and key and value pages into one ring.
//   warp 13          MMA issue, and owner of TMEM.
//   warp 14          work: blocks stay resident and take over the work of blocks
//                    that have not been launched yet (cluster launch control),
//                    in the grid's order, one item ahead of the other warps.
//   (warp 15 completes a warpgroup.)
// TMEM: S/P of A [0,128), of B [128,256), O of A [256,384), of B [384,512).
//
// P is rounded once to the inputs' type (by at most 2^-8 of it in bf16, 2^-11 in
// fp16), the operand type that the tensor cores take with V: an error of at most
// that share of sum p |v|, and where weights differ, whose errors then add up like
// independent ones, about as much as the output's own rounding (2.3e-3 in all on
// normal data, where rounding the exact output gives 1.7e-3). Two terms per weight, as with
// few rows, would double the tensor work of P.V. The row sums are of the
// unrounded P, in fp32.
//
// Measured (bf16, 128-wide heads, two cards): an 8190-token prompt of 32 heads on 8
// key heads 540 to 549 us, 1000 to 1018 TFLOP/s (0.63 of the burst matrix rate, 0.74 of the
// sustained one; the run is power capped at 1.7 GHz); 4 x 32 heads x 2048 tokens over
// 4096 keys 464 to 474 us, 870 to 889 TFLOP/s; 509 tokens of 28 heads on 4 over 130k keys
// 967 to 989 us, 961 to 983 TFLOP/s. A key tile takes a pair of row tiles 3400 cycles: their
// chains (S, softmax, P.V, and the hand-overs between) alternate, and the tensor pipe
// waits nearly half of the time (54% active); an item's begin and end cost 5000 to 9000
// cycles more.
//
// With few row tiles over a long cache, `splits` items share a tile's keys and
// paged_join_kernel adds their pieces up.
#pragma once

#include "paged_common.cuh"

namespace pkb200 {
namespace paged {

template <int DP>
struct TilesCfg {
  static constexpr int KT = 128;
  static constexpr int kThreads = 512;
  static constexpr int HALVES = DP / 64;
  static constexpr int TILE = 128 * DP * 2;  // one 128-row tile of Q, K or V
  static constexpr int STAGES = DP == 128 ? 4 : 8;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_OUT = OFF_KV + STAGES * TILE;  // 4 KB per softmax warp
  static constexpr int OFF_WORK = OFF_OUT + 8 * 4096;     // TileWork[2]
  static constexpr int OFF_BAR = OFF_WORK + 2 * 64;
  static constexpr int kBarBytes = 512;
  static constexpr int SMEM = OFF_BAR + kBarBytes + 1024;
  static constexpr int kRegsSoftmax = 176, kRegsValues = 80, kRegsControl = 80;
  static_assert(2 * kRegsSoftmax + kRegsValues + kRegsControl == 4 * 128, "launch: 512 x 128");
  static_assert(SMEM <= 232448, "shared memory of an SM");
};

constexpr int kEarly = 2;  // quarters of a tile's keys whose P is handed over ahead of the rest

// One item of work, as the work warp hands it to the others.
struct alignas(64) TileWork {
  int b;              // sequence; -1: no more items
  Seq s;
  int first, count;   // tokens of both tiles
  int hk, tile0, nt;  // key head, key tiles [tile0, tile0 + nt)
  int pieces, slot;   // pieces of these rows' keys, and where this one goes
  int all_lo, all_hi; // keys that every row sees
  int special;        // values that are not finite were taken out of masked tiles
};
static_assert(sizeof(TileWork) == 64, "");

// Asks for the work of a block that has not been launched yet; the answer, 16
// bytes at `answer`, completes `bar`.
__device__ __forceinline__ void take_block_async(void* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
// The index of the block taken over, -1 if there is none left.
__device__ __forceinline__ int taken_block(const void* answer) {
  int got;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "mov.s32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
      : "=r"(got)
      : "r"(smem_u32(answer))
      : "memory");
  return got;
}

template <typename T>
constexpr uint32_t mma_desc(int n, bool b_mn_major) {
  return std::is_same<T, __half>::value ? make_idesc_f16(128, n, false, b_mn_major)
                                        : make_idesc_bf16(128, n, false, b_mn_major);
}

// The MMAs of one tile, issued warp-wide (tc_mma_f16_warp); descriptors advance by
// constants. S [128 x 128] = Q K^T: 16 columns of the head per MMA, 32 bytes
// within a 128-byte row, 16 KB between 64-column halves.
template <typename T, int DP>
__device__ __forceinline__ void issue_s(uint32_t s_tmem, uint64_t q_desc, uint64_t k_desc) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const uint64_t off = (kk >> 2) * 1024 + (kk & 3) * 2;
    tc_mma_f16_warp(s_tmem, q_desc + off, k_desc + off, mma_desc<T>(128, false), kk != 0);
  }
}
// O [128 x DP] (+)= P V for the keys [16 FROM, 16 TO): 8 TMEM columns and 2 KB of V each.
template <typename T, int DP, int FROM, int TO>
__device__ __forceinline__ void issue_pv(uint32_t o_tmem, uint32_t p_tmem, uint64_t v_desc, uint32_t add) {
#pragma unroll
  for (int kk = FROM; kk < TO; ++kk)
    tc_mma_f16_tmem_a_warp(o_tmem, p_tmem + kk * 8, v_desc + kk * 128, mma_desc<T>(DP, true),
                           kk == FROM ? add : 1u);
}

// Goes over the values of a warp's 32 rows again, and puts what decides their
// columns into O: all of them if a value in O is not finite (`counts`: of a row for
// which that matters), else those of masked tiles, from which they were taken out.
template <typename T, int DP>
__device__ __forceinline__ void decide_rows(const AttnParams& p, const TileWork& w, int x, int tok, uint32_t o_tmem,
                                            bool counts, int* state) {
  constexpr int KT = TilesCfg<DP>::KT;
  const int row0 = x * tok * p.G + (warp_id() & 3) * 32;  // of the item; the warp's first
  const int rows = max(0, min(32, min((x + 1) * tok, w.count) * p.G - row0));
  bool odd = false;
#pragma unroll 1
  for (int c = 0; c < DP / 32; ++c) {
    uint32_t o[32];
    tmem_ld32(o_tmem + c * 32, o);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 32; ++k) odd |= !(fabsf(__uint_as_float(o[k])) < INFINITY);
  }
  const int begin = w.tile0 * KT, end = begin + w.nt * KT;
  int from = begin, to = end;  // keys of the item, or first those of its masked tiles at one end
  const int low = min(end, (w.all_lo + KT - 1) / KT * KT), high = max(begin, w.all_hi / KT * KT);
  const bool ends = !__any_sync(0xffffffffu, odd && counts) && low < high;
  if (ends) to = low;
  uint32_t marks[DP / 16] = {};
#pragma unroll 1
  while (true) {
    mark_values<T, DP>(p, w.b, w.hk, w.s, w.first * p.G + row0, rows, from, to, marks, [&] { atomicAdd(state, 2); });
    if (to == end) break;
    from = high;
    to = end;
  }
#pragma unroll 1
  for (int c = 0; c < DP / 32; ++c) {
    uint32_t o[32];
    tmem_ld32(o_tmem + c * 32, o);
    tmem_ld_wait();
#pragma unroll
    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(marked<DP>(__uint_as_float(o[k]), marks, c * 32 + k));
    tmem_st32(o_tmem + c * 32, o);
  }
  tmem_st_wait();
}

template <typename T, int DP>
__global__ void __launch_bounds__(TilesCfg<DP>::kThreads, 1)
    paged_tiles_kernel(const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const AttnParams p) {
  using C = TilesCfg<DP>;
  constexpr int KT = C::KT, STAGES = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  TileWork* work = reinterpret_cast<TileWork*>(smem + C::OFF_WORK);  // [2]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [STAGES]
  uint64_t* empty = full + STAGES;                                  // [STAGES]
  // A masked value tile is on its way into that stage (the stage's earlier
  // phases are over, so that its `full` can be waited on by parity), and its
  // values are cleared and looked at. Per stage: several may be under way.
  uint64_t* v_look = empty + STAGES;   // [STAGES]
  uint64_t* v_fixed = v_look + STAGES; // [STAGES]
  uint64_t* q_full = v_fixed + STAGES;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;      // [2] S of the tile is in TMEM
  uint64_t* p_ready = s_full + 2;      // [2] P of the first keys is in TMEM and O is rescaled
  uint64_t* p_rest = p_ready + 2;      // [2] P of the others
  uint64_t* o_full = p_rest + 2;       // [2] the item's last P.V is added to O
  uint64_t* work_full = o_full + 2;    // [2]
  uint64_t* work_empty = work_full + 2;  // [2]
  uint64_t* taken = work_empty + 2;    // the answer about the next block is there
  uint64_t* ask = taken + 1;           // the item's loads are nearly all issued
  void* answer = taken + 2;            // 16 bytes, 16-byte aligned
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(taken + 4);
  // Bit 0: the kernel is given up; above it, counted up while values are gone over again.
  int* state = reinterpret_cast<int*>(tmem_slot + 1);
  const volatile int* watched = state;
  static_assert((4 * STAGES + 18) * 8 + 8 <= C::kBarBytes, "barrier area");
  static_assert((4 * STAGES + 16) % 2 == 0, "the answer is 16-byte aligned");
  const int warp = warp_id(), lane = lane_id();
  const int tok = 128 / p.G;  // tokens of a 128-row tile

  grid_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&v_look[i], 1);
      mbar_init(&v_fixed[i], 128);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_ready[x], 128);
      mbar_init(&p_rest[x], 128);
      mbar_init(&o_full[x], 1);
      mbar_init(&work_full[x], 1);
      mbar_init(&work_empty[x], 14);
    }
    mbar_init(taken, 1);
    mbar_init(ask, 1);
    *state = 0;
    fence_barrier_init();
  }
  if (warp == 13) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Whole-warp wait; false if the kernel is to be given up: another role did,
  // or the limit ran out (`late` then tells that this warp is the first). The
  // limit runs anew while softmax warps go over values again.
  bool ok = true, late = false;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    long long t0 = clock64();
    int seen = 0;
    while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
      const int now = *watched;
      if (now & 1) return false;
      if (now != seen) {
        seen = now;
        t0 = clock64();
      }
      if (clock64() - t0 > kSpinLimitCycles) {
        late = true;
        atomicOr(state, 1);
        return false;
      }
    }
    return true;
  };
  // For what is in flight into this block's memory when the kernel is given up.
  auto wait_late = [&](uint64_t* bar, uint32_t parity) {
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity) && clock64() - t0 < kSpinLimitCycles) {}
    return false;
  };
  // The next item for this warp (`item` counts them); false at the end.
  int item = 0;
  auto next_work = [&] {
    ok = wait(&work_full[item & 1], (item >> 1) & 1);
    return ok && work[item & 1].b >= 0;
  };
  auto release_work = [&] {
    __syncwarp();
    if (lane == 0) mbar_arrive(&work_empty[item & 1]);
    ++item;
  };
  auto masked = [&](const TileWork& w, int j) {
    const int key0 = (w.tile0 + j) * KT;
    return key0 + KT > w.all_hi || key0 < w.all_lo;
  };

  if (warp >= 12) {
    setmaxnreg_dec<C::kRegsControl>();
    if (warp == 12) {
      // ------------------------------------------------------------ fetch --
      if (lane == 0) {
        tma_prefetch_desc(&map_q);
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
      }
      const int boxes = KT / p.box;
      const int col = lane / boxes, bx = lane - col * boxes;
      const bool mine = col < C::HALVES;
      int stage = 0, issued = 0;
      uint32_t parity = 1;
      while (ok && next_work()) {
        const TileWork w = work[item & 1];
        const bool two = w.count > tok;
        // (not for keys that no row of the item sees: pages behind a window may be gone)
        const int seen_lo = key_lo(p, w.s, w.first), seen_hi = key_hi(p, w.s, w.first + w.count - 1);
        auto lookup = [&](int j) {
          const int key = (w.tile0 + j) * KT + bx * p.box;
          return mine && key + p.box > seen_lo && key < seen_hi ? page_of(p, w.b, key) : -1;
        };
        int page = lookup(0);
        for (int j = 0; j < w.nt && ok; ++j) {
          if (j == max(0, w.nt - 3) && lane == 0) mbar_arrive(ask);
          const int next = j + 1 < w.nt ? lookup(j + 1) : -1;
          const int row = ((w.tile0 + j) * KT + bx * p.box) % p.page_size;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * p.box * 128;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            ok = ok && wait(&empty[stage], parity);
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
            __syncwarp();
            if (page >= 0)
              tma_load_4d(smem + C::OFF_KV + stage * C::TILE + col * (KT * 128) + bx * p.box * 128,
                          kv ? &map_v : &map_k, &full[stage], col * 64, row, w.hk, page);
            if (kv && lane == 0 && masked(w, j)) mbar_arrive(&v_look[stage]);
            ++issued;
            if (++stage == STAGES) {
              stage = 0;
              parity ^= 1;
            }
            if (j == 0 && kv == 0) {  // Q, once the last item's scores are formed
              ok = wait(q_empty, (item & 1) ^ 1);
              if (!ok) break;
              if (lane == 0) {
                mbar_arrive_expect_tx(q_full, (two ? 2 : 1) * C::HALVES * tok * p.G * 128);
                for (int x = 0; x < (two ? 2 : 1); ++x)
                  for (int c = 0; c < C::HALVES; ++c)
                    tma_load_3d(smem + x * C::TILE + c * (128 * 128), &map_q, q_full, c * 64,
                                w.hk * p.G, w.s.t0 + w.first + x * tok);
              }
              __syncwarp();
            }
          }
          page = next;
        }
        if (ok) release_work();
      }
      if (*watched & 1) {
        wait_late(q_full, item & 1);
        for (int i = max(0, issued - STAGES); i < issued; ++i) wait_late(&full[i % STAGES], (i / STAGES) & 1);
      }
    } else if (warp == 13) {
      // -------------------------------------------------------- MMA issue --
      // The whole warp runs the loop; one elected lane issues. One warp serves both tiles
      // in turn: with a warp for each, their MMAs interleave in the tensor pipe,
      // both softmaxes wait at once, and the pipe runs dry. The loop is kept
      // short (one place for S, one for P.V): all roles share the instruction
      // cache with the softmax, whose loop is unrolled over a whole tile of keys.
      const uint64_t q_desc = make_sw128_desc(smem_u32(smem), 16, 1024);
      const uint64_t k_desc = make_sw128_desc(smem_u32(smem + C::OFF_KV), 16, 1024);
      const uint64_t v_desc = make_sw128_desc(smem_u32(smem + C::OFF_KV), KT * 128, 1024);
      uint32_t place = 0;  // of the item's first key tile in the ring
      uint32_t fixed = 0;  // phases of v_fixed, a bit per stage
      uint32_t done = 0;   // phases of p_ready, a bit per tile
      while (ok && next_work()) {
        const TileWork& w = work[item & 1];
        const int nt = w.nt, tile0 = w.tile0, all_lo = w.all_lo, all_hi = w.all_hi;
        const int last = w.count > tok ? 1 : 0;
        for (int j = -1; j < nt && ok; ++j) {  // P.V(j), then S(j + 1)
          const uint32_t cv = place + 2 * j + 1, ck = cv + 1;
          const uint32_t sv = cv % STAGES, sk = ck % STAGES;
          const bool more = j + 1 < nt;
          if (j >= 0) {
            const int key0 = (tile0 + j) * KT;
            ok = wait(&full[sv], (cv / STAGES) & 1);
            if (ok && (key0 + KT > all_hi || key0 < all_lo)) {
              ok = wait(&v_fixed[sv], (fixed >> sv) & 1);
              fixed ^= 1u << sv;
            }
          }
#pragma unroll 1
          for (int x = 0; x <= last && ok; ++x) {
            const uint32_t s_tmem = tmem + x * 128;
            if (j >= 0) {
              const uint32_t o_tmem = tmem + 256 + x * 128;
              const uint64_t vd = v_desc + sv * (C::TILE >> 4);
              ok = wait(&p_ready[x], (done >> x) & 1);
              if (!ok) break;
              tc_fence_after();
              issue_pv<T, DP, 0, 2 * kEarly>(o_tmem, s_tmem, vd, j != 0);
              ok = wait(&p_rest[x], (done >> x) & 1);
              if (!ok) break;
              tc_fence_after();
              issue_pv<T, DP, 2 * kEarly, 8>(o_tmem, s_tmem, vd, 1);
              done ^= 1u << x;
              if (x == last) tc_commit_warp(&empty[sv]);
              if (!more) tc_commit_warp(&o_full[x]);
            }
            if (more) {
              // S(j + 1) overwrites P(j), which the P.V just issued reads first:
              // MMAs run in the order of their issue.
              if (x == 0) {
                ok = wait(&full[sk], (ck / STAGES) & 1);
                if (ok && j < 0) ok = wait(q_full, item & 1);
                if (!ok) break;
                tc_fence_after();
              }
              issue_s<T, DP>(s_tmem, q_desc + x * (C::TILE >> 4), k_desc + sk * (C::TILE >> 4));
              tc_commit_warp(&s_full[x]);
              if (x == last) {
                tc_commit_warp(&empty[sk]);
                if (j + 2 == nt) tc_commit_warp(q_empty);
              }
            }
          }
        }
        place += 2 * nt;
        if (ok) release_work();
      }
    } else if (warp == 14) {
      // ------------------------------------------------------------- work --
      // Items in block order: row tiles fastest, a sequence's longest first,
      // then key heads, then pieces of the keys, so that items which run
      // together share keys in L2. The grid is the host's bound on them; the
      // blocks past the batch's own row tiles have nothing to do.
      // Lane i counts the row tiles of the i-th run of sequences.
      const int each = (p.B + 31) / 32, b0 = min(p.B, lane * each), b1 = min(p.B, b0 + each);
      auto tiles_of = [&](const Seq& s) {
        const int rows = s.nq * p.G;
        return rows >= p.min_rows && rows <= p.max_rows ? (s.nq + 2 * tok - 1) / (2 * tok) : 0;
      };
      int mine = 0;
#pragma unroll 4
      for (int b = b0; b < b1; ++b) mine = min(mine + tiles_of(load_seq(p, b, true)), p.tiles);
      // (the host's bound holds for sequences that do not overlap; where offsets
      // run backwards and they do, what is above it is left out)
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto = min(upto + y, p.tiles);
      }
      const int total = __shfl_sync(0xffffffffu, upto, 31);
      int ahead = __shfl_up_sync(0xffffffffu, upto, 1);  // row tiles of the lanes before
      if (lane == 0) ahead = 0;
      const int rows_all = total * p.Hkv;  // row tiles of all heads
      int block = blockIdx.x;
      int asked = 0;
      for (;; ++asked) {
        TileWork w;
        w.b = -1;
        Seq s;
        int split = 0, entry = 0, tile = 0, hk = 0, n_of = 0, before = 0;
        if (block < rows_all * p.splits) {
          split = block / rows_all;
          entry = block - split * rows_all;
          hk = entry / total;
          tile = entry - hk * total;
          // the lane whose sequences have this row tile, and the sequence
          const int from = __ffs(__ballot_sync(0xffffffffu, upto > tile)) - 1;
          int b = b0, first = ahead, n = 0;
          if (lane == from) {
            while (true) {
              n = tiles_of(load_seq(p, b));
              if (tile < first + n) break;
              first += n;
              ++b;
            }
          }
          w.b = __shfl_sync(0xffffffffu, b, from);
          n_of = __shfl_sync(0xffffffffu, n, from);
          before = __shfl_sync(0xffffffffu, first, from);
        } else if (block - rows_all * p.splits < p.tiles * p.Hkv - rows_all) {
          entry = rows_all + block - rows_all * p.splits;  // an entry that stays empty
        } else {
          split = 1;
        }
        bool live = w.b >= 0;
        w.pieces = 0;
        if (live) {
          s = load_seq(p, w.b);
          w.s = s;
          w.first = (n_of - 1 - (tile - before)) * 2 * tok;
          w.count = min(2 * tok, s.nq - w.first);
          w.hk = hk;
          int base;
          const int n = key_tiles<KT>(p, s, w.first, w.first + w.count - 1, base);
          w.pieces = min(p.splits, max(1, n / p.min_units));
          w.tile0 = base + static_cast<int>(static_cast<long long>(n) * split / w.pieces);
          w.nt = base + static_cast<int>(static_cast<long long>(n) * (split + 1) / w.pieces) - w.tile0;
          w.slot = entry * p.splits + split;
          w.all_hi = key_hi(p, s, w.first);
          w.all_lo = key_lo(p, s, w.first + w.count - 1);
          w.special = 0;
          live = split < w.pieces;
        }
        if (split == 0 && p.splits > 1 && lane == 0) {
          Entry e = {};
          if (live && w.pieces > 1) {
            e.pieces = w.pieces;
            e.t0 = s.t0;
            e.hk = hk;
            e.row0 = w.first * p.G;
            e.rows = w.count * p.G;
            e.slot0 = entry * p.splits;
            e.slot1 = e.slot0 + 1;
            e.step = 1;
          }
          reinterpret_cast<Entry*>(p.meta)[entry] = e;
        }
        if (live) {
          if (!wait(&work_empty[item & 1], ((item >> 1) & 1) ^ 1)) break;
          if (lane == 0) {
            work[item & 1] = w;
            mbar_arrive(&work_full[item & 1]);
          }
          __syncwarp();
          ++item;
        }
        // The next block is asked for when this item's loads are nearly done and
        // not before: what a block holds back, an idle one cannot take.
        if (live && !wait(ask, (item - 1) & 1)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(taken, 16);
          take_block_async(answer, taken);
        }
        __syncwarp();
        // (waited for to the limit even when the kernel is given up: the answer
        // is written into this block's memory)
        const bool answered = wait(taken, asked & 1) || wait_late(taken, asked & 1);
        block = answered ? taken_block(answer) : -1;
        fence_proxy_async_smem();  // before the next answer overwrites this one
        __syncwarp();
        if (block < 0) {
          if (answered && wait(&work_empty[item & 1], ((item >> 1) & 1) ^ 1) && lane == 0) {
            work[item & 1].b = -1;
            mbar_arrive(&work_full[item & 1]);
          }
          __syncwarp();
          break;
        }
      }
    }
  } else if (warp < 8) {
    // ----------------------------------------------------------- softmax --
    setmaxnreg_inc<C::kRegsSoftmax>();
    const int x = warp >> 2;
    const int r = static_cast<int>(threadIdx.x) & 127;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + x * 128 + lanes, o_tmem = tmem + 256 + x * 128 + lanes;
    uint8_t* stage = smem + C::OFF_OUT + warp * 4096;
    uint32_t tiles = 0, outputs = 0;
    while (ok && next_work()) {
      const TileWork& w = work[item & 1];
      const int nt = w.nt, tile0 = w.tile0;
      if (x == 1 && w.count <= tok) {
        release_work();
        continue;
      }
      // rows past the tile's last one repeat it; nobody reads them
      const int i = w.first + min(x * tok + r / p.G, w.count - 1);
      const int hi = key_hi(p, w.s, i), lo = key_lo(p, w.s, i);
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < nt; ++j, ++tiles) {
        ok = wait(&s_full[x], tiles & 1);
        if (!ok) break;
        tc_fence_after();
        const int key0 = (tile0 + j) * KT;
        const int begin = lo - key0, end = hi - key0;  // columns that this row sees
        const bool hides = __any_sync(0xffffffffu, end < KT || begin > 0);
        uint32_t sv[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[c * 32]));
        tmem_ld_wait();
        if (hides) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c < begin || c >= end) sv[c] = __float_as_uint(-INFINITY);
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 64; ++k)
          mx4[k & 3] = fmax3(mx4[k & 3], __uint_as_float(sv[2 * k]), __uint_as_float(sv[2 * k + 1]));
        const float mx = fmaxf(fmax3(mx4[0], mx4[1], mx4[2]), mx4[3]) * p.scale_log2;
        float alpha = 1.f;
        if (mx > m + kStaleMax || (m == -INFINITY && mx > -INFINITY)) {
          alpha = part_weight(m, mx);
          l *= alpha;
          m = mx;
        }
        if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
          // (P.V of the tile before this one precedes S in the tensor pipe)
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(o_tmem + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
            tmem_st16(o_tmem + c * 16, o);
          }
        }
        const float neg = m == -INFINITY ? 0.f : -m;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), ng2 = f2_pack(neg, neg);
        uint64_t sum2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int at = c * 32 + 2 * k;
            const uint64_t x2 =
                f2_fma(f2_pack(__uint_as_float(sv[at]), __uint_as_float(sv[at + 1])), sc2, ng2);
            float e0, e1;
            f2_unpack(x2, e0, e1);
            e0 = fast_exp2(e0);
            e1 = fast_exp2(e1);
            sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(e0, e1));
            pk[k] = pack2<T>(e0, e1);
          }
          tmem_st16(s_tmem + c * 16, pk);
          if (c == kEarly - 1) {  // P.V may start on the keys so far
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&p_ready[x]);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_rest[x]);
        float a0, a1, b0, b1;
        f2_unpack(sum2[0], a0, a1);
        f2_unpack(sum2[1], b0, b1);
        l += (a0 + b0) + (a1 + b1);
      }
      if (!ok) break;
      // ------------------------------------------------------------ output --
      ok = wait(&o_full[x], outputs & 1);
      if (!ok) break;
      ++outputs;
      tc_fence_after();
      const int row = x * tok * p.G + r;
      const bool valid = r < tok * p.G && row < w.count * p.G;
      const int tr = row / p.G, h = w.hk * p.G + row - tr * p.G;
      const long long t = w.s.t0 + w.first + tr;
      const bool whole = w.pieces == 1;
      const long long part = static_cast<long long>(w.slot) * 256 + row;
      const bool counts = valid && fabsf(l) < INFINITY;
      // due: values of the item's keys that are not finite are to be brought into O
      bool due = *reinterpret_cast<volatile int*>(&work[item & 1].special) != 0, decided = false;
      {
        // Through shared memory, 128 bytes of each of the warp's 32 rows at a
        // time (16-byte chunks swizzled by row), so that rows leave as whole
        // 128-byte lines: lane 8 q + c has chunk c of rows q, q + 4, ...
        const float inv = whole ? inverse_sum(l) : 1.f;
        uint8_t* mine = !valid ? nullptr
                        : whole ? reinterpret_cast<uint8_t*>(static_cast<T*>(p.out) + t * p.os_t + h * p.os_h)
                                : reinterpret_cast<uint8_t*>(p.part_o + part * DP);
        uint8_t* to[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
          to[q] = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine),
                                                         q * 4 + (lane >> 3)));
        const int row_bytes = whole ? p.D * 2 : DP * 4;
#pragma unroll 1
        for (int c0 = 0; c0 < (whole ? DP / 64 : DP / 32); ++c0) {
          if (due) {
            decide_rows<T, DP>(p, w, x, tok, o_tmem, counts, state);
            due = false;
            decided = true;
          }
          uint32_t o[32];
          const uint64_t zero = f2_pack(0.f, 0.f);
          uint64_t odd = zero;  // 0, NaN where a value is not finite
          if (whole) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              tmem_ld32(o_tmem + c0 * 64 + half * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; k += 2)
                odd = f2_fma(f2_pack(__uint_as_float(o[k]), __uint_as_float(o[k + 1])), zero, odd);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint4 v;
                v.x = pack2<T>(__uint_as_float(o[8 * k]) * inv, __uint_as_float(o[8 * k + 1]) * inv);
                v.y = pack2<T>(__uint_as_float(o[8 * k + 2]) * inv, __uint_as_float(o[8 * k + 3]) * inv);
                v.z = pack2<T>(__uint_as_float(o[8 * k + 4]) * inv, __uint_as_float(o[8 * k + 5]) * inv);
                v.w = pack2<T>(__uint_as_float(o[8 * k + 6]) * inv, __uint_as_float(o[8 * k + 7]) * inv);
                *reinterpret_cast<uint4*>(stage + lane * 128 + (((half * 4 + k) ^ (lane & 7)) << 4)) = v;
              }
            }
          } else {
            tmem_ld32(o_tmem + c0 * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; k += 2)
              odd = f2_fma(f2_pack(__uint_as_float(o[k]), __uint_as_float(o[k + 1])), zero, odd);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((k ^ (lane & 7)) << 4)) =
                  make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
          float n0, n1;
          f2_unpack(odd, n0, n1);
          if (!decided && __any_sync(0xffffffffu, counts && n0 + n1 != 0.f)) {
            due = true;
            --c0;  // once more
            continue;
          }
          __syncwarp();
          uint4 v[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int rr = q * 4 + (lane >> 3);
            v[q] = *reinterpret_cast<const uint4*>(stage + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4));
          }
          const int at = c0 * 128 + (lane & 7) * 16;
          const bool in_row = at < row_bytes;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (to[q] && in_row) *reinterpret_cast<uint4*>(to[q] + at) = v[q];
          __syncwarp();
        }
        if (valid) {
          if (!whole) p.part_ml[part] = make_float2(m, l);
          else if (p.lse) p.lse[t * p.Hq + h] = log_sum(m, l);
        }
      }
      tc_fence_before();
      release_work();
    }
  } else {
    // ---------------------------------------------- values of masked tiles --
    // 0 * inf and 0 * NaN are NaN: value rows that no row of the item sees (stale
    // memory, or not fetched) are cleared, and other values of masked tiles that are not finite
    // taken out: the rows that see them get them with the output.
    setmaxnreg_dec<C::kRegsValues>();
    const int t = static_cast<int>(threadIdx.x) - 256;
    uint32_t place = 0, looked = 0;  // looked: phases of v_look, a bit per stage
    while (ok && next_work()) {
      const TileWork w = work[item & 1];
      const int seen_lo = key_lo(p, w.s, w.first), seen_hi = key_hi(p, w.s, w.first + w.count - 1);
      for (int j = 0; j < w.nt && ok; ++j, place += 2) {
        if (!masked(w, j)) continue;
        const uint32_t at = place + 1, st = at % STAGES;
        ok = wait(&v_look[st], (looked >> st) & 1) &&
             wait(&full[st], (at / STAGES) & 1);
        if (!ok) break;
        looked ^= 1u << st;
        uint8_t* v = smem + C::OFF_KV + st * C::TILE;
        const int key0 = (w.tile0 + j) * KT, live_lo = seen_lo - key0, live_hi = seen_hi - key0;
        uint32_t bad = 0;
#pragma unroll
        for (int c = 0; c < C::HALVES; ++c) {
          uint4 u[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) u[k] = *reinterpret_cast<const uint4*>(v + c * (KT * 128) + (k * 128 + t) * 16);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int key = k * 16 + (t >> 3);
            uint4* at16 = reinterpret_cast<uint4*>(v + c * (KT * 128) + (k * 128 + t) * 16);
            if (key < live_lo || key >= live_hi) {
              *at16 = make_uint4(0u, 0u, 0u, 0u);
            } else if (not_finite4<T>(u[k])) {
              *at16 = finite_only4<T>(u[k]);
              bad = 1;
            }
          }
        }
        if (bad) *reinterpret_cast<volatile int*>(&work[item & 1].special) = 1;
        fence_proxy_async_smem();
        mbar_arrive(&v_fixed[st]);
      }
      if (ok) release_work();
    }
  }

  if (late && lane == 0)
    atomicCAS(p.err, 0, warp < 8 ? kErrTimeoutSoftmax : warp < 12 ? kErrTimeoutConvert
                        : warp == 13 ? kErrTimeoutMma : kErrTimeoutProducer);
  // Back to 128 registers a thread; those that grow wait until the softmax
  // warps have given theirs up.
  tc_fence_before();
  if (warp < 8) setmaxnreg_dec<128>();
  __syncthreads();
  if (warp >= 8) setmaxnreg_inc<128>();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace paged
}  // namespace pkb200
