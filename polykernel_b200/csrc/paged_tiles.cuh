// paged_tiles.cuh - attention over a paged cache for many rows per key head:
// prompts and chunks of them (tcgen05, sm_100a).
//
// Bound by the tensor cores and, equally, by exp: a pair of 128-row tiles costs
// 2048 cycles of tensor work per 128-key tile at head width 128, and 2 x 128 x
// 128 exponentials cost the same at 16 a cycle. One block therefore works on
// two 128-row tiles (A, B) that share every key tile, and alternates: while the
// tensor cores form P.V and the next S of one, a warpgroup takes the softmax of
// the other. Rows are the G heads of consecutive tokens, so a key tile is
// fetched once for the group.
//   warps 0-3, 4-7   softmax of A and of B: thread r owns row r (TMEM lane r),
//                    reads its 128 scores, and writes P back over them as
//                    16-bit pairs, the A operand of P.V.
//   warps 8-11       correction: rescale O in TMEM when a row's maximum moved
//                    by more than 2^8 (P stays below 2^8, the sums share the
//                    stale maximum, so the quotient is exact), and the epilogue.
//   warp 12          TMA: Q once, key and value pages into one ring.
//   warp 13          MMA issuer and TMEM owner.
//   warps 14, 15     clear value rows past the end of a sequence and look for
//                    values that are not finite in tiles that some row masks.
// TMEM: S/P of A [0,128), of B [128,256), O of A [256,384), of B [384,512).
//
// P is rounded once to the inputs' type (bf16: 2^-9 relative, fp16: 2^-12),
// the operand type that the tensor cores take with V; the errors of the keys
// are independent, so the output's stays at the level of its own rounding.
// The row sums are of the unrounded P, in fp32.
//
// With few row tiles over a long cache, `splits` blocks share a tile's keys and
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
  static constexpr int OFF_ALPHA = OFF_KV + STAGES * TILE;  // float[2][128]
  static constexpr int OFF_ML = OFF_ALPHA + 2 * 128 * 4;    // float2[2][128]
  static constexpr int OFF_BAR = OFF_ML + 2 * 128 * 8;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static constexpr int kRegsSoftmax = 192, kRegsCorrection = 80, kRegsControl = 48;
  static_assert(2 * kRegsSoftmax + kRegsCorrection + kRegsControl == 4 * 128, "launch: 512 x 128");
};
constexpr float kStaleMax = 8.f;  // log2 units a row's maximum may lag behind

template <typename T>
constexpr uint32_t mma_desc(int n, bool b_mn_major) {
  return std::is_same<T, __half>::value ? make_idesc_f16(128, n, false, b_mn_major)
                                        : make_idesc_bf16(128, n, false, b_mn_major);
}

// One row's attention over the keys [k0, k1) that it sees, by one warp, in fp32
// with plain loads: for tiles whose masked values are not finite. Lane d holds
// outputs d, d + 32, ...
template <typename T, int DP>
__device__ void exact_row(const AttnParams& p, int b, int hk, const T* q, int k0, int k1, float& m,
                          float& l, float (&o)[DP / 32]) {
  const int lane = lane_id();
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) o[c] = 0.f;
  auto row_of = [&](const void* pool, long long sp, long long sh, long long sr, int key) -> const T* {
    const int page = clip_page(__ldg(p.table + b * p.table_stride + key / p.page_size), p.num_pages);
    if (page == p.num_pages) return nullptr;  // zeros, as in the tiles
    return static_cast<const T*>(pool) + page * sp + hk * sh + (key % p.page_size) * sr;
  };
  for (int j0 = k0; j0 < k1; j0 += 32) {
    float s = -INFINITY;
    if (j0 + lane < k1) {
      const T* k = row_of(p.k, p.kp_p, p.kp_h, p.kp_r, j0 + lane);
      float dot = 0.f;
      if (k)
        for (int d = 0; d < p.D; d += 2) {
          const float2 x = unpack2<T>(*reinterpret_cast<const uint32_t*>(q + d));
          const float2 y = unpack2<T>(*reinterpret_cast<const uint32_t*>(k + d));
          dot = fmaf(x.x, y.x, dot);
          dot = fmaf(x.y, y.y, dot);
        }
      s = dot * p.scale_log2;
    }
    float top = s;
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    top = fmaxf(m, top);
    const float a = part_weight(m, top);
    const float e = s == -INFINITY ? 0.f : exp2f(s - top);
    m = top;
    float sum = e;
#pragma unroll
    for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    l = l * a + sum;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) o[c] *= a;
    for (int i = 0; i < min(32, k1 - j0); ++i) {
      const float w = __shfl_sync(0xffffffffu, e, i);
      const T* v = row_of(p.v, p.vp_p, p.vp_h, p.vp_r, j0 + i);
      if (!v) continue;
#pragma unroll
      for (int c = 0; c < DP / 32; ++c)
        if (lane + c * 32 < p.D) {
          const uint32_t u = reinterpret_cast<const uint16_t*>(v)[lane + c * 32];
          o[c] = fmaf(w, unpack2<T>(u).x, o[c]);
        }
    }
  }
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
  float* alpha_s = reinterpret_cast<float*>(smem + C::OFF_ALPHA);
  float2* ml_s = reinterpret_cast<float2*>(smem + C::OFF_ML);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [STAGES]
  uint64_t* empty = full + STAGES;                                  // [STAGES]
  uint64_t* q_full = empty + STAGES;
  uint64_t* s_full = q_full + 1;       // [2] S of the tile is in TMEM
  uint64_t* alpha_full = s_full + 2;   // [2] its rescale factors are in alpha_s
  uint64_t* p_ready = alpha_full + 2;  // [2] P is in TMEM and O is rescaled
  uint64_t* o_done = p_ready + 2;      // [2] P.V is added to O
  uint64_t* ml_full = o_done + 2;      // [2] final maxima and sums are in ml_s
  // A masked value tile is on its way into that stage (the stage's earlier
  // phases are over, so that its `full` can be waited on by parity), and its
  // values are cleared and looked at. Per stage: several may be under way.
  uint64_t* v_look = ml_full + 2;      // [STAGES]
  uint64_t* v_fixed = v_look + STAGES; // [STAGES]
  long long* scan = reinterpret_cast<long long*>(v_fixed + STAGES);  // [16]
  int* found = reinterpret_cast<int*>(scan + 16);               // sequence, tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(found + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* by_hand = abort_flag + 1;
  static_assert((4 * STAGES + 11) * 8 + 16 * 8 + 5 * 4 <= 512, "barrier area");
  const int warp = warp_id(), lane = lane_id();

  grid_launch_dependents();
  // Block order: row tiles fastest, the longest first, then key heads, then
  // pieces of the keys, so that blocks which run together share keys in L2.
  const int tile = static_cast<int>(blockIdx.x) % p.tiles;
  const int hk = static_cast<int>(blockIdx.x) / p.tiles % p.Hkv;
  const int split = static_cast<int>(blockIdx.x) / p.tiles / p.Hkv;
  const int entry = hk * p.tiles + tile;
  Entry* const meta = reinterpret_cast<Entry*>(p.meta) + entry;
  const int tok = 128 / p.G;  // tokens of a 128-row tile
  auto tiles_of = [&](const Seq& s) {
    const int rows = s.nq * p.G;
    return rows >= p.min_rows && rows <= p.max_rows ? (s.nq + 2 * tok - 1) / (2 * tok) : 0;
  };
  {
    const int each = (p.B + C::kThreads - 1) / C::kThreads;
    const int b0 = static_cast<int>(threadIdx.x) * each, b1 = min(p.B, b0 + each);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(load_seq(p, b, true));
    long long total;
    const long long before = block_prefix<C::kThreads>(mine, scan, total);
    if (tile >= total) {
      if (p.splits > 1 && split == 0 && threadIdx.x == 0) meta->pieces = 0;
      return;
    }
    if (tile >= before && tile < before + mine) {
      int at = static_cast<int>(before);
      for (int b = b0;; ++b) {
        const int n = tiles_of(load_seq(p, b));
        if (tile < at + n) {
          found[0] = b;
          found[1] = n - 1 - (tile - at);
          break;
        }
        at += n;
      }
    }
    __syncthreads();
  }
  const int b = found[0];
  const Seq s = load_seq(p, b);
  const int first = found[1] * 2 * tok;                  // first token
  const int count = min(2 * tok, s.nq - first);          // tokens of both tiles
  const int rows = count * p.G;
  const bool two = count > tok;
  int tile0, tile1;
  int pieces;
  {
    int base;
    const int n = key_tiles<KT>(p, s, first, first + count - 1, base);
    pieces = min(p.splits, max(1, n / p.min_units));
    if (split >= pieces) return;
    tile0 = base + static_cast<int>(static_cast<long long>(n) * split / pieces);
    tile1 = base + static_cast<int>(static_cast<long long>(n) * (split + 1) / pieces);
  }
  const int nt = tile1 - tile0;
  if (split == 0 && p.splits > 1 && threadIdx.x == 0) {
    Entry e;
    e.pieces = pieces > 1 ? pieces : 0;
    e.t0 = s.t0;
    e.hk = hk;
    e.row0 = first * p.G;
    e.rows = rows;
    e.slot0 = entry * p.splits;
    e.slot1 = e.slot0 + 1;
    e.step = 1;
    *meta = e;
  }
  // keys that every row of the block sees
  const int all_hi = key_hi(p, s, first), all_lo = key_lo(p, s, first + count - 1);
  auto masked = [&](int j) {
    const int key0 = (tile0 + j) * KT;
    return key0 + KT > all_hi || key0 < all_lo;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
      mbar_init(&v_look[i], 1);
      mbar_init(&v_fixed[i], 64);
    }
    mbar_init(q_full, 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&alpha_full[x], 128);
      mbar_init(&p_ready[x], 256);
      mbar_init(&o_done[x], 1);
      mbar_init(&ml_full[x], 128);
    }
    *abort_flag = 0;
    *by_hand = 0;
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

  if (warp >= 12) {
    setmaxnreg_dec<C::kRegsControl>();
    if (warp == 12) {
      // ------------------------------------------------------------ fetch --
      if (lane == 0) {
        mbar_arrive_expect_tx(q_full, (two ? 2 : 1) * C::HALVES * tok * p.G * 128);
        for (int x = 0; x < (two ? 2 : 1); ++x)
          for (int c = 0; c < C::HALVES; ++c)
            tma_load_3d(smem + x * C::TILE + c * (128 * 128), &map_q, q_full, c * 64, hk * p.G,
                        s.t0 + first + x * tok);
      }
      __syncwarp();
      const int boxes = KT / p.box;
      const int col = lane / boxes, bx = lane - col * boxes;
      const bool mine = col < C::HALVES;
      auto lookup = [&](int j) {
        const int key = (tile0 + j) * KT + bx * p.box;
        return mine && key < s.len ? page_of(p, b, key) : -1;
      };
      int stage = 0, issued = 0;
      uint32_t parity = 1;
      bool ok = true;
      int page = lookup(0);
      for (int j = 0; j < nt && ok; ++j) {
        const int next = j + 1 < nt ? lookup(j + 1) : -1;
        const int row = ((tile0 + j) * KT + bx * p.box) % p.page_size;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * p.box * 128;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&empty[stage], parity, p.err, abort_flag,
                                                       kErrTimeoutProducer));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&full[stage], bytes);
          __syncwarp();
          if (page >= 0)
            tma_load_4d(smem + C::OFF_KV + stage * C::TILE + col * (KT * 128) + bx * p.box * 128,
                        kv ? &map_v : &map_k, &full[stage], col * 64, row, hk, page);
          if (kv && lane == 0 && masked(j)) mbar_arrive(&v_look[stage]);
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            parity ^= 1;
          }
        }
        page = next;
      }
      if (!ok || *abort_flag) {  // do not leave while copies into this block's memory are in flight
        const long long t0 = clock64();
        while (!mbar_try_wait(q_full, 0) && clock64() - t0 < kSpinLimitCycles) {}
        for (int i = max(0, issued - STAGES); i < issued; ++i)
          while (!mbar_try_wait(&full[i % STAGES], (i / STAGES) & 1) && clock64() - t0 < kSpinLimitCycles) {}
      }
    } else if (warp == 13) {
      // ------------------------------------------------------- MMA issuer --
      // The whole warp runs the loop; one elected lane issues.
      constexpr uint32_t desc_s = mma_desc<T>(KT, false), desc_o = mma_desc<T>(DP, true);
      const uint32_t q_addr = smem_u32(smem), kv_addr = smem_u32(smem + C::OFF_KV);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.err, abort_flag, kErrTimeoutMma));
      };
      auto issue_s = [&](int x, int j) {
        const uint32_t k_addr = kv_addr + (2 * j % STAGES) * C::TILE;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t at = (kk >> 2) * (128 * 128) + (kk & 3) * 32;
          tc_mma_f16_warp(tmem + x * 128, make_sw128_desc(q_addr + x * C::TILE + at, 16, 1024),
                          make_sw128_desc(k_addr + at, 16, 1024), desc_s, kk != 0);
        }
        tc_commit_warp(&s_full[x]);
      };
      auto issue_pv = [&](int x, int j) {
        const uint32_t v_addr = kv_addr + ((2 * j + 1) % STAGES) * C::TILE;
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk)
          tc_mma_f16_tmem_a_warp(tmem + 256 + x * 128, tmem + x * 128 + kk * 8,
                                 make_sw128_desc(v_addr + kk * 2048, KT * 128, 1024), desc_o,
                                 (j != 0 || kk != 0));
        tc_commit_warp(&o_done[x]);
      };
      const int last = two ? 1 : 0;
      bool ok = wait(q_full, 0) && wait(&full[0], 0);
      if (ok) {
        tc_fence_after();
        for (int x = 0; x <= last; ++x) issue_s(x, 0);
        tc_commit_warp(&empty[0]);
      }
      uint32_t fixed = 0;  // phases of v_fixed, a bit per stage
      for (int j = 0; j < nt && ok; ++j) {
        const int cv = 2 * j + 1, ck = 2 * j + 2;  // places of V(j) and K(j + 1) in the ring
        ok = wait(&full[cv % STAGES], (cv / STAGES) & 1);
        if (ok && masked(j)) {
          ok = wait(&v_fixed[cv % STAGES], (fixed >> (cv % STAGES)) & 1);
          fixed ^= 1u << (cv % STAGES);
        }
        for (int x = 0; x <= last && ok; ++x) {
          ok = wait(&p_ready[x], j & 1);
          if (!ok) break;
          tc_fence_after();
          issue_pv(x, j);
          if (x == last) tc_commit_warp(&empty[cv % STAGES]);
          if (j + 1 < nt) {
            // S(j + 1) overwrites P(j), which the P.V just issued reads first:
            // MMAs run in the order of their issue.
            if (x == 0) {
              ok = wait(&full[ck % STAGES], (ck / STAGES) & 1);
              if (!ok) break;
              tc_fence_after();
            }
            issue_s(x, j + 1);
            if (x == last) tc_commit_warp(&empty[ck % STAGES]);
          }
        }
      }
    } else {
      // ------------------------------------------ values of masked tiles --
      const int t = static_cast<int>(threadIdx.x) - 14 * 32;
      uint32_t looked = 0;  // phases of v_look, a bit per stage
      for (int j = 0; j < nt; ++j) {
        if (!masked(j)) continue;
        const int cv = 2 * j + 1, st = cv % STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(&v_look[st], (looked >> st) & 1, p.err, abort_flag,
                                               kErrTimeoutConvert) &&
                                         mbar_wait(&full[st], (cv / STAGES) & 1, p.err, abort_flag,
                                                   kErrTimeoutConvert)))
          break;
        looked ^= 1u << st;
        uint8_t* v = smem + C::OFF_KV + st * C::TILE;
        const int key0 = (tile0 + j) * KT;
        bool bad = false;
#pragma unroll 4
        for (int i = t; i < KT * C::HALVES * 8; i += 64) {
          const int key = (i >> 3) % KT;
          uint4* w = reinterpret_cast<uint4*>(v + i * 16);
          if (key0 + key >= s.len) *w = make_uint4(0u, 0u, 0u, 0u);
          else {
            const uint4 u = *w;
            bad |= not_finite2<T>(u.x) || not_finite2<T>(u.y) || not_finite2<T>(u.z) || not_finite2<T>(u.w);
          }
        }
        if (bad) *by_hand = 1;
        fence_proxy_async_smem();
        mbar_arrive(&v_fixed[st]);
      }
    }
  } else if (warp < 8) {
    // ----------------------------------------------------------- softmax --
    setmaxnreg_inc<C::kRegsSoftmax>();
    const int x = warp >> 2;
    const int r = static_cast<int>(threadIdx.x) & 127;
    // rows past the tile's last one repeat it; nobody reads them
    const int i = first + min(x * tok + r / p.G, count - 1);
    const int hi = key_hi(p, s, i), lo = key_lo(p, s, i);
    const uint32_t sp = tmem + x * 128 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < nt && (x == 0 || two); ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[x], j & 1, p.err, abort_flag, kErrTimeoutSoftmax)))
        break;
      tc_fence_after();
      uint32_t sv[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(sp + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&sv[c * 32]));
      tmem_ld_wait();
      const int key0 = (tile0 + j) * KT;
      if (__any_sync(0xffffffffu, key0 + KT > hi || key0 < lo)) {
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (key0 + c >= hi || key0 + c < lo) sv[c] = __float_as_uint(-INFINITY);
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < 64; ++k)
        mx4[k & 3] = fmax3(mx4[k & 3], __uint_as_float(sv[2 * k]), __uint_as_float(sv[2 * k + 1]));
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
      float alpha = 1.f;
      if (mx > m + kStaleMax || (m == -INFINITY && mx > -INFINITY)) {
        alpha = part_weight(m, mx);
        l *= alpha;
        m = mx;
      }
      alpha_s[x * 128 + r] = alpha;
      mbar_arrive(&alpha_full[x]);
      const float neg = m == -INFINITY ? 0.f : -m;
      const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2), ng2 = f2_pack(neg, neg);
      uint64_t sum2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int at = c * 32 + 2 * k;
          float e0, e1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(sv[at]), __uint_as_float(sv[at + 1])), sc2, ng2), e0, e1);
          e0 = fast_exp2(e0);
          e1 = fast_exp2(e1);
          sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(e0, e1));
          pk[k] = pack2<T>(e0, e1);
        }
        tmem_st16(sp + c * 16, pk);
      }
      {
        float a0, a1, b0, b1;
        f2_unpack(sum2[0], a0, a1);
        f2_unpack(sum2[1], b0, b1);
        l += (a0 + b0) + (a1 + b1);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_ready[x]);
    }
    ml_s[x * 128 + r] = make_float2(m, l);
    mbar_arrive(&ml_full[x]);
  } else {
    // -------------------------------------------------------- correction --
    setmaxnreg_dec<C::kRegsCorrection>();
    const int r = static_cast<int>(threadIdx.x) - 256;
    const uint32_t lane_base = tmem + 256 + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    bool ok = true;
    for (int j = 0; j < nt && ok; ++j) {
      for (int x = 0; x < (two ? 2 : 1); ++x) {
        ok = __all_sync(0xffffffffu, mbar_wait(&alpha_full[x], j & 1, p.err, abort_flag, kErrTimeoutSoftmax));
        if (!ok) break;
        const float a = alpha_s[x * 128 + r];
        // (S(j) follows P.V(j - 1) in the tensor pipe: this one is over by now)
        if (j > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait(&o_done[x], (j - 1) & 1, p.err, abort_flag, kErrTimeoutSoftmax));
          if (!ok) break;
        }
        if (j > 0 && __any_sync(0xffffffffu, a != 1.f)) {
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(lane_base + x * 128 + c * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * a);
            tmem_st32(lane_base + x * 128 + c * 32, o);
          }
          tmem_st_wait();
          tc_fence_before();
        }
        mbar_arrive(&p_ready[x]);
      }
    }
    // ---------------------------------------------------------- epilogue --
    for (int x = 0; x < (two ? 2 : 1) && ok; ++x) {
      ok = __all_sync(0xffffffffu, mbar_wait(&ml_full[x], 0, p.err, abort_flag, kErrTimeoutSoftmax)) &&
           __all_sync(0xffffffffu, mbar_wait(&o_done[x], (nt - 1) & 1, p.err, abort_flag, kErrTimeoutEpilogue));
      if (!ok) break;
      tc_fence_after();
      const float2 ml = ml_s[x * 128 + r];
      const int row = x * tok * p.G + r;
      const bool valid = r < tok * p.G && row < rows;
      if (pieces == 1) {
        const float inv = inverse_sum(ml.y);
        const int tr = (valid ? row : 0) / p.G, h = hk * p.G + (valid ? row : 0) % p.G;
        const long long t = s.t0 + first + tr;
        T* dst = static_cast<T*>(p.out) + t * p.os_t + h * p.os_h;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(lane_base + x * 128 + c * 32, o);
          tmem_ld_wait();
          if (valid) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              if (c * 32 + k < p.D) {
                uint4 w;
                w.x = pack2<T>(__uint_as_float(o[k]) * inv, __uint_as_float(o[k + 1]) * inv);
                w.y = pack2<T>(__uint_as_float(o[k + 2]) * inv, __uint_as_float(o[k + 3]) * inv);
                w.z = pack2<T>(__uint_as_float(o[k + 4]) * inv, __uint_as_float(o[k + 5]) * inv);
                w.w = pack2<T>(__uint_as_float(o[k + 6]) * inv, __uint_as_float(o[k + 7]) * inv);
                *reinterpret_cast<uint4*>(dst + c * 32 + k) = w;
              }
            }
          }
        }
        if (valid && p.lse) p.lse[t * p.Hq + h] = log_sum(ml.x, ml.y);
      } else {
        const long long at = (static_cast<long long>(entry) * p.splits + split) * 256 + row;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(lane_base + x * 128 + c * 32, o);
          tmem_ld_wait();
          if (valid) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<uint4*>(p.part_o + at * DP + c * 32 + k) =
                  make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        }
        if (valid) p.part_ml[at] = ml;
      }
    }
    tc_fence_before();
  }

  tc_fence_before();
  // Back to 128 registers a thread for the common tail; those that grow wait
  // until the softmax warps have given theirs up.
  if (warp < 8) setmaxnreg_dec<128>();
  __syncthreads();
  if (warp >= 8) setmaxnreg_inc<128>();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (*by_hand && !*abort_flag) {
    for (int row = warp; row < rows; row += C::kThreads / 32) {
      const int tr = first + row / p.G, h = hk * p.G + row % p.G;
      const long long t = s.t0 + tr;
      const T* q = static_cast<const T*>(p.q) + t * p.qs_t + h * p.qs_h;
      float m, l, o[DP / 32];
      exact_row<T, DP>(p, b, hk, q, max(tile0 * KT, key_lo(p, s, tr)), min(tile1 * KT, key_hi(p, s, tr)), m, l, o);
      const long long at = (static_cast<long long>(entry) * p.splits + split) * 256 + row;
      const float inv = inverse_sum(l);
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) {
        const int d = lane + c * 32;
        if (pieces > 1) p.part_o[at * DP + d] = o[c];
        else if (d < p.D)
          reinterpret_cast<uint16_t*>(static_cast<T*>(p.out) + t * p.os_t + h * p.os_h)[d] =
              static_cast<uint16_t>(pack2<T>(o[c] * inv, 0.f));
      }
      if (lane == 0) {
        if (pieces > 1) p.part_ml[at] = make_float2(m, l);
        else if (p.lse) p.lse[t * p.Hq + h] = log_sum(m, l);
      }
    }
  }
}

}  // namespace paged
}  // namespace pkb200
