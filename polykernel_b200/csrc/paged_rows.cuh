// paged_rows.cuh - attention over a paged cache for few rows per key head:
// single tokens, drafted tokens, small groups of heads (sm_100a).
//
// Bound by reading every visible key and value once from HBM, so the work is
// split by keys: all 64-key tiles of the batch, over (sequence, key head, row
// tile), form one line that the grid cuts into equal runs, whatever the lengths
// are. A block that covers a row tile's keys from end to end writes the
// output; otherwise pieces go to the workspace (at most two per block: the
// tail of the tile it starts in and the head of the one it ends in) and
// paged_join_kernel adds them up. The lengths are read on the device.
//
// One warp per block fetches pages by TMA into a ring of key and value tiles;
// four warps work on them with mma.sync (M = 16 rows: a tcgen05 tile would be
// 7/8 empty, and the tensor work is a small part of the time of the reads).
// With MR = 16 rows each warp takes 16 of a tile's 64 keys with statistics of
// its own, merged at the end of the row tile; with MR = 32 or 64 two or all
// four warps take different rows. Up to 32 rows P enters the P.V product as two
// 16-bit terms (value and remainder), so the output carries no rounding of P:
// the second product costs nothing that the reads do not hide. With 64 rows the
// tensor work (8 cycles per mma.sync and sub-partition) comes near the time of the
// reads, and P is rounded once to the inputs' type, as in the tile kernel.
//
// Values that are not finite are kept out of the loop: see mark_values.
//
// Measured (8 key heads of 128, groups of 4, bf16): 64 sequences of up to 16k
// keys, 2.2 GB, in 333 us: 6.6 TB/s, the rate of a copy. One token over 4096 keys takes
// 11.2 us on the GPU (14 for a call among others), of which the reads are 2.6: two
// launches, the cut of the line, one tile's latency and the join. With 48 rows of
// 64-wide heads the chain of a tile (S, softmax, P.V, in one warp, two to a
// sub-partition) bounds it: 42 us on the GPU against 15 for the reads.
#pragma once

#include "paged_common.cuh"

namespace pkb200 {
namespace paged {

template <int DP, int MR>
struct RowsCfg {
  static constexpr int KT = 64;
  static constexpr int kThreads = 160;  // 4 compute warps, 1 that fetches
  static constexpr int WM = MR / 16, WK = 4 / WM, KW = KT / WK;  // warps by rows and by keys
  static constexpr int SLOT = KT * DP * 2;
  static constexpr bool kSplitP = MR <= 32;
  // Blocks per SM, as many as their registers allow: the work on a tile is a
  // chain of short steps. 130 to 150 KB per SM are in flight.
  static constexpr int kBlocks = DP <= 128 ? 2 : 1;
  static constexpr int SLOTS = DP == 64 ? 10 : 4;
  // Merge: each warp's 16 rows of fp32, rows 32 bytes apart in the banks
  static constexpr int STRIDE = DP + 8;
  static constexpr int OFF_STAGE = SLOTS * SLOT;
  static constexpr int OFF_ML = OFF_STAGE + 4 * 16 * STRIDE * 4;  // float2[4][16]
  static constexpr int OFF_MARKS = OFF_ML + 4 * 16 * 8;           // the rows' marks, uint32_t[MR][DP / 16]
  static constexpr int OFF_BAR = OFF_MARKS + MR * DP / 4;         // full[SLOTS], empty[SLOTS]
  static constexpr int OFF_SCAN = OFF_BAR + 2 * SLOTS * 8;        // long long[5], start of the run, flags
  static constexpr int SMEM = OFF_SCAN + 5 * 8 + 32 + 1024;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void compute_warps_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
// The same, and whether `ok` holds in all of them: one answer for all four warps.
__device__ __forceinline__ bool compute_warps_all(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok))
      : "memory");
  return all != 0;
}

constexpr int kAhead = 3;  // steps between the load of a fragment and its products

// 64-bit division is a long subroutine; most counts fit 32 bits.
__device__ __forceinline__ long long divide(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

// Place in the line of work: a row tile `rt` of key head `hk` of sequence `b`.
template <int MR>
struct RowCursor {
  const AttnParams& p;
  int b, hk, rt;
  Seq s;
  int rows, row_tiles;  // rows of the sequence
  int seen_lo, seen_hi; // keys that some row of this row tile sees
  int tile0, n;         // its key tiles

  __device__ explicit RowCursor(const AttnParams& p_) : p(p_) {}
  __device__ static int rows_of(const AttnParams& p, const Seq& s) {
    const int rows = s.nq * p.G;
    return rows >= p.min_rows && rows <= p.max_rows ? rows : 0;
  }
  // Tokens of the row tile, the first and the last.
  __device__ static int first_of(const AttnParams& p, int rows, int rt) { return rows <= MR ? 0 : rt * MR / p.G; }
  __device__ static int last_of(const AttnParams& p, const Seq& s, int rows, int rt) {
    return rows <= MR ? s.nq - 1 : (min(rows, rt * MR + MR) - 1) / p.G;
  }
  // Key tiles of a whole sequence (one key head).
  __device__ static long long units_of(const AttnParams& p, const Seq& s) {
    const int rows = rows_of(p, s);
    long long n = 0;
    int tile0;
    for (int rt = 0; rt * MR < rows; ++rt) n += key_tiles<64>(p, s, first_of(p, rows, rt), last_of(p, s, rows, rt), tile0);
    return n;
  }
  __device__ void load() {
    s = load_seq(p, b);
    rows = rows_of(p, s);
    row_tiles = (rows + MR - 1) / MR;
  }
  __device__ void set_tiles() {
    seen_lo = key_lo(p, s, first_of(p, rows, rt));
    seen_hi = key_hi(p, s, last_of(p, s, rows, rt));
    n = tiles_of_keys(seen_lo, seen_hi, 64, tile0);
  }
  // Start in sequence b, `rem` key tiles after its first one; returns the
  // offset within the row tile.
  __device__ int start(int b_, long long rem) {
    b = b_;
    load();
    const long long per_head = units_of(p, s);
    hk = static_cast<int>(divide(rem, per_head));
    rem -= hk * per_head;
    for (rt = 0;; ++rt) {
      set_tiles();
      if (rem < n) return static_cast<int>(rem);
      rem -= n;
    }
  }
  __device__ void next() {
    if (++rt == row_tiles) {
      rt = 0;
      if (++hk == p.Hkv) {
        hk = 0;
        do {
          ++b;
          load();
        } while (rows == 0);
      }
    }
    set_tiles();
  }
};

template <typename T, int DP, int MR>
__global__ void __launch_bounds__(RowsCfg<DP, MR>::kThreads, RowsCfg<DP, MR>::kBlocks)
    paged_rows_kernel(const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const AttnParams p) {
  using C = RowsCfg<DP, MR>;
  constexpr int KT = C::KT, KW = C::KW, WK = C::WK, SLOTS = C::SLOTS;
  constexpr int HALVES = DP / 64;  // 128-byte wide columns of a tile
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + SLOTS;
  long long* scan = reinterpret_cast<long long*>(smem + C::OFF_SCAN);
  long long* start_rem = scan + 5;
  int* start_b = reinterpret_cast<int*>(scan + 6);
  volatile int* abort_flag = start_b + 1;
  // [2] values of a run's keys were found that are not finite (by the run's parity)
  volatile int* special = start_b + 2;
  volatile int* alive = start_b + 4;  // see mbar_wait_alive
  const int warp = warp_id(), lane = lane_id();
  Entry* const meta = reinterpret_cast<Entry*>(p.meta) + blockIdx.x;

  grid_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    *abort_flag = special[0] = special[1] = *alive = 0;
    fence_barrier_init();
  }
  // This block's run [u0, u1) of the batch's key tiles.
  long long u0, u1, per_block;
  {
    const int each = (p.B + C::kThreads - 1) / C::kThreads;
    const int b0 = static_cast<int>(threadIdx.x) * each, b1 = min(p.B, b0 + each);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += p.Hkv * RowCursor<MR>::units_of(p, load_seq(p, b, true));
    long long total;
    const long long before = block_prefix<C::kThreads>(mine, scan, total);
    per_block = max(static_cast<long long>(p.min_units), divide(total + gridDim.x - 1, gridDim.x));
    u0 = blockIdx.x * per_block;
    u1 = min(total, u0 + per_block);
    if (u0 >= u1) {
      if (threadIdx.x == 0) meta->pieces = 0;
      return;
    }
    if (u0 >= before && u0 < before + mine) {
      long long at = before;
      for (int b = b0;; ++b) {
        const long long n = p.Hkv * RowCursor<MR>::units_of(p, load_seq(p, b));
        if (u0 < at + n) {
          *start_b = b;
          *start_rem = u0 - at;
          break;
        }
        at += n;
      }
    }
    __syncthreads();
  }
  RowCursor<MR> at(p);
  int off = at.start(*start_b, *start_rem);

  if (warp == 4) {
    // ------------------------------------------------------------- fetch --
    if (lane == 0) {
      tma_prefetch_desc(&map_k);
      tma_prefetch_desc(&map_v);
    }
    const int boxes = KT / p.box;  // per tile and column
    const int col = lane / boxes, bx = lane - col * boxes;
    const bool mine = col < HALVES;
    int slot = 0, issued = 0;
    uint32_t parity = 1;
    bool ok = true;
    if (p.hold_back) {
      const long long t0 = clock64();
      while (clock64() - t0 < p.hold_back) {}
    }
    for (long long u = u0; u < u1 && ok;) {
      const int run = static_cast<int>(min(static_cast<long long>(at.n - off), u1 - u));
      // Keys that no row of the tile sees are not looked up: pages behind a
      // window may be gone.
      auto lookup = [&](int tile) {  // this lane's page in that key tile
        const int key = (at.tile0 + tile) * KT + bx * p.box;
        return mine && key + p.box > at.seen_lo && key < at.seen_hi ? page_of(p, at.b, key) : -1;
      };
      int page = lookup(off);
      for (int i = 0; i < run && ok; ++i) {
        const int key = (at.tile0 + off + i) * KT + bx * p.box;
        const int next = i + 1 < run ? lookup(off + i + 1) : -1;
        const int row = key % p.page_size;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, page >= 0)) * p.box * 128;
#pragma unroll
        for (int kv = 0; kv < 2 && ok; ++kv) {
          ok = __all_sync(0xffffffffu, mbar_wait_alive(&empty[slot], parity, p.err, abort_flag,
                                                       kErrTimeoutProducer, p.wait_limit, alive));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&full[slot], bytes);
          __syncwarp();
          if (page >= 0)
            tma_load_4d(smem + slot * C::SLOT + col * (KT * 128) + bx * p.box * 128, kv ? &map_v : &map_k,
                        &full[slot], col * 64, row, at.hk, page);
          ++issued;
          if (++slot == SLOTS) {
            slot = 0;
            parity ^= 1;
          }
        }
        page = next;
      }
      u += run;
      off = 0;
      if (u < u1) at.next();
    }
    if (!ok) {  // do not leave while copies into this block's memory are in flight
      for (int i = max(0, issued - SLOTS); i < issued; ++i) {
        const long long t0 = clock64();
        while (!mbar_try_wait(&full[i % SLOTS], (i / SLOTS) & 1) && clock64() - t0 < kSpinLimitCycles) {}
      }
    }
    return;
  }

  // ----------------------------------------------------------- attention --
  const int wm = warp / WK, wk = warp % WK;
  const int g = lane >> 2, t4 = lane & 3;
  float* stage = reinterpret_cast<float*>(smem + C::OFF_STAGE);
  float2* ml_s = reinterpret_cast<float2*>(smem + C::OFF_ML);
  const uint32_t slots_addr = smem_u32(smem);
  // ldmatrix row addresses of this lane within a tile. K: matrices (keys 0-7,
  // chunk c), (keys 0-7, c + 1), (keys 8-15, c), (keys 8-15, c + 1); V
  // (transposed): (keys 0-7, c), (keys 8-15, c), (keys 0-7, c + 1), (keys 8-15, c + 1).
  const int key_k = wk * KW + (lane & 7) + ((lane >> 4) << 3), chunk_k = (lane >> 3) & 1;
  const int key_v = wk * KW + (lane & 15), chunk_v = lane >> 4;
  int slot = 0;
  uint32_t parity = 0;
  bool wrote_meta = false;
  int which = 0;  // parity of the run
  bool ok = true;

  for (long long u = u0; u < u1 && ok;) {
    const int run = static_cast<int>(min(static_cast<long long>(at.n - off), u1 - u));
    const int row0 = at.rt * MR + wm * 16;
    const int ra = min(row0 + g, at.rows - 1), rb = min(row0 + g + 8, at.rows - 1);
    const int tok_a = ra / p.G, tok_b = rb / p.G;
    // Q rows (A operand), rows g and g + 8 of this warp
    uint32_t qf[DP / 16][4];
    {
      const T* qa = static_cast<const T*>(p.q) + (at.s.t0 + tok_a) * p.qs_t + (at.hk * p.G + ra - tok_a * p.G) * p.qs_h;
      const T* qb = static_cast<const T*>(p.q) + (at.s.t0 + tok_b) * p.qs_t + (at.hk * p.G + rb - tok_b * p.G) * p.qs_h;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        const int d = i * 16 + t4 * 2;
        qf[i][0] = d < p.D ? *reinterpret_cast<const uint32_t*>(qa + d) : 0u;
        qf[i][1] = d < p.D ? *reinterpret_cast<const uint32_t*>(qb + d) : 0u;
        qf[i][2] = d + 8 < p.D ? *reinterpret_cast<const uint32_t*>(qa + d + 8) : 0u;
        qf[i][3] = d + 8 < p.D ? *reinterpret_cast<const uint32_t*>(qb + d + 8) : 0u;
      }
    }
    const int hi_a = key_hi(p, at.s, tok_a), hi_b = key_hi(p, at.s, tok_b);
    const int lo_a = key_lo(p, at.s, tok_a), lo_b = key_lo(p, at.s, tok_b);
    // keys that all rows of the tile see
    const int all_lo = key_lo(p, at.s, (min(at.rows, at.rt * MR + MR) - 1) / p.G);
    const int all_hi = key_hi(p, at.s, at.rt * MR / p.G);
    float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    for (int i = 0; i < run; ++i) {
      const int key0 = (at.tile0 + off + i) * KT;
      // ---- S = Q K^T
      float s[KW / 8][4];
#pragma unroll
      for (int n = 0; n < KW / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], parity, p.err, abort_flag, kErrTimeoutSoftmax,
                                               p.wait_limit));
      if (!ok) break;
      {
        const uint32_t base = slots_addr + slot * C::SLOT;
        // fragments are loaded kAhead steps before the products that use them
        uint32_t kf[kAhead + 1][4];
        auto load = [&](int i) {
          const int ks = i / (KW / 16), key = key_k + i % (KW / 16) * 16, c = (ks & 3) * 2 + chunk_k;
          ldmatrix4(base + (ks >> 2) * (KT * 128) + key * 128 + ((c ^ (key & 7)) << 4), kf[i % (kAhead + 1)]);
        };
        constexpr int N = DP / 16 * (KW / 16);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(i);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (i + kAhead < N) load(i + kAhead);
          const int ks = i / (KW / 16), n = i % (KW / 16), f = i % (kAhead + 1);
          mma16816<T>(s[2 * n], qf[ks], kf[f][0], kf[f][1]);
          mma16816<T>(s[2 * n + 1], qf[ks], kf[f][2], kf[f][3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);
      if (++slot == SLOTS) {
        slot = 0;
        parity ^= 1;
      }
      // ---- softmax
      const bool masked = key0 + KT > all_hi || key0 < all_lo;
      if (masked) {
#pragma unroll
        for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int key = key0 + wk * KW + n * 8 + t4 * 2 + c;
            if (key < lo_a || key >= hi_a) s[n][c] = -INFINITY;
            if (key < lo_b || key >= hi_b) s[n][2 + c] = -INFINITY;
          }
        }
      }
      float mx_a = fmaxf(s[0][0], s[0][1]), mx_b = fmaxf(s[0][2], s[0][3]);
#pragma unroll
      for (int n = 1; n < KW / 8; ++n) {
        mx_a = fmax3(mx_a, s[n][0], s[n][1]);
        mx_b = fmax3(mx_b, s[n][2], s[n][3]);
      }
      // The running maximum moves only when a score passes it by 2^8 (P stays
      // below 2^8; P and the sums share the stale maximum, so the quotient is
      // exact): after a row's first tiles that is rare, and one vote rules it out.
      if (__any_sync(0xffffffffu, fmaf(mx_a, p.scale_log2, -kStaleMax) > m_a ||
                                      fmaf(mx_b, p.scale_log2, -kStaleMax) > m_b)) {
#pragma unroll
        for (int x = 1; x <= 2; x <<= 1) {
          mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, x));
          mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, x));
        }
        const float new_a = fmaxf(m_a, mx_a * p.scale_log2), new_b = fmaxf(m_b, mx_b * p.scale_log2);
        const float fa = part_weight(m_a, new_a), fb = part_weight(m_b, new_b);
        m_a = new_a;
        m_b = new_b;
        l_a *= fa;
        l_b *= fb;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          o[d][0] *= fa;
          o[d][1] *= fa;
          o[d][2] *= fb;
          o[d][3] *= fb;
        }
      }
      {
        const float sub_a = m_a == -INFINITY ? 0.f : -m_a, sub_b = m_b == -INFINITY ? 0.f : -m_b;
        const uint64_t sc2 = f2_pack(p.scale_log2, p.scale_log2);
        const uint64_t a2 = f2_pack(sub_a, sub_a), b2 = f2_pack(sub_b, sub_b);
        uint64_t la2 = f2_pack(l_a, 0.f), lb2 = f2_pack(l_b, 0.f);
#pragma unroll
        for (int n = 0; n < KW / 8; ++n) {
          f2_unpack(f2_fma(f2_pack(s[n][0], s[n][1]), sc2, a2), s[n][0], s[n][1]);
          f2_unpack(f2_fma(f2_pack(s[n][2], s[n][3]), sc2, b2), s[n][2], s[n][3]);
#pragma unroll
          for (int c = 0; c < 4; ++c) s[n][c] = fast_exp2(s[n][c]);
          la2 = f2_add(la2, f2_pack(s[n][0], s[n][1]));
          lb2 = f2_add(lb2, f2_pack(s[n][2], s[n][3]));
        }
        float x, y;
        f2_unpack(la2, x, y);
        l_a = x + y;
        f2_unpack(lb2, x, y);
        l_b = x + y;
      }
      // ---- O += P V
      ok = __all_sync(0xffffffffu, mbar_wait(&full[slot], parity, p.err, abort_flag, kErrTimeoutSoftmax,
                                               p.wait_limit));
      if (!ok) break;
      const uint32_t base = slots_addr + slot * C::SLOT;
      if (masked) {
        // A masked key has P = 0, but 0 * inf and 0 * NaN are NaN. Rows that no
        // row sees (stale memory, or not fetched) are cleared here, and values that
        // are not finite taken out: the rows that see them get them at the end.
        const int seen_lo = at.seen_lo - key0, seen_hi = at.seen_hi - key0;
        bool bad = false;
        for (int x = lane; x < KW * HALVES * 8; x += 32) {
          const int key = wk * KW + x / (HALVES * 8), c = x % (HALVES * 8);
          uint4* w = reinterpret_cast<uint4*>(smem + slot * C::SLOT + (c >> 3) * (KT * 128) + key * 128 + (c & 7) * 16);
          if (key < seen_lo || key >= seen_hi) {
            *w = make_uint4(0u, 0u, 0u, 0u);
          } else if (not_finite4<T>(*w)) {
            *w = finite_only4<T>(*w);
            bad = true;
          }
        }
        if (bad) special[which] = 1;
        fence_proxy_async_smem();
        __syncwarp();  // other lanes read what was cleared here
      }
      {
        uint32_t vf[kAhead + 1][4];
        auto load = [&](int i) {
          const int d = i % (DP / 16), key = key_v + i / (DP / 16) * 16, c = (d & 3) * 2 + chunk_v;
          ldmatrix4_trans(base + (d >> 2) * (KT * 128) + key * 128 + ((c ^ (key & 7)) << 4), vf[i % (kAhead + 1)]);
        };
        constexpr int N = KW / 16 * (DP / 16);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) load(i);
#pragma unroll
        for (int kb = 0; kb < KW / 16; ++kb) {
          uint32_t ph[4], pl[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float v0 = s[2 * kb + (x >> 1)][(x & 1) * 2], v1 = s[2 * kb + (x >> 1)][(x & 1) * 2 + 1];
            ph[x] = pack2<T>(v0, v1);
            if constexpr (C::kSplitP) {
              const float2 r = unpack2<T>(ph[x]);
              pl[x] = pack2<T>(v0 - r.x, v1 - r.y);
            }
          }
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) {
            const int i = kb * (DP / 16) + d, f = i % (kAhead + 1);
            if (i + kAhead < N) load(i + kAhead);
            mma16816<T>(o[2 * d], ph, vf[f][0], vf[f][1]);
            mma16816<T>(o[2 * d + 1], ph, vf[f][2], vf[f][3]);
            if constexpr (C::kSplitP) {
              mma16816<T>(o[2 * d], pl, vf[f][0], vf[f][1]);
              mma16816<T>(o[2 * d + 1], pl, vf[f][2], vf[f][3]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);
      if (++slot == SLOTS) {
        slot = 0;
        parity ^= 1;
      }
    }

    // ---- join the warps that took the same rows' keys, through shared memory;
    // rows leave as whole lines: the output, or a piece for the joining pass
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      l_a += __shfl_xor_sync(0xffffffffu, l_a, x);
      l_b += __shfl_xor_sync(0xffffffffu, l_b, x);
    }
    {
      float* own = stage + warp * 16 * C::STRIDE;
      uint64_t na = f2_pack(0.f, 0.f), nb = na;  // 0, NaN once a value is not finite
      const uint64_t zero = na;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        na = f2_fma(f2_pack(o[d][0], o[d][1]), zero, na);
        nb = f2_fma(f2_pack(o[d][2], o[d][3]), zero, nb);
        *reinterpret_cast<float2*>(own + g * C::STRIDE + d * 8 + t4 * 2) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(own + (g + 8) * C::STRIDE + d * 8 + t4 * 2) = make_float2(o[d][2], o[d][3]);
      }
      float n0, n1, n2, n3;
      f2_unpack(na, n0, n1);
      f2_unpack(nb, n2, n3);
      if ((n0 + n1 != 0.f && fabsf(l_a) < INFINITY) || (n2 + n3 != 0.f && fabsf(l_b) < INFINITY)) special[which] = 1;
      if (t4 == 0) {
        ml_s[warp * 16 + g] = make_float2(m_a, l_a);
        ml_s[warp * 16 + g + 8] = make_float2(m_b, l_b);
      }
    }
    // A warp whose wait ended without its tile comes here too, and the four leave
    // together: a barrier that one of them never reaches would hold the others for good.
    ok = compute_warps_all(ok);
    if (!ok) break;
    const bool redo = special[which] != 0;
    uint4* const marks = reinterpret_cast<uint4*>(smem + C::OFF_MARKS);
    if (redo) {
      const int r0 = warp * (MR / 4), rows = min(MR / 4, max(at.rows - at.rt * MR - r0, 0));
      uint32_t m[DP / 16] = {};
      mark_values<T, DP>(p, at.b, at.hk, at.s, at.rt * MR + r0, rows, (at.tile0 + off) * KT,
                         (at.tile0 + off + run) * KT, m, [&] { ++*alive; });
      if (lane < rows) {
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
          marks[(r0 + lane) * (DP / 64) + c] = make_uint4(m[4 * c], m[4 * c + 1], m[4 * c + 2], m[4 * c + 3]);
      }
      compute_warps_sync();
    }
    const bool begins = off == 0, ends = off + run == at.n;
    const bool whole = begins && ends;
    const long long slot_row = (2LL * blockIdx.x + (begins ? 1 : 0)) * MR;
    constexpr int ACROSS = DP / 4;  // threads of a row, four values each
    const int col = static_cast<int>(threadIdx.x) % ACROSS * 4;
#pragma unroll 1
    for (int r = static_cast<int>(threadIdx.x) / ACROSS; r < MR; r += 128 / ACROSS) {
      const int seq_row = at.rt * MR + r;
      if (seq_row >= at.rows) break;
      const float2* ml = ml_s + (r / 16) * WK * 16 + r % 16;
      float m = ml[0].x;
#pragma unroll
      for (int w = 1; w < WK; ++w) m = fmaxf(m, ml[w * 16].x);
      float l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float2 part = ml[w * 16];
        const float f = part_weight(part.x, m);
        const float4 x = *reinterpret_cast<const float4*>(stage + (((r / 16) * WK + w) * 16 + r % 16) * C::STRIDE + col);
        l = fmaf(part.y, f, l);
        v.x = fmaf(x.x, f, v.x);
        v.y = fmaf(x.y, f, v.y);
        v.z = fmaf(x.z, f, v.z);
        v.w = fmaf(x.w, f, v.w);
      }
      if (redo) {
        uint32_t m[DP / 16];
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) {
          const uint4 w = marks[r * (DP / 64) + c];
          m[4 * c] = w.x, m[4 * c + 1] = w.y, m[4 * c + 2] = w.z, m[4 * c + 3] = w.w;
        }
        v = make_float4(marked<DP>(v.x, m, col), marked<DP>(v.y, m, col + 1), marked<DP>(v.z, m, col + 2),
                        marked<DP>(v.w, m, col + 3));
      }
      if (whole) {
        const int tr = seq_row / p.G, h = at.hk * p.G + seq_row - tr * p.G;
        const long long t = at.s.t0 + tr;
        const float inv = inverse_sum(l);
        if (col < p.D)
          *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + t * p.os_t + h * p.os_h + col) =
              make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
        if (p.lse && col == 0) p.lse[t * p.Hq + h] = log_sum(m, l);
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot_row + r) * DP + col) = v;
        if (col == 0) p.part_ml[slot_row + r] = make_float2(m, l);
      }
    }
    compute_warps_sync();  // the stage is free again
    if (threadIdx.x == 0) special[which] = 0;  // (the run after next is the first to use it again)
    which ^= 1;
    if (begins && !ends) {  // only ever the run's last row tile
      wrote_meta = true;
      if (threadIdx.x == 0) {
        Entry e;
        e.pieces = static_cast<int>(divide(u + at.n - 1, per_block) - blockIdx.x) + 1;
        e.t0 = at.s.t0;
        e.hk = at.hk;
        e.row0 = at.rt * MR;
        e.rows = min(MR, at.rows - at.rt * MR);
        e.slot0 = 2 * blockIdx.x + 1;
        e.slot1 = 2 * (blockIdx.x + 1);
        e.step = 2;
        *meta = e;
      }
    }
    u += run;
    off = 0;
    if (u < u1) at.next();
  }
  if (!wrote_meta && threadIdx.x == 0) meta->pieces = 0;
}

}  // namespace paged
}  // namespace pkb200
