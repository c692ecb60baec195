// paged_common.cuh - what the kernels of attention over a paged cache share:
// the batch description, its sequences' key ranges, and the final pass that
// joins the pieces of rows whose keys several blocks went over.
//
// For a new token at position p of a sequence of `len` tokens and a query head h
// of key head h / G:
//   o = sum_j softmax_j(scale * q . k_j) v_j  over the keys j that it sees:
//   j < len, j <= p if causal, j > p - window if a window is set.
// Rows of a sequence are numbered token * G + (head in the group), so one tile
// of rows shares its keys: the G heads of a few tokens.
//
// Statistics (running maximum, in log2 units, and sum) and the accumulated
// output are fp32 in every kernel. A row that sees no key gives zeros and a
// log-sum of -inf.
#pragma once

#include <type_traits>

#include "paged_index.h"
#include "sm100.cuh"

namespace pkb200 {
namespace paged {

struct AttnParams {
  const void* q;
  void* out;
  float* lse;  // [T, Hq], or null
  const void* k;
  const void* v;
  long long qs_t, qs_h, os_t, os_h;
  long long kp_p, kp_h, kp_r, vp_p, vp_h, vp_r;  // page, head and row strides of the pools
  const int* table;
  long long table_stride;
  const int* cu;
  const int* lens;
  int B, T, Hq, Hkv, G, D, page_size, num_pages, table_width;
  int causal, window;  // window 0: none
  float scale_log2;    // scale * log2(e)
  int box;             // keys of one TMA box: divides the page size and the key tile
  int min_rows, max_rows;  // this launch takes the sequences with that many rows
  int min_units;       // least key tiles of a piece of work
  int splits, tiles;   // tile kernel: pieces of a row tile's keys, bound on row tiles
  float* part_o;       // [slot][rows][DP] partial outputs, not divided by their sums
  float2* part_ml;     // [slot][rows] their maxima and sums
  int* meta;           // [entry][8], see Entry
  int* err;
  long long wait_limit;  // rows kernel: cycles after which a wait gives the block up
  long long hold_back;   // and cycles before its first copies (a self test's, else 0)
};

// A tile of rows whose pieces the joining pass adds up.
struct Entry {
  int pieces;  // 0: nothing to join
  int t0, hk, row0, rows;
  int slot0, slot1, step;  // piece k is in slot0, or slot1 + (k - 1) * step
};
static_assert(sizeof(Entry) == 32, "");

// Sequence b of the batch.
__device__ __forceinline__ Seq load_seq(const AttnParams& p, int b, bool report = false) {
  bool bad;
  const Seq s = clip_seq(__ldg(p.cu + b), __ldg(p.cu + b + 1), __ldg(p.lens + b), p.T,
                         static_cast<long long>(p.table_width) * p.page_size, bad);
  if (report && bad) atomicCAS(p.err, 0, kErrBadBatch);
  return s;
}
__device__ __forceinline__ int key_hi(const AttnParams& p, const Seq& s, int i) {
  return clip_hi(s, i, p.causal);
}
__device__ __forceinline__ int key_lo(const AttnParams& p, const Seq& s, int i) {
  return clip_lo(s, i, p.window);
}
template <int KT>
__device__ __forceinline__ int key_tiles(const AttnParams& p, const Seq& s, int first, int last,
                                         int& tile0) {
  return clip_tiles(s, first, last, p.causal, p.window, KT, tile0);
}

// The pool page that holds key `key` (below the sequence's length) of sequence
// b, or num_pages for a page outside the pool.
__device__ __forceinline__ int page_of(const AttnParams& p, int b, int key) {
  const int page = clip_page(__ldg(p.table + b * p.table_stride + key / p.page_size), p.num_pages);
  if (page == p.num_pages) atomicCAS(p.err, 0, kErrBadBatch);
  return page;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return unpack_bf16x2(v); }
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return unpack_f16x2(v); }

// Nonzero if one of the eight values in `w` is infinite or NaN (all exponent bits
// set): adding one at the lowest exponent bit then carries into the sign bit.
template <typename T>
__device__ __forceinline__ uint32_t not_finite4(const uint4& w) {
  constexpr bool half = std::is_same<T, __half>::value;
  constexpr uint32_t e = half ? 0x7c007c00u : 0x7f807f80u, one = half ? 0x04000400u : 0x00800080u;
  const uint32_t t = ((w.x & e) + one) | ((w.y & e) + one) | ((w.z & e) + one) | ((w.w & e) + one);
  return t & 0x80008000u;
}

// The same values with zeros in the place of those.
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
  return w & ~__vcmpeq2(w & e, e);
}
template <typename T>
__device__ __forceinline__ uint4 finite_only4(const uint4& w) {
  return make_uint4(finite_only<T>(w.x), finite_only<T>(w.y), finite_only<T>(w.z), finite_only<T>(w.w));
}

// mbar_wait for a role whose wait may last as long as others go over many keys
// again (mark_values): the limit runs anew while they count `alive` up.
__device__ __forceinline__ bool mbar_wait_alive(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag,
                                                int code, long long limit, const volatile int* alive) {
  if (mbar_try_wait(bar, parity)) return true;
  long long t0 = clock64();
  int seen = *alive;
  while (true) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > limit) {
      const int now = *alive;
      if (now == seen) {
        atomicCAS(err, 0, code);
        *abort_flag = 1;
        return false;
      }
      seen = now;
      t0 = clock64();
    }
  }
}

// --------------------------------------------- values that are not finite --
// A visible key's weight is positive, so a value of it that is infinite decides
// its column: inf of its sign, or NaN with one of the other sign, or if a value is
// NaN. Products formed from weights of 16 bits do not keep that: a weight may round
// to 0, or be split into a value and a remainder of the other sign, and 0 * inf and
// inf - inf are NaN. So where a finished row is not finite although its sum of
// exponentials is, or where values were taken out of a tile (finite_only), the kernels
// go over the values of its keys again (rare, and as fast as they can be read)
// and mark what decides its columns.
//
// A row's marks are 2 W words, W = DP / 32: column d is bit d / W of word d % W; the first
// W words are for inf, the others for -inf, NaN is both. (Lane i reads columns W i ... W i + W - 1.)
template <typename T, int DP>
__device__ __forceinline__ void load_values(const void* row, bool mine, uint32_t (&w)[DP / 64]) {
  const uint32_t* src = static_cast<const uint32_t*>(row) + lane_id() * (DP / 64);
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) w[c] = mine ? __ldg(src + c) : 0u;
}
template <typename T, int N>
__device__ __forceinline__ bool any_not_finite(const uint32_t (&w)[N]) {
  bool bad = false;
#pragma unroll
  for (int c = 0; c < N; ++c) bad |= finite_only<T>(w[c]) != w[c];
  return bad;
}

// One warp, for `rows` rows of a sequence from row0 on (at most 32), one per lane, and those
// of the keys [k0, k1) that they see; adds to their marks. One lane calls `alive` on the
// way, for those who wait.
template <typename T, int DP, class Alive>
__device__ __forceinline__ void mark_values(const AttnParams& p, int b, int hk, const Seq& s, int row0, int rows,
                                            int k0, int k1, uint32_t (&marks)[DP / 16], Alive alive) {
  constexpr int W = DP / 32, N = DP / 64;
  constexpr int ACROSS = DP / 8, KEYS = 32 / ACROSS;  // lanes of a row of 16 bytes each, and rows of a load
  if (rows <= 0) return;
  const int lane = lane_id();
  const int token = (row0 + min(lane, rows - 1)) / p.G;
  const int lo = key_lo(p, s, token), hi = key_hi(p, s, token);
  const int from = max(k0, __shfl_sync(0xffffffffu, lo, 0)), to = min(k1, __shfl_sync(0xffffffffu, hi, 31));
  const bool mine = lane * W < p.D;
  auto place = [&](const void* pool, long long sp, long long sh, long long sr, int page, int row) {
    return static_cast<const T*>(pool) + page * sp + hk * sh + row * sr;
  };
  auto page_at = [&](int key) {  // a page outside the pool has zeros, keys past the end are none of its
    return key < to ? clip_page(__ldg(p.table + b * p.table_stride + key / p.page_size), p.num_pages) : p.num_pages;
  };
  int page = page_at(from + lane);
  for (int j0 = from; j0 < to; j0 += 32) {
    const int row = (j0 + lane) % p.page_size, next = page_at(j0 + 32 + lane);
    uint32_t which = 0;  // keys with such values
#pragma unroll
    for (int i0 = 0; i0 < 32; i0 += 8 * KEYS) {
      uint4 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = (i0 + i * KEYS + lane / ACROSS) & 31;
        const int pg = __shfl_sync(0xffffffffu, page, key), r = __shfl_sync(0xffffffffu, row, key);
        const int d = lane % ACROSS * 8;
        v[i] = pg < p.num_pages && d < p.D
                   ? __ldg(reinterpret_cast<const uint4*>(place(p.v, p.vp_p, p.vp_h, p.vp_r, pg, r) + d))
                   : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (not_finite4<T>(v[i])) which |= 1u << ((i0 + i * KEYS + lane / ACROSS) & 31);
    }
    which = __reduce_or_sync(0xffffffffu, which);
    while (which) {
      const int i = __ffs(which) - 1, key = j0 + i;
      which &= which - 1;
      const int pg = __shfl_sync(0xffffffffu, page, i), r = __shfl_sync(0xffffffffu, row, i);
      uint32_t w[N], kw[N], up[W], down[W];
      load_values<T, DP>(place(p.v, p.vp_p, p.vp_h, p.vp_r, pg, r), mine, w);
      load_values<T, DP>(place(p.k, p.kp_p, p.kp_h, p.kp_r, pg, r), mine, kw);
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const float2 two = unpack2<T>(w[c / 2]);
        const float v = c % 2 ? two.y : two.x;
        up[c] = __ballot_sync(0xffffffffu, v != v || v == INFINITY);
        down[c] = __ballot_sync(0xffffffffu, v != v || v == -INFINITY);
      }
      // A key that is not finite scores inf or NaN, and the row's sum is NaN
      // whatever is marked, or -inf: its weight is 0 and the product with it NaN.
      const bool odd_key = __any_sync(0xffffffffu, any_not_finite<T>(kw));
      if (odd_key) {
#pragma unroll
        for (int c = 0; c < W; ++c) up[c] = down[c] = up[c] | down[c];
      }
      if (key >= lo && key < hi) {
#pragma unroll
        for (int c = 0; c < W; ++c) {
          marks[c] |= up[c];
          marks[W + c] |= down[c];
        }
      }
    }
    page = next;
    if (lane == 0) alive();
  }
}

// Column d of a row with those marks, o where it has none.
template <int DP>
__device__ __forceinline__ float marked(float o, const uint32_t (&marks)[DP / 16], int d) {
  constexpr int W = DP / 32;
  const bool up = marks[d % W] >> (d / W) & 1u, down = marks[W + d % W] >> (d / W) & 1u;
  return up ? (down ? NAN : INFINITY) : down ? -INFINITY : o;
}

constexpr float kStaleMax = 8.f;  // log2 units a row's maximum may lag behind

// Weight of a part whose maximum is m within a row whose maximum is top.
__device__ __forceinline__ float part_weight(float m, float top) {
  return m == top ? 1.f : fast_exp2(m - top);
}
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float m, float l) {
  constexpr float kLn2 = 0.69314718055994531f;
  return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Position of a sequence of work items in a batch: inclusive sum of `mine` over
// the block's threads before this one, and the block's total.
template <int THREADS>
__device__ __forceinline__ long long block_prefix(long long mine, long long* warp_sums,
                                                  long long& total) {
  const int lane = lane_id(), warp = warp_id();
  long long x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + x - mine;
}

// ------------------------------------------------------------------- join --
// Adds up the pieces of row tiles whose keys several blocks went over, `rows`
// rows per block. A row with few pieces is one warp's; with many, four warps
// share it, each taking every fourth piece. The order of the sums is fixed, so results do not depend on timing.
// Launched to overlap the attention kernel's tail (grid_dependency_wait).
constexpr int kJoinThreads = 512, kJoinFew = 8;

template <typename T, int DP>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const AttnParams p, int slot_rows,
                                                                  int block_rows) {
  constexpr int C = (DP + 127) / 128;  // float4 per lane
  __shared__ float4 o_s[3][4][32 * C];
  __shared__ float2 ml_s[3][4];
  grid_dependency_wait();
  const Entry e = reinterpret_cast<const Entry*>(p.meta)[blockIdx.x];
  const int first = static_cast<int>(blockIdx.y) * block_rows, end = min(first + block_rows, e.rows);
  if (e.pieces == 0 || first >= end) return;
  const int warp = warp_id(), lane = lane_id();
  float m, l;
  float4 o[C];
  auto add = [&](float mk, float lk, const float4 (&ok)[C]) {
    const float top = fmaxf(m, mk);
    const float a = part_weight(m, top), b = part_weight(mk, top);
    m = top;
    l = l * a + lk * b;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      o[c].x = o[c].x * a + ok[c].x * b;
      o[c].y = o[c].y * a + ok[c].y * b;
      o[c].z = o[c].z * a + ok[c].z * b;
      o[c].w = o[c].w * a + ok[c].w * b;
    }
  };
  auto gather = [&](int row, int from, int step) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = from; k < e.pieces; k += step) {
      const long long at = static_cast<long long>(k == 0 ? e.slot0 : e.slot1 + (k - 1) * e.step) * slot_rows + row;
      const float2 ml = p.part_ml[at];
      float4 ok[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int d = lane * 4 + c * 128;
        ok[c] = d < DP ? *reinterpret_cast<const float4*>(p.part_o + at * DP + d)
                       : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      add(ml.x, ml.y, ok);
    }
  };
  // The same for a row with infinities: a weight that is too small for 32 bits is
  // not 0, and keeps one.
  auto gather_special = [&](int row) {
    gather(row, 0, 1);
    const float top = m;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < e.pieces; ++k) {
      const long long at = static_cast<long long>(k == 0 ? e.slot0 : e.slot1 + (k - 1) * e.step) * slot_rows + row;
      const float w = part_weight(p.part_ml[at].x, top);
      auto part = [&](float& to, float x) { to += w != 0.f ? x * w : fabsf(x) < INFINITY ? 0.f : x; };
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const int d = lane * 4 + c * 128;
        if (d >= DP) continue;
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + at * DP + d);
        part(o[c].x, x.x);
        part(o[c].y, x.y);
        part(o[c].z, x.z);
        part(o[c].w, x.w);
      }
    }
  };
  auto store = [&](int row) {
    bool odd = false;
#pragma unroll
    for (int c = 0; c < C; ++c) odd |= !(fabsf(o[c].x) + fabsf(o[c].y) + fabsf(o[c].z) + fabsf(o[c].w) < INFINITY);
    if (__any_sync(0xffffffffu, odd) && fabsf(l) < INFINITY) gather_special(row);
    const int r = e.row0 + row, tr = r / p.G, h = e.hk * p.G + r - tr * p.G;
    const long long t = e.t0 + tr;
    const float inv = inverse_sum(l);
    T* dst = static_cast<T*>(p.out) + t * p.os_t + h * p.os_h;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int d = lane * 4 + c * 128;
      if (d < p.D)
        *reinterpret_cast<uint2*>(dst + d) =
            make_uint2(pack2<T>(o[c].x * inv, o[c].y * inv), pack2<T>(o[c].z * inv, o[c].w * inv));
    }
    if (p.lse && lane == 0) p.lse[t * p.Hq + h] = log_sum(m, l);
  };
  if (e.pieces <= kJoinFew) {
    for (int row = first + warp; row < end; row += kJoinThreads / 32) {
      gather(row, 0, 1);
      store(row);
    }
    return;
  }
  const int part = warp >> 2, mine = warp & 3;
  for (int row0 = first; row0 < end; row0 += 4) {
    const int row = row0 + mine;
    if (row < end) gather(row, part, 4);
    if (part > 0 && row < end) {
#pragma unroll
      for (int c = 0; c < C; ++c) o_s[part - 1][mine][c * 32 + lane] = o[c];
      if (lane == 0) ml_s[part - 1][mine] = make_float2(m, l);
    }
    __syncthreads();
    if (part == 0 && row < end) {
      for (int w = 0; w < 3; ++w) {
        float4 ok[C];
#pragma unroll
        for (int c = 0; c < C; ++c) ok[c] = o_s[w][mine][c * 32 + lane];
        const float2 ml = ml_s[w][mine];
        add(ml.x, ml.y, ok);
      }
      store(row);
    }
    __syncthreads();
  }
}

}  // namespace paged
}  // namespace pkb200
