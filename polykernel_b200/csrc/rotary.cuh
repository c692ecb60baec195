// rotary.cuh - rotary positions and the append of new tokens to a paged
// key/value cache, with the rotation applied on the way (sm_100a).
//
// The first 2 * half values of a head row form `half` pairs (a, b): values
// (i, half + i), or (2i, 2i + 1) in the interleaved layout. With the angle
// t = position * frequency_i a pair becomes
//   a' = factor * (a cos t - b sin t),  b' = factor * (b cos t + a sin t)
// and the gradient of that map is the same with -t. Values past 2 * half are
// copied. Arithmetic in fp32, one rounding at the end.
//
// Both kernels are bound by HBM (one read and one write per value). The angles
// are computed here, from 4 bytes of frequency per pair, instead of being read
// from a table; a thread keeps the cosines of its pairs for the head rows (up
// to four) that it moves. No thread waits for another (a block that formed the
// cosines for its tokens in shared memory took 49 us against 39 for the prompt
// below: its phases ran one after the other), and registers are kept to four to
// six blocks per SM, for the loads in flight that the bandwidth needs.
// Measured: 4 x 32 x 2048 x 128 bf16 rotated in 25.6 us (5.2 TB/s, 0.80 of the
// copy rate), 5003 x 24 x 96 fp32 in 18.5 us (5.0 TB/s); 15618 tokens of 16 ragged
// chunks, q and k rotated, appended in 70 us (5.5 TB/s); 16381 tokens of 16 heads of 64,
// only moved, in 30 us (4.5 TB/s: a warp's rows are the heads of few tokens, and go to
// places a page apart).
#pragma once

#include "paged_index.h"
#include "sm100.cuh"

namespace pkb200 {
namespace rotary {

// Two 16-bit values in a word.
template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) { return unpack_f16x2(w); }
template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }

// A unit is P values that move as one access of P * sizeof(T) bytes.
template <typename T, int P>
struct alignas(P * sizeof(T)) Unit {
  T v[P];
};

// A row of D values splits into items of two units. Items below `rot_items`
// hold P whole pairs (units i and i + half / P, or 2i and 2i + 1 when
// interleaved); the rest of the row follows as plain unit pairs.
struct RowShape {
  int D;
  int half;         // rotated pairs
  int rot_items;    // half / P
  int items;        // rot_items + ceil((D - 2 * half) / (2P))
  int interleaved;
};

template <int P>
__device__ __forceinline__ void item_offsets(const RowShape& s, int item, int& u0, int& u1,
                                             bool& two) {
  two = true;
  if (item < s.rot_items) {
    u0 = s.interleaved ? 2 * item * P : item * P;
    u1 = s.interleaved ? u0 + P : s.half + u0;
  } else {
    u0 = 2 * s.half + 2 * (item - s.rot_items) * P;
    u1 = u0 + P;
    two = u1 < s.D;
  }
}

// cos and sin of one item's pairs at `position`. The angle in turns is formed in
// 64 bits and reduced there: position * frequency has no fraction left in 32
// bits once it passes 2^24 radians, and only 8 bits of one at 2^16. For 16-bit
// values the reduced angle goes to the SFU, whose error on [-pi, pi], 2^-21.4,
// is far below their rounding (2^-8 and 2^-11); the accurate functions took
// more instructions than everything else together. Rounding the reduced part to 32
// bits (by at most 2^-26 of a turn, 2^-23.3 radians) is less than the sine's own error for
// 16-bit values, and moves fp32 ones by at most 2^-23.3 of their pair (5.5e-8 in all on
// normal data, where 32-bit products with cosines rounded from 64 bits have 3.9e-8).
template <typename T, int P>
__device__ __forceinline__ void angles(const float* __restrict__ inv_freq, long long position, float factor,
                                       bool backward, float (&c)[P], float (&s)[P]) {
  constexpr double kTurnsPerRadian = 0.15915494309189533577;  // 1 / (2 pi)
  constexpr double kRound = 6755399441055744.0;               // 1.5 * 2^52: adding it rounds to whole numbers
  constexpr float kTwoPi = 6.28318530717958648f;
  const double pos = static_cast<double>(position) * kTurnsPerRadian;
  const float sign = backward ? -factor : factor;
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const double turns = pos * static_cast<double>(__ldg(inv_freq + k));
    const float part = static_cast<float>(turns - ((turns + kRound) - kRound));  // in [-1/2, 1/2]
    float sn, cs;
    if constexpr (sizeof(T) == 2) {
      sn = __sinf(part * kTwoPi);
      cs = __cosf(part * kTwoPi);
    } else {
      sincospif(2.f * part, &sn, &cs);
    }
    c[k] = cs * factor;
    s[k] = sn * sign;
  }
}

__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
  const float a0 = a;
  a = a0 * c - b * s;
  b = b * c + a0 * s;
}

// Rotates the P pairs that units x and y hold.
template <typename T, int P>
__device__ __forceinline__ void turn(Unit<T, P>& x, Unit<T, P>& y, const float (&c)[P], const float (&s)[P],
                                     bool interleaved) {
  if constexpr (sizeof(T) == 4) {
    if (interleaved && P >= 2) {
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        turn_pair(x.v[2 * k], x.v[2 * k + 1], c[k], s[k]);
        turn_pair(y.v[2 * k], y.v[2 * k + 1], c[P / 2 + k], s[P / 2 + k]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) turn_pair(x.v[k], y.v[k], c[k], s[k]);
    }
  } else if constexpr (P == 1) {  // one value each, whatever the layout
    const uint32_t w = *reinterpret_cast<const uint16_t*>(&x) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&y)) << 16;
    float2 v = unpack<T>(w);
    turn_pair(v.x, v.y, c[0], s[0]);
    const uint32_t r = pack<T>(v.x, v.y);
    *reinterpret_cast<uint16_t*>(&x) = static_cast<uint16_t>(r);
    *reinterpret_cast<uint16_t*>(&y) = static_cast<uint16_t>(r >> 16);
  } else {
    uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
    uint32_t* yw = reinterpret_cast<uint32_t*>(&y);
    if (interleaved) {
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        float2 v = unpack<T>(xw[k]), w = unpack<T>(yw[k]);
        turn_pair(v.x, v.y, c[k], s[k]);
        turn_pair(w.x, w.y, c[P / 2 + k], s[P / 2 + k]);
        xw[k] = pack<T>(v.x, v.y);
        yw[k] = pack<T>(w.x, w.y);
      }
    } else {
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        float2 v = unpack<T>(xw[k]), w = unpack<T>(yw[k]);
        turn_pair(v.x, w.x, c[2 * k], s[2 * k]);
        turn_pair(v.y, w.y, c[2 * k + 1], s[2 * k + 1]);
        xw[k] = pack<T>(v.x, v.y);
        yw[k] = pack<T>(w.x, w.y);
      }
    }
  }
}

// A thread moves one item of the rows lane, lane + lanes, ... of a token's (at
// most `rows` of them). Threads are numbered by item first, then by token and
// lane in the order of the strides.
struct Share {
  int lanes, rows;
  int token_first;  // neighbours take the next token, not the next lane
};
constexpr int kRows = 4;    // most rows of a thread
// Rows whose loads a thread has under way at once, 64 bytes of 16-bit values or 128
// of fp32 ones (which leave the registers for it: 18.8 against 20.5 us for 5003
// tokens x 24 heads x 96).
template <typename T>
constexpr int kFlight = sizeof(T) == 4 ? 4 : 2;

struct Place {
  long long token;
  int lane, item;
};
__device__ __forceinline__ Place place_of(long long index, const RowShape& r, const Share& s, long long tokens) {
  Place p;
  long long rest;
  if (index <= 0x7fffffff) {  // 32-bit division where it will do
    const unsigned i = static_cast<unsigned>(index), items = r.items;
    rest = i / items;
    p.item = static_cast<int>(i - static_cast<unsigned>(rest) * items);
    const unsigned q = static_cast<unsigned>(rest), d = s.token_first ? static_cast<unsigned>(tokens) : s.lanes;
    const unsigned hi = q / d, lo = q - hi * d;
    p.token = s.token_first ? lo : hi;
    p.lane = s.token_first ? hi : lo;
    return p;
  }
  rest = index / r.items;
  p.item = static_cast<int>(index - rest * r.items);
  const long long d = s.token_first ? tokens : s.lanes, hi = rest / d, lo = rest - hi * d;
  p.token = s.token_first ? lo : hi;
  p.lane = static_cast<int>(s.token_first ? hi : lo);
  return p;
}

// Moves one item of a thread's rows. `source(i)` gives the i-th row, or null;
// `ready` looks up what `target(i)` (null: drop the row) and the cosines need,
// while the first rows are on their way.
template <typename T, int P, bool ROTATES, class Source, class Ready, class Target, class Turns>
__device__ __forceinline__ void move_rows(const RowShape& s, int item, int rows, Source source, Ready ready,
                                          Target target, Turns turns) {
  using U = Unit<T, P>;
  int u0, u1;
  bool two;
  item_offsets<P>(s, item, u0, u1, two);
  constexpr int N = kFlight<T>;
  U x[N], y[N];
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const T* src = i0 + i < rows ? source(i0 + i) : nullptr;
      if (src) {
        x[i] = *reinterpret_cast<const U*>(src + u0);
        if (two) y[i] = *reinterpret_cast<const U*>(src + u1);
      }
    }
  };
  load(0);
  float c[P], sn[P];
  if (!ready(c, sn)) return;
  for (int i0 = 0; i0 < rows; i0 += N) {
    if (i0) load(i0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      T* dst = i0 + i < rows ? target(i0 + i) : nullptr;
      if (dst) {
        if (ROTATES && turns(i0 + i)) turn<T, P>(x[i], y[i], c, sn, s.interleaved != 0);
        *reinterpret_cast<U*>(dst + u0) = x[i];
        if (two) *reinterpret_cast<U*>(dst + u1) = y[i];
      }
    }
  }
}

struct RopeParams {
  const void* x;
  void* y;
  const long long* positions;
  long long pos_stride_b;  // positions[b * pos_stride_b + s]
  const float* inv_freq;
  long long xs_b, xs_s, xs_h, ys_b, ys_s, ys_h;  // strides, in values
  long long S;
  int H;
  RowShape row;
  Share share;
  float factor;
  int backward;
};

// grid: x over the shares of one batch entry, y over the batch.
template <typename T, int P>
__global__ void __launch_bounds__(256, 4) rope_kernel(const RopeParams p) {
  const long long index = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (index >= p.S * p.share.lanes * p.row.items) return;
  const Place at = place_of(index, p.row, p.share, p.S);
  const long long b = blockIdx.y;
  const T* src = static_cast<const T*>(p.x) + b * p.xs_b + at.token * p.xs_s + at.lane * p.xs_h;
  T* dst = static_cast<T*>(p.y) + b * p.ys_b + at.token * p.ys_s + at.lane * p.ys_h;
  const bool rotated = at.item < p.row.rot_items;
  const int rows = min(p.share.rows, (p.H - at.lane + p.share.lanes - 1) / p.share.lanes);
  move_rows<T, P, true>(
      p.row, at.item, rows, [&](int i) { return src + i * p.share.lanes * p.xs_h; },
      [&](float(&c)[P], float(&s)[P]) {
        if (rotated)
          angles<T, P>(p.inv_freq + at.item * P, p.positions[b * p.pos_stride_b + at.token], p.factor,
                    p.backward != 0, c, s);
        return true;
      },
      [&](int i) { return dst + i * p.share.lanes * p.ys_h; }, [&](int) { return rotated; });
}

struct AppendParams {
  const void *k, *v, *q;
  void *k_pages, *v_pages, *q_out;
  long long ks_t, ks_h, vs_t, vs_h, qs_t, qs_h, os_t, os_h;  // token and head strides, in values
  long long kp_p, kp_h, kp_r, vp_p, vp_h, vp_r;              // page, head and row strides
  const int* page_table;
  long long table_stride;
  const int* cu;
  const int* lens;
  const float* inv_freq;
  int T, B, Hq, Hkv, page_size, num_pages, table_width;
  RowShape row;
  Share share;
  float factor;
  int* err;
};

// grid: x over the shares; the q, k and v heads of a token are numbered through.
template <typename T, int P, bool ROTATES>
__global__ void __launch_bounds__(256, ROTATES ? 5 : 6) paged_append_kernel(const AppendParams p) {
  const long long index = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (index >= static_cast<long long>(p.T) * p.share.lanes * p.row.items) return;
  const Place at = place_of(index, p.row, p.share, p.T);
  const long long token = at.token;
  const int all = p.Hq + 2 * p.Hkv;
  const int rows = min(p.share.rows, (all - at.lane + p.share.lanes - 1) / p.share.lanes);
  const bool rotated = ROTATES && at.item < p.row.rot_items;
  auto head = [&](int i) { return at.lane + i * p.share.lanes; };
  T *k_row = nullptr, *v_row = nullptr;  // this token's row of head 0 in the pools, null to drop it
  move_rows<T, P, ROTATES>(
      p.row, at.item, rows,
      [&](int i) {
        const int h = head(i);
        return h < p.Hq           ? static_cast<const T*>(p.q) + token * p.qs_t + h * p.qs_h
               : h < p.Hq + p.Hkv ? static_cast<const T*>(p.k) + token * p.ks_t + (h - p.Hq) * p.ks_h
                                  : static_cast<const T*>(p.v) + token * p.vs_t + (h - p.Hq - p.Hkv) * p.vs_h;
      },
      [&](float(&c)[P], float(&s)[P]) {
        int seq;
        long long position;
        const auto where =
            paged::place_token(p.cu, p.B, token, [&](int b) { return __ldg(p.lens + b); }, seq, position);
        if (where != paged::kPlaced) {  // rows of no sequence stay as they are
          if (where == paged::kMisplaced) atomicCAS(p.err, 0, kErrBadBatch);
          return false;
        }
        const unsigned at32 = static_cast<unsigned>(position);  // lengths have 31 bits
        const int slot = at32 / static_cast<unsigned>(p.page_size);
        const int row = at32 - slot * p.page_size;
        const int page = slot < p.table_width
                             ? paged::clip_page(__ldg(p.page_table + seq * p.table_stride + slot), p.num_pages)
                             : p.num_pages;
        if (page < p.num_pages) {
          k_row = static_cast<T*>(p.k_pages) + page * p.kp_p + row * p.kp_r;
          v_row = static_cast<T*>(p.v_pages) + page * p.vp_p + row * p.vp_r;
        } else {
          atomicCAS(p.err, 0, kErrBadBatch);
        }
        if (rotated) angles<T, P>(p.inv_freq + at.item * P, position, p.factor, false, c, s);
        return true;
      },
      [&](int i) -> T* {
        const int h = head(i);
        return h < p.Hq    ? static_cast<T*>(p.q_out) + token * p.os_t + h * p.os_h
               : !k_row    ? nullptr
               : h < p.Hq + p.Hkv ? k_row + (h - p.Hq) * p.kp_h
                                  : v_row + (h - p.Hq - p.Hkv) * p.vp_h;
      },
      [&](int i) { return rotated && head(i) < p.Hq + p.Hkv; });
}

}  // namespace rotary
}  // namespace pkb200
