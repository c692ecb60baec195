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
// are therefore computed here, from 4 bytes of frequency per pair, instead of
// being read from a table; one thread keeps the cosines of its pairs for all
// the heads that it visits.
#pragma once

#include "paged_index.h"
#include "sm100.cuh"

namespace pkb200 {
namespace rotary {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }

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

// cos and sin of one item's pairs at `position`. The angle in turns is formed
// in 64 bits and reduced there: position * frequency has no fraction left in
// 32 bits once it passes 2^24 radians, and only 8 bits of one at 2^16.
template <int P>
__device__ __forceinline__ void angles(const float* __restrict__ inv_freq, int item, long long position,
                                       float factor, bool backward, float (&c)[P], float (&s)[P]) {
  constexpr double kTurnsPerRadian = 0.15915494309189533577;  // 1 / (2 pi)
  const double pos = static_cast<double>(position);
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const double turns = pos * (static_cast<double>(__ldg(inv_freq + item * P + k)) * kTurnsPerRadian);
    const float part = static_cast<float>(turns - rint(turns));  // in [-1/2, 1/2]
    float sn, cs;
    sincospif(2.f * part, &sn, &cs);
    c[k] = cs * factor;
    s[k] = (backward ? -sn : sn) * factor;
  }
}

template <typename T, int P>
__device__ __forceinline__ void turn(Unit<T, P>& x, Unit<T, P>& y, const float (&c)[P],
                                     const float (&s)[P], bool interleaved) {
  if (interleaved) {
    if constexpr (P >= 2) {
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        const float a = to_f32(x.v[2 * k]), b = to_f32(x.v[2 * k + 1]);
        x.v[2 * k] = from_f32<T>(a * c[k] - b * s[k]);
        x.v[2 * k + 1] = from_f32<T>(b * c[k] + a * s[k]);
        const float e = to_f32(y.v[2 * k]), f = to_f32(y.v[2 * k + 1]);
        y.v[2 * k] = from_f32<T>(e * c[P / 2 + k] - f * s[P / 2 + k]);
        y.v[2 * k + 1] = from_f32<T>(f * c[P / 2 + k] + e * s[P / 2 + k]);
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const float a = to_f32(x.v[k]), b = to_f32(y.v[k]);
    x.v[k] = from_f32<T>(a * c[k] - b * s[k]);
    y.v[k] = from_f32<T>(b * c[k] + a * s[k]);
  }
}

// Head rows that one thread has in flight: it issues their loads together.
constexpr int kFlight = 4;

// Moves one item of `heads` rows from src to dst (rotated when asked).
template <typename T, int P>
__device__ __forceinline__ void move_rows(const T* src, long long src_stride, T* dst,
                                          long long dst_stride, int heads, int u0, int u1, bool two,
                                          bool rotate, bool interleaved, const float (&c)[P],
                                          const float (&s)[P]) {
  using U = Unit<T, P>;
  for (int h0 = 0; h0 < heads; h0 += kFlight) {
    U x[kFlight], y[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      if (h0 + i < heads) {
        const T* row = src + (h0 + i) * src_stride;
        x[i] = *reinterpret_cast<const U*>(row + u0);
        if (two) y[i] = *reinterpret_cast<const U*>(row + u1);
      }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      if (h0 + i < heads) {
        if (rotate) turn<T, P>(x[i], y[i], c, s, interleaved);
        T* row = dst + (h0 + i) * dst_stride;
        *reinterpret_cast<U*>(row + u0) = x[i];
        if (two) *reinterpret_cast<U*>(row + u1) = y[i];
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
  int H, heads_per_thread;
  RowShape row;
  float factor;
  int backward;
};

// grid: x over (token, item), y over groups of heads, z over the batch.
template <typename T, int P>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long token = i / p.row.items;
  if (token >= p.S) return;
  const int item = static_cast<int>(i - token * p.row.items);
  const int h0 = blockIdx.y * p.heads_per_thread;
  const int heads = min(p.heads_per_thread, p.H - h0);
  int u0, u1;
  bool two;
  item_offsets<P>(p.row, item, u0, u1, two);
  const bool rotate = item < p.row.rot_items;
  float c[P], s[P];
  if (rotate)
    angles<P>(p.inv_freq, item, p.positions[blockIdx.z * p.pos_stride_b + token], p.factor,
              p.backward != 0, c, s);
  const long long b = blockIdx.z;
  move_rows<T, P>(static_cast<const T*>(p.x) + b * p.xs_b + token * p.xs_s + h0 * p.xs_h, p.xs_h,
                  static_cast<T*>(p.y) + b * p.ys_b + token * p.ys_s + h0 * p.ys_h, p.ys_h, heads, u0,
                  u1, two, rotate, p.row.interleaved != 0, c, s);
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
  int heads_per_thread, q_groups, kv_groups;  // y: q groups, then k groups, then v groups
  RowShape row;
  float factor;
  int* err;
};

// Sequences whose offsets one block keeps in shared memory for its lookups;
// a larger batch is searched in global memory.
constexpr int kAppendSeqs = 2048;

// grid: x over (token, item), y over groups of q, k and v heads.
template <typename T, int P>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendParams p) {
  __shared__ int cu_s[kAppendSeqs + 1];
  const bool shared = p.B <= kAppendSeqs;
  if (shared) {
    for (int i = threadIdx.x; i <= p.B; i += blockDim.x) cu_s[i] = __ldg(p.cu + i);
    __syncthreads();
  }
  const int* cu = shared ? cu_s : p.cu;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long token = i / p.row.items;
  if (token >= p.T) return;
  const int item = static_cast<int>(i - token * p.row.items);
  int seq;
  long long position;
  const auto place = paged::place_token(cu, p.B, token, [&](int b) { return __ldg(p.lens + b); }, seq, position);
  if (place != paged::kPlaced) {  // rows of no sequence stay as they are
    if (place == paged::kMisplaced && item == 0) atomicCAS(p.err, 0, kErrBadBatch);
    return;
  }
  int u0, u1;
  bool two;
  item_offsets<P>(p.row, item, u0, u1, two);
  const int group = blockIdx.y;
  const bool is_q = group < p.q_groups;
  const bool is_v = group >= p.q_groups + p.kv_groups;
  const bool rotate = !is_v && item < p.row.rot_items;
  float c[P], s[P];
  if (rotate) angles<P>(p.inv_freq, item, position, p.factor, false, c, s);
  const bool il = p.row.interleaved != 0;
  if (is_q) {
    const int h0 = group * p.heads_per_thread;
    move_rows<T, P>(static_cast<const T*>(p.q) + token * p.qs_t + h0 * p.qs_h, p.qs_h,
                    static_cast<T*>(p.q_out) + token * p.os_t + h0 * p.os_h, p.os_h,
                    min(p.heads_per_thread, p.Hq - h0), u0, u1, two, rotate, il, c, s);
    return;
  }
  const long long slot = position / p.page_size;
  const int page =
      slot < p.table_width ? paged::clip_page(__ldg(p.page_table + seq * p.table_stride + slot), p.num_pages)
                           : p.num_pages;
  if (page == p.num_pages) {
    if (item == 0) atomicCAS(p.err, 0, kErrBadBatch);
    return;
  }
  const int row = static_cast<int>(position - slot * p.page_size);
  const int h0 = (group - p.q_groups - (is_v ? p.kv_groups : 0)) * p.heads_per_thread;
  const int heads = min(p.heads_per_thread, p.Hkv - h0);
  if (is_v)
    move_rows<T, P>(static_cast<const T*>(p.v) + token * p.vs_t + h0 * p.vs_h, p.vs_h,
                    static_cast<T*>(p.v_pages) + page * p.vp_p + row * p.vp_r + h0 * p.vp_h, p.vp_h,
                    heads, u0, u1, two, false, il, c, s);
  else
    move_rows<T, P>(static_cast<const T*>(p.k) + token * p.ks_t + h0 * p.ks_h, p.ks_h,
                    static_cast<T*>(p.k_pages) + page * p.kp_p + row * p.kp_r + h0 * p.kp_h, p.kp_h,
                    heads, u0, u1, two, rotate, il, c, s);
}

}  // namespace rotary
}  // namespace pkb200
