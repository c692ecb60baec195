// paged.cu - C ABI of the paged-cache operators (include/pkb200.h): rotary
// positions, the append of new keys and values, and attention over the cache.
// Host-side checks, launch shapes and the choice between kernels.
#include <cmath>

#include "internal.h"
#include "rotary.cuh"
#include "../../include/pkb200.h"

using namespace pkb200;

namespace {

cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }

int value_size(int dtype) {
  return dtype == PKB200_BF16 || dtype == PKB200_FP16 ? 2 : dtype == PKB200_FP32 ? 4 : 0;
}

// The largest unit of 1, 2, 4 or 8 values (at most 16 bytes) that divides every
// number in `counts` and whose size in bytes divides every address.
int unit_for(int size, const long long* counts, int nc, const void* const* ptrs, int np) {
  int p = 16 / size;
  for (; p > 1; p >>= 1) {
    bool ok = true;
    for (int i = 0; i < nc && ok; ++i) ok = counts[i] % p == 0;
    for (int i = 0; i < np && ok; ++i) ok = reinterpret_cast<uintptr_t>(ptrs[i]) % (p * size) == 0;
    if (ok) break;
  }
  return p;
}

rotary::RowShape row_shape(int D, int half, int interleaved, int p) {
  rotary::RowShape r;
  r.D = D;
  r.half = half;
  r.rot_items = half / p;
  r.items = r.rot_items + (D - 2 * half + 2 * p - 1) / (2 * p);
  r.interleaved = interleaved;
  return r;
}

// Heads that one thread visits: as many (up to 8) as still leave every SM
// about a thousand threads. The sines of a pair are computed once per thread.
int heads_per_thread(long long threads_per_head, int heads, int sms) {
  int n = 1;
  while (n < 8 && threads_per_head * ((heads + 2 * n - 1) / (2 * n)) >= 1024LL * sms) n *= 2;
  return n;
}

template <typename T>
void launch_rope(int p, dim3 grid, cudaStream_t s, const rotary::RopeParams& a) {
  if constexpr (sizeof(T) == 2) {
    if (p == 8) return rotary::rope_kernel<T, 8><<<grid, 256, 0, s>>>(a);
  }
  if (p == 4) rotary::rope_kernel<T, 4><<<grid, 256, 0, s>>>(a);
  else if (p == 2) rotary::rope_kernel<T, 2><<<grid, 256, 0, s>>>(a);
  else rotary::rope_kernel<T, 1><<<grid, 256, 0, s>>>(a);
}

template <typename T>
void launch_append(int p, dim3 grid, cudaStream_t s, const rotary::AppendParams& a) {
  if (p == 8) rotary::paged_append_kernel<T, 8><<<grid, 256, 0, s>>>(a);
  else if (p == 4) rotary::paged_append_kernel<T, 4><<<grid, 256, 0, s>>>(a);
  else if (p == 2) rotary::paged_append_kernel<T, 2><<<grid, 256, 0, s>>>(a);
  else rotary::paged_append_kernel<T, 1><<<grid, 256, 0, s>>>(a);
}

// What every paged entry point requires of the cache and the batch.
bool cache_ok(const pkb200_paged_cache* c) {
  return c && (c->dtype == PKB200_BF16 || c->dtype == PKB200_FP16) && c->num_pages >= 0 &&
         c->page_size > 0 && c->heads > 0 && c->dim > 0 && (c->num_pages == 0 || (c->k && c->v));
}
bool batch_ok(const pkb200_paged_batch* b) {
  return b && b->num_seqs >= 0 && b->num_tokens >= 0 && b->table_width >= 0 &&
         (b->num_seqs == 0 ||
          (b->cu_seqlens && b->seq_lens && (b->page_table || b->table_width == 0)));
}

}  // namespace

extern "C" {

int pkb200_rope(const void* x, void* y, int dtype, const long long* positions,
                long long positions_stride, const float* inv_freq, int rot_pairs, int B,
                long long tokens, int H, int D, const long long* x_strides,
                const long long* y_strides, float factor, int interleaved, int backward,
                void* stream) {
  const int size = value_size(dtype);
  if (!size || B < 0 || tokens < 0 || H < 0 || D < 0 || rot_pairs < 0 || 2LL * rot_pairs > D ||
      !std::isfinite(factor))
    return cudaErrorInvalidValue;
  if (B == 0 || tokens == 0 || H == 0 || D == 0) return cudaSuccess;
  if (!x || !y || !x_strides || !y_strides || (rot_pairs && (!positions || !inv_freq)) || B > 65535)
    return cudaErrorInvalidValue;
  int sms, *err;
  if (const int e = internal::device(&sms, &err)) return e;
  const long long counts[] = {rot_pairs,    D,            x_strides[0], x_strides[1],
                              x_strides[2], y_strides[0], y_strides[1], y_strides[2]};
  const void* ptrs[] = {x, y};
  const int p = unit_for(size, counts, 8, ptrs, 2);
  rotary::RopeParams a;
  a.x = x;
  a.y = y;
  a.positions = positions;
  a.pos_stride_b = positions_stride;
  a.inv_freq = inv_freq;
  a.xs_b = x_strides[0];
  a.xs_s = x_strides[1];
  a.xs_h = x_strides[2];
  a.ys_b = y_strides[0];
  a.ys_s = y_strides[1];
  a.ys_h = y_strides[2];
  a.S = tokens;
  a.H = H;
  a.row = row_shape(D, rot_pairs, interleaved, p);
  a.factor = factor;
  a.backward = backward;
  a.heads_per_thread = heads_per_thread(tokens * a.row.items * B, H, sms);
  const long long blocks = (tokens * a.row.items + 255) / 256;
  const int groups = (H + a.heads_per_thread - 1) / a.heads_per_thread;
  if (blocks > 0x7fffffffLL || groups > 65535) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), groups, B);
  if (dtype == PKB200_BF16) launch_rope<__nv_bfloat16>(p, grid, S(stream), a);
  else if (dtype == PKB200_FP16) launch_rope<__half>(p, grid, S(stream), a);
  else launch_rope<float>(p, grid, S(stream), a);
  internal::count_launch(internal::kOther);
  return cudaGetLastError();
}

int pkb200_paged_kv_append(const pkb200_paged_cache* cache, const pkb200_paged_batch* batch,
                           const void* k, const long long* k_strides, const void* v,
                           const long long* v_strides, const void* q, const long long* q_strides,
                           void* q_out, const long long* q_out_strides, int q_heads,
                           const float* inv_freq, int rot_pairs, float factor, int interleaved,
                           void* stream) {
  if (!cache_ok(cache) || !batch_ok(batch) || q_heads < 0 || rot_pairs < 0 ||
      2LL * rot_pairs > cache->dim || !std::isfinite(factor))
    return cudaErrorInvalidValue;
  if (batch->num_tokens == 0 || batch->num_seqs == 0) return cudaSuccess;
  if (!k || !v || !k_strides || !v_strides || (rot_pairs && !inv_freq) ||
      (q_heads && (!q || !q_out || !q_strides || !q_out_strides)))
    return cudaErrorInvalidValue;
  int sms, *err;
  if (const int e = internal::device(&sms, &err)) return e;
  static const long long kNoStrides[2] = {0, 0};
  if (!q_heads) q_strides = q_out_strides = kNoStrides;
  const long long counts[] = {rot_pairs,          cache->dim,         k_strides[0],
                              k_strides[1],       v_strides[0],       v_strides[1],
                              q_strides[0],       q_strides[1],       q_out_strides[0],
                              q_out_strides[1],   cache->k_stride[0], cache->k_stride[1],
                              cache->k_stride[2], cache->v_stride[0], cache->v_stride[1],
                              cache->v_stride[2]};
  const void* ptrs[] = {k, v, cache->k, cache->v, q_heads ? q : k, q_heads ? q_out : k};
  const int p = unit_for(2, counts, 16, ptrs, 6);
  rotary::AppendParams a;
  a.k = k;
  a.v = v;
  a.q = q;
  a.k_pages = cache->k;
  a.v_pages = cache->v;
  a.q_out = q_out;
  a.ks_t = k_strides[0];
  a.ks_h = k_strides[1];
  a.vs_t = v_strides[0];
  a.vs_h = v_strides[1];
  a.qs_t = q_strides[0];
  a.qs_h = q_strides[1];
  a.os_t = q_out_strides[0];
  a.os_h = q_out_strides[1];
  a.kp_p = cache->k_stride[0];
  a.kp_h = cache->k_stride[1];
  a.kp_r = cache->k_stride[2];
  a.vp_p = cache->v_stride[0];
  a.vp_h = cache->v_stride[1];
  a.vp_r = cache->v_stride[2];
  a.page_table = batch->page_table;
  a.table_stride = batch->table_stride;
  a.cu = batch->cu_seqlens;
  a.lens = batch->seq_lens;
  a.inv_freq = inv_freq;
  a.T = batch->num_tokens;
  a.B = batch->num_seqs;
  a.Hq = q_heads;
  a.Hkv = cache->heads;
  a.page_size = cache->page_size;
  a.num_pages = cache->num_pages;
  a.table_width = batch->table_width;
  a.row = row_shape(cache->dim, rot_pairs, interleaved, p);
  a.factor = factor;
  a.err = err;
  const long long per_head = static_cast<long long>(a.T) * a.row.items;
  a.heads_per_thread = heads_per_thread(per_head, q_heads + 2 * cache->heads, sms);
  a.q_groups = (q_heads + a.heads_per_thread - 1) / a.heads_per_thread;
  a.kv_groups = (cache->heads + a.heads_per_thread - 1) / a.heads_per_thread;
  const long long blocks = (per_head + 255) / 256;
  const long long groups = a.q_groups + 2LL * a.kv_groups;
  if (blocks > 0x7fffffffLL || groups > 65535) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups));
  if (cache->dtype == PKB200_BF16) launch_append<__nv_bfloat16>(p, grid, S(stream), a);
  else launch_append<__half>(p, grid, S(stream), a);
  internal::count_launch(internal::kOther);
  return cudaGetLastError();
}

}  // extern "C"
