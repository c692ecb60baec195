// paged.cu - C ABI of the paged-cache operators (include/pkb200.h): rotary
// positions, the append of new keys and values, and attention over the cache.
// Host-side checks, launch shapes and the choice between kernels.
#include <atomic>
#include <cmath>

#include "internal.h"
#include "paged_rows.cuh"
#include "paged_tiles.cuh"
#include "rotary.cuh"
#include "../../include/pkb200.h"

using namespace pkb200;

namespace {

// pkb200_selftest_paged_limits
std::atomic<long long> g_wait_limit{kSpinLimitCycles}, g_hold_back{0};

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

// How many of a token's `heads` rows a thread takes: four, for which it forms the
// cosines once, unless that leaves the SMs without threads.
rotary::Share share_of(const rotary::RowShape& r, long long tokens, int heads, int sms, bool token_first) {
  rotary::Share s;
  s.rows = rotary::kRows;
  while (s.rows > 1 && tokens * r.items * ((heads + s.rows - 1) / s.rows) < 1024LL * sms) s.rows /= 2;
  s.lanes = (heads + s.rows - 1) / s.rows;
  s.token_first = token_first;
  return s;
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

template <typename T, bool ROTATES>
void launch_append(int p, dim3 grid, cudaStream_t s, const rotary::AppendParams& a) {
  if (p == 8) rotary::paged_append_kernel<T, 8, ROTATES><<<grid, 256, 0, s>>>(a);
  else if (p == 4) rotary::paged_append_kernel<T, 4, ROTATES><<<grid, 256, 0, s>>>(a);
  else if (p == 2) rotary::paged_append_kernel<T, 2, ROTATES><<<grid, 256, 0, s>>>(a);
  else rotary::paged_append_kernel<T, 1, ROTATES><<<grid, 256, 0, s>>>(a);
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

// ---------------------------------------------------------- attention plan --
// Which kernels a call of paged attention runs, decided from sizes that the host
// knows: lengths live on the device, so every kernel takes any lengths, and
// max_q_len only says which kernel is the faster one for them.
struct Plan {
  int dp = 0;         // head width of the kernels: 64, 128 or 256
  int rows_mr = 0;    // row tile of the rows kernel, 0: not launched
  int rows_max = 0;   // sequences that it takes: those of at most so many rows
  int rows_grid = 0;
  bool tiles = false;  // tile kernel, for the sequences above rows_max
  int tiles_n = 0, splits = 1;
  size_t rows_o = 0, rows_ml = 0, rows_meta = 0, tiles_o = 0, tiles_ml = 0, tiles_meta = 0, bytes = 0;
};

// Rows (new tokens x heads of a group) up to which the rows kernel takes a
// sequence when all are that short. With 128-wide heads the tile kernel is the
// faster one from 33 rows on (24 sequences of 8000 keys, 4 key heads, 48 rows:
// 113 against 127 us; 2 of 60000: 65 against 95), with 64-wide ones it is not
// (107 against 94 us at 8000 keys).
constexpr int kRowsMost = 64, kRowsMostWide = 32;
constexpr int kRowsMinUnits = 2, kTilesMinUnits = 4;

size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

Plan make_plan(const pkb200_paged_cache* c, const pkb200_paged_batch* b, int q_heads, int max_q_len,
               int window, int sms) {
  Plan pl;
  const int G = q_heads / c->heads;
  pl.dp = c->dim <= 64 ? 64 : c->dim <= 128 ? 128 : 256;
  const long long T = b->num_tokens, B = b->num_seqs;
  const long long most = max_q_len < T ? max_q_len : T;
  const long long rows = most * G;  // of the longest sequence
  const bool tiles_can = pl.dp <= 128 && G <= 128;
  const int few = pl.dp == 128 ? kRowsMostWide : kRowsMost;
  if (rows <= few || !tiles_can) {
    pl.rows_mr = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    pl.rows_max = 0x7fffffff;
  } else {
    pl.tiles = true;
    // Single tokens among the prompts go to the rows kernel, unless the sizes
    // say that there are none. (With G <= few the longest sequence has more rows
    // than rows_max, so that the tile kernel's bound on row tiles is at least one.)
    if (B > 1 && T < B * most && G <= few) {
      pl.rows_mr = G <= 16 ? 16 : G <= 32 ? 32 : 64;
      pl.rows_max = pl.rows_mr;
    }
  }
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at += up256(n);
    return o;
  };
  if (pl.rows_mr) {
    pl.rows_grid = sms * (pl.dp == 64 ? paged::RowsCfg<64, 16>::kBlocks : pl.dp == 128 ? paged::RowsCfg<128, 16>::kBlocks
                                                                        : paged::RowsCfg<256, 16>::kBlocks);
    const size_t slots = 2 * static_cast<size_t>(pl.rows_grid) + 2;
    pl.rows_o = take(slots * pl.rows_mr * pl.dp * 4);
    pl.rows_ml = take(slots * pl.rows_mr * 8);
    pl.rows_meta = take(static_cast<size_t>(pl.rows_grid) * sizeof(paged::Entry));
  }
  if (pl.tiles) {
    // Row tiles: every sequence of the tile kernel may end in one that is not full,
    // and has more rows than the rows kernel takes.
    const long long per = 2 * (128 / G);  // tokens of a row tile
    const long long least = pl.rows_mr ? pl.rows_max / G + 1 : 1, seqs = B < T / least ? B : T / least;
    const long long n = (T + seqs * (per - 1)) / per;
    const long long blocks = n * c->heads;
    // Split the keys where that fills the SMs better: time in key tiles of the
    // last block to finish, with 8 tiles' worth for a block's start and end.
    long long units = (static_cast<long long>(b->table_width) * c->page_size + 127) / 128;
    if (window > 0 && units > (window + per) / 128 + 2) units = (window + per) / 128 + 2;
    double best = 0;
    for (int s = 1; s <= 64; ++s) {
      if (s > 1 && (s * kTilesMinUnits > units || blocks * s > 8LL * sms)) break;
      const double cost = static_cast<double>((blocks * s + sms - 1) / sms) * (static_cast<double>(units) / s + 8);
      if (s == 1 || cost < 0.93 * best) {
        best = cost;
        pl.splits = s;
      }
    }
    pl.tiles_n = static_cast<int>(n);
    if (pl.splits > 1) {
      const size_t entries = static_cast<size_t>(blocks), slots = entries * pl.splits;
      pl.tiles_o = take(slots * 256 * pl.dp * 4);
      pl.tiles_ml = take(slots * 256 * 8);
      pl.tiles_meta = take(entries * sizeof(paged::Entry));
    }
  }
  pl.bytes = at;
  return pl;
}

bool attention_ok(const pkb200_paged_cache* c, const pkb200_paged_batch* b, int q_heads, int max_q_len) {
  return cache_ok(c) && batch_ok(b) && q_heads > 0 && q_heads % c->heads == 0 && max_q_len >= 0 &&
         c->dim % 8 == 0 && c->dim <= 256 && c->page_size % 8 == 0 &&
         static_cast<long long>(b->num_tokens) * (q_heads / c->heads) < 0x7fffffffLL;
}

// Map of a pool [pages, heads, rows, dim] with boxes of 64 values x `box` rows.
bool pool_map(CUtensorMap* m, const pkb200_paged_cache* c, const void* base, const long long* st, int box) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c->dim), static_cast<cuuint64_t>(c->page_size),
                              static_cast<cuuint64_t>(c->heads), static_cast<cuuint64_t>(c->num_pages)};
  // the stride of an axis of one is never taken, but has to be a legal one
  const cuuint64_t row = static_cast<cuuint64_t>(c->dim) * 2;
  const cuuint64_t strides[3] = {c->page_size > 1 ? static_cast<cuuint64_t>(st[2]) * 2 : row,
                                 c->heads > 1 ? static_cast<cuuint64_t>(st[1]) * 2 : row,
                                 c->num_pages > 1 ? static_cast<cuuint64_t>(st[0]) * 2 : row};
  const cuuint32_t bx[4] = {64, static_cast<cuuint32_t>(box), 1, 1};
  return internal::tensor_map(m, c->dtype == PKB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              4, base, dims, strides, bx);
}

// The largest power of two that divides the page size, up to `most`.
int box_for(int page_size, int most) {
  int box = most;
  while (page_size % box) box >>= 1;
  return box;
}

// Launches the joining pass so that it may start while the attention kernel drains.
template <typename T, int DP>
int launch_join(const paged::AttnParams& a, int entries, int slot_rows, int block_rows, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(entries, slot_rows / block_rows);
  cfg.blockDim = dim3(paged::kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged::paged_join_kernel<T, DP>, a, slot_rows, block_rows);
  internal::count_launch(internal::kOther);
  return e;
}

template <typename T, int DP, int MR>
int launch_rows(const pkb200_paged_cache* c, paged::AttnParams a, const Plan& pl, char* ws, cudaStream_t s) {
  using C = paged::RowsCfg<DP, MR>;
  const auto kernel = paged::paged_rows_kernel<T, DP, MR>;
  if (const int e = internal::smem_attr(reinterpret_cast<const void*>(kernel), C::SMEM)) return e;
  CUtensorMap mk, mv;
  a.box = box_for(c->page_size, C::KT);
  if (!pool_map(&mk, c, c->k, c->k_stride, a.box) || !pool_map(&mv, c, c->v, c->v_stride, a.box))
    return cudaErrorInvalidValue;
  a.min_rows = 1;
  a.max_rows = pl.rows_max;
  a.min_units = kRowsMinUnits;
  a.part_o = reinterpret_cast<float*>(ws + pl.rows_o);
  a.part_ml = reinterpret_cast<float2*>(ws + pl.rows_ml);
  a.meta = reinterpret_cast<int*>(ws + pl.rows_meta);
  kernel<<<pl.rows_grid, C::kThreads, C::SMEM, s>>>(mk, mv, a);
  internal::count_launch(internal::kOther);
  if (const int e = cudaGetLastError()) return e;
  return launch_join<T, DP>(a, pl.rows_grid, MR, MR / 4, s);
}

template <typename T, int DP>
int launch_tiles(const pkb200_paged_cache* c, paged::AttnParams a, const Plan& pl, char* ws, cudaStream_t s) {
  using C = paged::TilesCfg<DP>;
  const auto kernel = paged::paged_tiles_kernel<T, DP>;
  if (const int e = internal::smem_attr(reinterpret_cast<const void*>(kernel), C::SMEM)) return e;
  CUtensorMap mq, mk, mv;
  a.box = box_for(c->page_size, C::KT);
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.Hq),
                              static_cast<cuuint64_t>(a.T)};
  const cuuint64_t row = static_cast<cuuint64_t>(a.D) * 2;
  const cuuint64_t strides[2] = {a.Hq > 1 ? static_cast<cuuint64_t>(a.qs_h) * 2 : row,
                                 a.T > 1 ? static_cast<cuuint64_t>(a.qs_t) * 2 : row};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(a.G), static_cast<cuuint32_t>(128 / a.G)};
  if (!internal::tensor_map(&mq, c->dtype == PKB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            3, a.q, dims, strides, box) ||
      !pool_map(&mk, c, c->k, c->k_stride, a.box) || !pool_map(&mv, c, c->v, c->v_stride, a.box))
    return cudaErrorInvalidValue;
  a.min_rows = pl.rows_mr ? pl.rows_max + 1 : 1;
  a.max_rows = 0x7fffffff;
  a.min_units = kTilesMinUnits;
  a.tiles = pl.tiles_n;
  a.splits = pl.splits;
  if (pl.splits > 1) {
    a.part_o = reinterpret_cast<float*>(ws + pl.tiles_o);
    a.part_ml = reinterpret_cast<float2*>(ws + pl.tiles_ml);
    a.meta = reinterpret_cast<int*>(ws + pl.tiles_meta);
  }
  const long long entries = static_cast<long long>(pl.tiles_n) * a.Hkv;
  if (entries * pl.splits > 0x7fffffffLL) return cudaErrorInvalidValue;
  kernel<<<static_cast<unsigned>(entries * pl.splits), C::kThreads, C::SMEM, s>>>(mq, mk, mv, a);
  internal::count_launch(internal::kAttnTensor);
  if (const int e = cudaGetLastError()) return e;
  return pl.splits > 1 ? launch_join<T, DP>(a, static_cast<int>(entries), 256, 16, s) : 0;
}

template <typename T, int DP>
int launch_attention(const pkb200_paged_cache* c, const paged::AttnParams& a, const Plan& pl, char* ws,
                     cudaStream_t s) {
  if (pl.rows_mr) {
    const int e = pl.rows_mr == 16   ? launch_rows<T, DP, 16>(c, a, pl, ws, s)
                  : pl.rows_mr == 32 ? launch_rows<T, DP, 32>(c, a, pl, ws, s)
                                     : launch_rows<T, DP, 64>(c, a, pl, ws, s);
    if (e) return e;
  }
  if constexpr (DP <= 128) {
    if (pl.tiles) return launch_tiles<T, DP>(c, a, pl, ws, s);
  }
  return 0;
}

template <typename T>
int launch_attention(const pkb200_paged_cache* c, const paged::AttnParams& a, const Plan& pl, char* ws,
                     cudaStream_t s) {
  return pl.dp == 64    ? launch_attention<T, 64>(c, a, pl, ws, s)
         : pl.dp == 128 ? launch_attention<T, 128>(c, a, pl, ws, s)
                        : launch_attention<T, 256>(c, a, pl, ws, s);
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
  a.share = share_of(a.row, tokens * B, H, sms, a.xs_s < a.xs_h);
  const long long blocks = (tokens * a.share.lanes * a.row.items + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks), B);
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
  a.share = share_of(a.row, a.T, q_heads + 2 * cache->heads, sms, false);
  const long long blocks = (static_cast<long long>(a.T) * a.share.lanes * a.row.items + 255) / 256;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  // without a rotation the values are only moved: one 16-bit type does for both
  if (rot_pairs == 0) launch_append<__half, false>(p, grid, S(stream), a);
  else if (cache->dtype == PKB200_BF16) launch_append<__nv_bfloat16, true>(p, grid, S(stream), a);
  else launch_append<__half, true>(p, grid, S(stream), a);
  internal::count_launch(internal::kOther);
  return cudaGetLastError();
}

size_t pkb200_paged_attention_workspace_size(const pkb200_paged_cache* cache,
                                             const pkb200_paged_batch* batch, int q_heads,
                                             int max_q_len, int window) {
  if (!attention_ok(cache, batch, q_heads, max_q_len) || batch->num_tokens == 0 || batch->num_seqs == 0)
    return 0;
  int sms, *err;
  if (internal::device(&sms, &err)) return 0;
  return make_plan(cache, batch, q_heads, max_q_len, window, sms).bytes;
}

int pkb200_paged_attention(const pkb200_paged_cache* cache, const pkb200_paged_batch* batch,
                           const void* q, const long long* q_strides, void* out,
                           const long long* out_strides, float* lse, int q_heads, int max_q_len,
                           int causal, int window, float scale, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (!attention_ok(cache, batch, q_heads, max_q_len) || window < 0 || (window && !causal) ||
      !(scale > 0.f) || !std::isfinite(scale))
    return cudaErrorInvalidValue;
  if (batch->num_tokens == 0 || batch->num_seqs == 0) return cudaSuccess;
  if (!q || !out || !q_strides || !out_strides || cache->num_pages == 0) return cudaErrorInvalidValue;
  for (const void* x : {static_cast<const void*>(cache->k), static_cast<const void*>(cache->v), q,
                        static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(x) & 15u) return cudaErrorInvalidValue;
  for (int i = 0; i < 3; ++i)
    if (cache->k_stride[i] % 8 || cache->v_stride[i] % 8) return cudaErrorInvalidValue;
  for (int i = 0; i < 2; ++i)
    if (q_strides[i] % 8 || out_strides[i] % 8) return cudaErrorInvalidValue;
  int sms, *err;
  if (const int e = internal::device(&sms, &err)) return e;
  const Plan pl = make_plan(cache, batch, q_heads, max_q_len, window, sms);
  if (workspace_bytes < pl.bytes || (pl.bytes && !workspace)) return cudaErrorInvalidValue;
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return cudaErrorInvalidValue;
  paged::AttnParams a = {};
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.k = cache->k;
  a.v = cache->v;
  a.qs_t = q_strides[0];
  a.qs_h = q_strides[1];
  a.os_t = out_strides[0];
  a.os_h = out_strides[1];
  a.kp_p = cache->k_stride[0];
  a.kp_h = cache->k_stride[1];
  a.kp_r = cache->k_stride[2];
  a.vp_p = cache->v_stride[0];
  a.vp_h = cache->v_stride[1];
  a.vp_r = cache->v_stride[2];
  a.table = batch->page_table;
  a.table_stride = batch->table_stride;
  a.cu = batch->cu_seqlens;
  a.lens = batch->seq_lens;
  a.B = batch->num_seqs;
  a.T = batch->num_tokens;
  a.Hq = q_heads;
  a.Hkv = cache->heads;
  a.G = q_heads / cache->heads;
  a.D = cache->dim;
  a.page_size = cache->page_size;
  a.num_pages = cache->num_pages;
  a.table_width = batch->table_width;
  a.causal = causal;
  a.window = window;
  a.scale_log2 = scale * 1.4426950408889634f;  // log2(e)
  a.err = err;
  a.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
  a.hold_back = g_hold_back.load(std::memory_order_relaxed);
  char* ws = static_cast<char*>(workspace);
  return cache->dtype == PKB200_BF16 ? launch_attention<__nv_bfloat16>(cache, a, pl, ws, S(stream))
                                     : launch_attention<__half>(cache, a, pl, ws, S(stream));
}

int pkb200_selftest_paged_limits(long long wait_limit, long long hold_back) {
  if (wait_limit < 0 || wait_limit > kSpinLimitCycles || hold_back < 0 || hold_back > kSpinLimitCycles)
    return cudaErrorInvalidValue;
  g_wait_limit = wait_limit ? wait_limit : kSpinLimitCycles;
  g_hold_back = hold_back;
  return cudaSuccess;
}

}  // extern "C"
