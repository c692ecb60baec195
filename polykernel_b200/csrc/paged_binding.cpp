// paged_binding.cpp - the Python side of the paged-cache operators
// (polykernel_b200/paged.py) over the C ABI of libpkb200.so. A decode step calls
// them once per layer with a few microseconds of GPU work each, so the argument
// checks, which took 15 to 30 us through ctypes, are made here.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>

#include "../../include/pkb200.h"
#include "overlap.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

template <typename... A>
[[noreturn]] void bad_value(const A&... a) { throw py::value_error(c10::str(a...)); }
template <typename... A>
[[noreturn]] void bad_type(const A&... a) { throw py::type_error(c10::str(a...)); }

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    case at::kByte: return "torch.uint8";
    default: return c10::toString(t);
  }
}

void check_device(const Tensor& t, const char* name, const at::Device* device) {
  if (!t.is_cuda()) bad_value(name, " must be a CUDA tensor");
  if (device && t.device() != *device) bad_value(name, " must be on ", *device, ", got ", t.device());
}
void check_type(const Tensor& t, const char* name, at::ScalarType type) {
  if (t.scalar_type() != type) bad_type(name, " must be ", type_name(type), ", got ", type_name(t.scalar_type()));
}
void check_dims(const Tensor& t, const char* name, int64_t dims) {
  if (t.dim() != dims) bad_value(name, " must have ", dims, " dims, got shape ", t.sizes());
}
void check_last(const Tensor& t, const char* name) {
  if (t.stride(-1) != 1 && t.size(-1) > 1) bad_value(name, " must have a contiguous last axis");
}
void check(const Tensor& t, const char* name, at::ScalarType type, int64_t dims, const at::Device* device) {
  check_device(t, name, device);
  check_type(t, name, type);
  check_dims(t, name, dims);
}
// [tokens, heads, dim] of one type, with a contiguous last axis.
void check_rows(const Tensor& t, const char* name, at::ScalarType type, const at::Device& device,
                at::IntArrayRef shape) {
  check(t, name, type, static_cast<int64_t>(shape.size()), &device);
  if (t.sizes() != shape) bad_value(name, " must have shape ", shape, ", got ", t.sizes());
  check_last(t, name);
}
pkb200::View view_of(const Tensor& t) {
  pkb200::View v{reinterpret_cast<std::uintptr_t>(t.data_ptr()), static_cast<int>(t.dim()), {}, {},
                 static_cast<long long>(t.element_size())};
  for (int i = 0; i < v.axes; ++i) {
    v.n[i] = t.size(i);
    v.stride[i] = t.stride(i) * v.size;
  }
  return v;
}
// What is written must not share memory with what is read or written beside it;
// `itself`: but may be the very same tensor.
void check_apart(const Tensor& out, const char* name, const Tensor& other, const char* other_name, bool itself = false) {
  const pkb200::View a = view_of(out), b = view_of(other);
  if (itself && a.same_places(b)) return;
  if (pkb200::share_memory(a, b)) bad_value(name, " overlaps ", other_name);
}
// Memory that is written must not be one place under several indexes.
void check_written(const Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) bad_value(name, " must not be an expanded tensor");
}
// 16-byte rows: what the copies of attention start on.
void check_aligned(const Tensor& t, const char* name) {
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % 8 == 0);
  if (!ok) bad_value(name, " must start on 16 bytes, with strides that are multiples of 8 values");
}
// A stride that is never taken may be anything.
long long stride_of(const Tensor& t, int64_t axis) { return t.size(axis) > 1 ? t.stride(axis) : 0; }

void check_status(int status, const char* what) {
  if (status) throw std::runtime_error(c10::str("pkb200: ", what, " failed with CUDA status ", status));
}
void* stream_of(const at::Device& d) { return at::cuda::getCurrentCUDAStream(d.index()).stream(); }

int type_code(const Tensor& t, const char* name, bool fp32) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return PKB200_BF16;
    case at::kHalf: return PKB200_FP16;
    case at::kFloat:
      if (fp32) return PKB200_FP32;
      [[fallthrough]];
    default:
      bad_type(name, " must be torch.bfloat16 or torch.float16", fp32 ? " or torch.float32" : "", ", got ",
               type_name(t.scalar_type()));
  }
}

const float* frequencies(const Tensor& f, const at::Device& device, int64_t dim) {
  check(f, "inv_freq", at::kFloat, 1, &device);
  if (!f.is_contiguous()) bad_value("inv_freq must be contiguous");
  if (2 * f.size(0) > dim) bad_value("inv_freq has ", f.size(0), " pairs for a head of ", dim, " values");
  return f.data_ptr<float>();
}

Tensor rope(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, bool interleaved, double factor,
            const OptTensor& out, bool backward) {
  if (x.dim() != 3 && x.dim() != 4) bad_value("x must be a tensor [T, H, D] or [B, H, S, D]");
  check_device(x, "x", nullptr);
  const int type = type_code(x, "x", true);
  check_last(x, "x");
  const at::Device dev = x.device();
  const bool packed = x.dim() == 3;
  const int64_t B = packed ? 1 : x.size(0), S = packed ? x.size(0) : x.size(2), H = x.size(1), D = x.size(-1);
  const float* freq = frequencies(inv_freq, dev, D);
  if (positions.dim() != 1 && positions.dim() != 2) bad_value("positions must be a tensor of one position per token");
  check(positions, "positions", at::kLong, positions.dim(), &dev);
  check_last(positions, "positions");
  if (positions.size(-1) != S || (positions.dim() == 2 && (packed || positions.size(0) != B)))
    bad_value("positions ", positions.sizes(), " do not match x ", x.sizes());
  if (!std::isfinite(factor)) bad_value("factor must be finite");
  Tensor y;
  if (out) {
    y = *out;
    check_rows(y, "out", x.scalar_type(), dev, x.sizes());
    check_apart(y, "out", x, "x", true);
    check_written(y, "out");
  } else {
    y = at::empty(x.sizes(), x.options());
  }
  auto strides = [&](const Tensor& t, long long (&s)[3]) {
    s[0] = packed ? 0 : t.stride(0);
    s[1] = packed ? t.stride(0) : t.stride(2);
    s[2] = t.stride(1);
  };
  long long xs[3], ys[3];
  strides(x, xs);
  strides(y, ys);
  if (B > 65535 || H > 0x7fffffff || D > 0x7fffffff) bad_value("x is too large: ", x.sizes());
  const c10::cuda::CUDAGuard guard(dev);
  check_status(pkb200_rope(x.data_ptr(), y.data_ptr(), type,
                           reinterpret_cast<const long long*>(positions.data_ptr<int64_t>()),
                           positions.dim() == 2 ? positions.stride(0) : 0, freq, static_cast<int>(inv_freq.size(0)),
                           static_cast<int>(B), S, static_cast<int>(H), static_cast<int>(D), xs, ys,
                           static_cast<float>(factor), interleaved, backward, stream_of(dev)),
               "rope");
  return y;
}

struct Paged {
  at::Device device{at::kCUDA};
  pkb200_paged_cache cache;
  pkb200_paged_batch batch;
};

Paged paged(const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table, const Tensor& cu_seqlens,
            const Tensor& seq_lens, int64_t tokens) {
  Paged p;
  check_device(k_pages, "k_pages", nullptr);
  p.cache.dtype = type_code(k_pages, "k_pages", false);
  check_dims(k_pages, "k_pages", 4);
  p.device = k_pages.device();
  check(v_pages, "v_pages", k_pages.scalar_type(), 4, &p.device);
  if (v_pages.sizes() != k_pages.sizes())
    bad_value("k_pages ", k_pages.sizes(), " and v_pages ", v_pages.sizes(), " differ");
  check_last(k_pages, "k_pages");
  check_last(v_pages, "v_pages");
  check(page_table, "page_table", at::kInt, 2, &p.device);
  check_last(page_table, "page_table");
  check(cu_seqlens, "cu_seqlens", at::kInt, 1, &p.device);
  check(seq_lens, "seq_lens", at::kInt, 1, &p.device);
  const int64_t B = page_table.size(0);
  if (cu_seqlens.size(0) != B + 1 || seq_lens.size(0) != B)
    bad_value("page_table has ", B, " sequences, cu_seqlens ", cu_seqlens.size(0) - 1, ", seq_lens ", seq_lens.size(0));
  if (!cu_seqlens.is_contiguous() || !seq_lens.is_contiguous())
    bad_value("cu_seqlens and seq_lens must be contiguous");
  for (int64_t i = 1; i < 4; ++i)
    if (k_pages.size(i) == 0) bad_value("k_pages must have heads, rows and values, got ", k_pages.sizes());
  for (int64_t i = 0; i < 4; ++i)
    if (k_pages.size(i) > 0x7fffffff) bad_value("k_pages is too large: ", k_pages.sizes());
  if (tokens > 0x7fffffff || B > 0x7ffffffe || page_table.size(1) > 0x7fffffff) bad_value("the batch is too large");
  p.cache.k = k_pages.data_ptr();
  p.cache.v = v_pages.data_ptr();
  for (int i = 0; i < 3; ++i) {
    p.cache.k_stride[i] = stride_of(k_pages, i);
    p.cache.v_stride[i] = stride_of(v_pages, i);
  }
  p.cache.num_pages = static_cast<int>(k_pages.size(0));
  p.cache.heads = static_cast<int>(k_pages.size(1));
  p.cache.page_size = static_cast<int>(k_pages.size(2));
  p.cache.dim = static_cast<int>(k_pages.size(3));
  p.batch.page_table = page_table.data_ptr<int>();
  p.batch.cu_seqlens = cu_seqlens.data_ptr<int>();
  p.batch.seq_lens = seq_lens.data_ptr<int>();
  p.batch.table_stride = stride_of(page_table, 0);
  p.batch.table_width = static_cast<int>(page_table.size(1));
  p.batch.num_seqs = static_cast<int>(B);
  p.batch.num_tokens = static_cast<int>(tokens);
  return p;
}

struct RowStrides {
  long long s[2];
  explicit RowStrides(const Tensor& t) : s{stride_of(t, 0), stride_of(t, 1)} {}
};

py::object paged_kv_append(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                           const Tensor& page_table, const Tensor& cu_seqlens, const Tensor& seq_lens,
                           const OptTensor& inv_freq, bool interleaved, double factor, const OptTensor& q,
                           const OptTensor& q_out) {
  check_dims(k, "k", 3);
  const int64_t n = k.size(0);
  const Paged p = paged(k_pages, v_pages, page_table, cu_seqlens, seq_lens, n);
  const at::ScalarType type = k_pages.scalar_type();
  const int64_t heads = p.cache.heads, dim = p.cache.dim;
  check_written(k_pages, "k_pages");
  check_written(v_pages, "v_pages");
  check_rows(k, "k", type, p.device, {n, heads, dim});
  check_rows(v, "v", type, p.device, {n, heads, dim});
  if (!inv_freq && (q || q_out)) bad_value("q is only rotated: it needs inv_freq");
  if (q_out && !q) bad_value("q_out without q");
  const float* freq = inv_freq ? frequencies(*inv_freq, p.device, dim) : nullptr;
  if (!std::isfinite(factor)) bad_value("factor must be finite");
  const c10::cuda::CUDAGuard guard(p.device);
  Tensor rotated;
  int64_t q_heads = 0;
  if (q) {
    check_dims(*q, "q", 3);
    q_heads = q->size(1);
    if (q->size(0) != n || q_heads == 0) bad_value("q must be [", n, ", heads, ", dim, "], got ", q->sizes());
    check_rows(*q, "q", type, p.device, {n, q_heads, dim});
    if (q_out) {
      rotated = *q_out;
      check_rows(rotated, "q_out", type, p.device, q->sizes());
      check_apart(rotated, "q_out", *q, "q", true);
      check_apart(rotated, "q_out", k, "k");
      check_apart(rotated, "q_out", v, "v");
      check_written(rotated, "q_out");
    } else {
      rotated = at::empty(q->sizes(), q->options());
    }
  }
  check_apart(v_pages, "v_pages", k_pages, "k_pages");
  for (const auto& [pool, name] : {std::pair<const Tensor&, const char*>{k_pages, "k_pages"}, {v_pages, "v_pages"}}) {
    check_apart(pool, name, k, "k");
    check_apart(pool, name, v, "v");
    if (q) check_apart(pool, name, *q, "q");
    if (q) check_apart(pool, name, rotated, "q_out");
  }
  const RowStrides ks(k), vs(v), qs(q ? *q : k), os(q ? rotated : k);
  check_status(pkb200_paged_kv_append(&p.cache, &p.batch, k.data_ptr(), ks.s, v.data_ptr(), vs.s,
                                      q ? q->data_ptr() : nullptr, qs.s, q ? rotated.data_ptr() : nullptr, os.s,
                                      static_cast<int>(q_heads), freq,
                                      inv_freq ? static_cast<int>(inv_freq->size(0)) : 0, static_cast<float>(factor),
                                      interleaved, stream_of(p.device)),
               "paged_kv_append");
  return q ? py::cast(rotated) : py::none();
}

py::object paged_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                           const Tensor& cu_seqlens, const Tensor& seq_lens, std::optional<int64_t> max_q_len,
                           bool causal, std::optional<int64_t> window, std::optional<double> scale_arg,
                           bool return_lse, const OptTensor& out_arg, const OptTensor& lse_arg,
                           const OptTensor& workspace_arg) {
  check_dims(q, "q", 3);
  const int64_t n = q.size(0), hq = q.size(1);
  const Paged p = paged(k_pages, v_pages, page_table, cu_seqlens, seq_lens, n);
  const int64_t heads = p.cache.heads, dim = p.cache.dim;
  check_rows(q, "q", k_pages.scalar_type(), p.device, {n, hq, dim});
  if (hq == 0 || hq % heads) bad_value(hq, " query heads do not divide among ", heads, " key heads");
  if (dim % 8 || dim > 256) bad_value("dim must be a multiple of 8 up to 256, got ", dim);
  if (p.cache.page_size % 8) bad_value("the page size must be a multiple of 8, got ", p.cache.page_size);
  if (p.cache.num_pages == 0) bad_value("k_pages has no pages");
  if (n * (hq / heads) >= 0x7fffffff) bad_value("too many tokens for one call");
  if (window && (*window < 1 || !causal)) bad_value("window must be at least 1, and needs causal");
  const double scale = scale_arg ? *scale_arg : 1.0 / std::sqrt(static_cast<double>(dim));
  if (!(scale > 0) || !std::isfinite(static_cast<float>(scale)) || !(static_cast<float>(scale) > 0))
    bad_value("scale must be positive and finite");
  if (max_q_len && *max_q_len < 0) bad_value("max_q_len must not be negative");
  const int64_t most = max_q_len ? std::min(*max_q_len, n) : n <= p.batch.num_seqs ? 1 : n;
  check_aligned(q, "q");
  check_aligned(k_pages, "k_pages");
  check_aligned(v_pages, "v_pages");
  const c10::cuda::CUDAGuard guard(p.device);
  Tensor out, lse;
  if (out_arg) {
    out = *out_arg;
    check_rows(out, "out", q.scalar_type(), p.device, q.sizes());
    check_aligned(out, "out");
    check_written(out, "out");
    check_apart(out, "out", q, "q", true);
    check_apart(out, "out", k_pages, "k_pages");
    check_apart(out, "out", v_pages, "v_pages");
  } else {
    out = at::empty(q.sizes(), q.options());
  }
  if (lse_arg) {
    lse = *lse_arg;
    check(lse, "lse", at::kFloat, 2, &p.device);
    if (lse.size(0) != n || lse.size(1) != hq || !lse.is_contiguous())
      bad_value("lse must be contiguous, of shape [", n, ", ", hq, "]");
  } else if (return_lse) {
    lse = at::empty({n, hq}, q.options().dtype(at::kFloat));
  }
  const int win = window ? static_cast<int>(std::min<int64_t>(*window, 0x7fffffff)) : 0;
  const int64_t need = static_cast<int64_t>(pkb200_paged_attention_workspace_size(
      &p.cache, &p.batch, static_cast<int>(hq), static_cast<int>(most), win));
  Tensor ws;
  if (workspace_arg) {
    check(*workspace_arg, "workspace", at::kByte, 1, &p.device);
    if (!workspace_arg->is_contiguous() || reinterpret_cast<uintptr_t>(workspace_arg->data_ptr()) % 256)
      bad_value("workspace must be contiguous and start on 256 bytes");
    if (workspace_arg->numel() >= need) ws = *workspace_arg;
  }
  if (!ws.defined() && need) ws = at::empty({need}, q.options().dtype(at::kByte));
  const RowStrides qs(q), os(out);
  check_status(pkb200_paged_attention(&p.cache, &p.batch, q.data_ptr(), qs.s, out.data_ptr(), os.s,
                                      lse.defined() ? lse.data_ptr<float>() : nullptr, static_cast<int>(hq),
                                      static_cast<int>(most), causal, win, static_cast<float>(scale),
                                      ws.defined() ? ws.data_ptr() : nullptr, static_cast<size_t>(need),
                                      stream_of(p.device)),
               "paged_attention");
  if (return_lse) return py::make_tuple(out, lse);
  return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_paged, m) {
  m.def("rope", &rope);
  m.def("paged_kv_append", &paged_kv_append);
  m.def("paged_attention", &paged_attention);
}
