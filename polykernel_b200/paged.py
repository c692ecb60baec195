"""Serving a ragged batch over a paged key/value cache: rotary positions, the
append of new tokens, and attention over the pages. Reached as `ops.rope`,
`ops.paged_kv_append`, ... next to `ops.qkv_projection`, `ops.kv_cache_update` and
`ops.attention_prefill`, which serve one length with a contiguous cache.

A ragged batch is described by three int32 CUDA tensors. The new tokens of
sequence b are rows cu_seqlens[b]..cu_seqlens[b + 1] of the packed tensors, and the
last of its seq_lens[b] tokens; token p of the sequence lives in row
p % page_size of page page_table[b, p // page_size] of the pools
[pages, heads, page_size, dim]. (Pools kept as [pages, page_size, heads, dim] are
passed as `.transpose(1, 2)`.) The lengths are only read on the device: nothing
here synchronises, and a captured graph follows the tensors' contents. Rows from
cu_seqlens[-1] on belong to no sequence and are left as they were.

Tensors are bf16 or fp16 (`rope`: also fp32), strided as they come out of a
fused projection, with a contiguous last axis.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import PagedBatch, PagedCache, check, lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_LL2, _LL3 = ctypes.c_longlong * 2, ctypes.c_longlong * 3


def _tensor(t, name, dtypes, dims, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dims, got shape {tuple(t.shape)}")
    return t


def _rows(t, name, dtype, device, shape):
    """A tensor [tokens, heads, dim] with a contiguous last axis."""
    _tensor(t, name, (dtype,), len(shape), device)
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return _last(t, name)


def _last(t, name):
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have a contiguous last axis")
    return t


def _call(device, f, *args):
    """f(*args, stream) on the tensors' device and its current stream."""
    if device.index == torch.cuda.current_device():
        return f(*args, torch.cuda.current_stream().cuda_stream)
    with torch.cuda.device(device):
        return f(*args, torch.cuda.current_stream().cuda_stream)


def rope_frequencies(rot_dim, base=10000.0, scaling=None, device="cuda"):
    """(inv_freq, factor) for `rope` and `paged_kv_append`: radians per position
    of each of the rot_dim / 2 pairs, base^(-2i / rot_dim), as an fp32 tensor, and
    the factor on cos and sin. `scaling` stretches them for contexts longer than
    the `original_length` of the training:

      {"type": "linear", "factor": s}: every frequency divided by s.
      {"type": "ntk", "factor": s}: base * s^(rot_dim / (rot_dim - 2)).
      {"type": "yarn", "factor": s, "original_length": L, "beta_fast": 32,
       "beta_slow": 1, "attention_factor": 0.1 ln s + 1}: pairs that turn more
       than beta_fast times within L are kept, those that turn less than
       beta_slow times are divided by s, with a linear ramp over the index
       between; cos and sin are scaled by attention_factor.
      {"type": "bands", "factor": s, "original_length": L, "low": a, "high": b}:
       pairs that turn more than b times within L are kept, fewer than a times
       divided by s, with a blend linear in the number of turns between.
    """
    if rot_dim < 0 or rot_dim % 2:
        raise ValueError("rot_dim must be even and not negative")
    if not base > 0:
        raise ValueError("base must be positive")
    half = rot_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    scaling = dict(scaling or {"type": None})
    kind, s = scaling.pop("type"), float(scaling.pop("factor", 1.0))
    if not (math.isfinite(s) and s > 0):
        raise ValueError("scaling factor must be positive")
    factor = 1.0
    if kind == "ntk":
        if rot_dim <= 2:
            raise ValueError("ntk scaling needs rot_dim above 2")
        base = base * s ** (rot_dim / (rot_dim - 2))
    f = base ** (-2.0 * i / max(rot_dim, 1))
    if kind == "linear":
        f = f / s
    elif kind == "yarn":
        length = scaling.pop("original_length")
        fast, slow = scaling.pop("beta_fast", 32.0), scaling.pop("beta_slow", 1.0)
        given = scaling.pop("attention_factor", None)
        factor = 0.1 * math.log(s) + 1.0 if given is None and s > 1 else 1.0 if given is None else given

        def index(turns):  # the (fractional) pair that turns this often within `length`
            return half * math.log(length / (2 * math.pi * turns)) / math.log(base)

        low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rot_dim - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f / s * ramp + f * (1 - ramp)
    elif kind == "bands":
        length, low, high = (scaling.pop(n) for n in ("original_length", "low", "high"))
        if not high > low:
            raise ValueError("bands need high above low")
        keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f / s * (1 - keep) + f * keep
    elif kind not in (None, "ntk"):
        raise ValueError(f"unknown scaling type {kind!r} (linear, ntk, yarn or bands)")
    if scaling:
        raise ValueError(f"unknown scaling entries {sorted(scaling)}")
    return f.float().to(device), float(factor)


def _frequencies(inv_freq, device, dim):
    _tensor(inv_freq, "inv_freq", (torch.float32,), 1, device)
    if not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous")
    if 2 * inv_freq.shape[0] > dim:
        raise ValueError(f"inv_freq has {inv_freq.shape[0]} pairs for a head of {dim} values")
    return inv_freq


def _rope(x, positions, inv_freq, interleaved, factor, out, backward):
    if not isinstance(x, torch.Tensor) or x.dim() not in (3, 4):
        raise ValueError("x must be a tensor [T, H, D] or [B, H, S, D]")
    _last(_tensor(x, "x", tuple(_DTYPES), x.dim()), "x")
    dev = x.device
    packed = x.dim() == 3
    B, S, H, D = (1, *x.shape) if packed else (x.shape[0], x.shape[2], x.shape[1], x.shape[3])
    _frequencies(inv_freq, dev, D)
    if not isinstance(positions, torch.Tensor) or positions.dim() not in (1, 2):
        raise ValueError("positions must be a tensor of one position per token")
    _last(_tensor(positions, "positions", (torch.int64,), positions.dim(), dev), "positions")
    if positions.shape[-1] != S or (positions.dim() == 2 and (packed or positions.shape[0] != B)):
        raise ValueError(f"positions {tuple(positions.shape)} do not match x {tuple(x.shape)}")
    if not math.isfinite(factor):
        raise ValueError("factor must be finite")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        _rows(out, "out", x.dtype, dev, x.shape)
        if out.data_ptr() == x.data_ptr() and out.stride() != x.stride():
            raise ValueError("out may be x itself, not another view of its memory")

    def strides(t):
        return _LL3(0, t.stride(0), t.stride(1)) if packed else _LL3(t.stride(0), t.stride(2), t.stride(1))

    check(_call(dev, lib().pkb200_rope, x.data_ptr(), out.data_ptr(), _DTYPES[x.dtype],
                positions.data_ptr(), positions.stride(0) if positions.dim() == 2 else 0,
                inv_freq.data_ptr(), inv_freq.shape[0], B, S, H, D, strides(x), strides(out),
                float(factor), int(bool(interleaved)), int(backward)), "rope")
    return out


def rope(x, positions, inv_freq, interleaved=False, factor=1.0, out=None):
    """Rotary positions. x is [T, H, D] (packed tokens) or [B, H, S, D] (what
    `qkv_projection` returns); positions int64 [T], [S] or [B, S]. The first
    2 * len(inv_freq) values of a head are rotated in pairs (i, half + i), or
    (2i, 2i + 1) if interleaved, by position * inv_freq[i], and scaled by factor;
    the others are copied. Angles are exact for positions up to 2^31. `out` may
    be x."""
    return _rope(x, positions, inv_freq, interleaved, factor, out, False)


def rope_backward(grad, positions, inv_freq, interleaved=False, factor=1.0, out=None):
    """The gradient of `rope` with respect to x, from that of its result: the
    rotation by the negative angles (arguments as for `rope`)."""
    return _rope(grad, positions, inv_freq, interleaved, factor, out, True)


def _paged(k_pages, v_pages, page_table, cu_seqlens, seq_lens, num_tokens):
    """The C descriptions of the cache and the batch."""
    _tensor(k_pages, "k_pages", (torch.bfloat16, torch.float16), 4)
    dev = k_pages.device
    _tensor(v_pages, "v_pages", (k_pages.dtype,), 4, dev)
    if v_pages.shape != k_pages.shape:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} differ")
    _last(k_pages, "k_pages")
    _last(v_pages, "v_pages")
    i32 = (torch.int32,)
    _last(_tensor(page_table, "page_table", i32, 2, dev), "page_table")
    _tensor(cu_seqlens, "cu_seqlens", i32, 1, dev)
    _tensor(seq_lens, "seq_lens", i32, 1, dev)
    B, width = page_table.shape
    if cu_seqlens.shape[0] != B + 1 or seq_lens.shape[0] != B:
        raise ValueError(f"page_table has {B} sequences, cu_seqlens {cu_seqlens.shape[0] - 1}, "
                         f"seq_lens {seq_lens.shape[0]}")
    if not (cu_seqlens.is_contiguous() and seq_lens.is_contiguous()):
        raise ValueError("cu_seqlens and seq_lens must be contiguous")
    pages, heads, page, dim = k_pages.shape
    if heads == 0 or page == 0 or dim == 0:
        raise ValueError(f"k_pages must have heads, rows and values, got {tuple(k_pages.shape)}")
    cache = PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), _LL3(*k_pages.stride()[:3]),
                       _LL3(*v_pages.stride()[:3]), pages, heads, page, dim, _DTYPES[k_pages.dtype])
    batch = PagedBatch(page_table.data_ptr(), cu_seqlens.data_ptr(), seq_lens.data_ptr(),
                       page_table.stride(0), width, B, num_tokens)
    return dev, cache, batch


def _tokens(t, name):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"{name} must be a tensor [tokens, heads, dim]")
    return t.shape[0]


def paged_kv_append(k, v, k_pages, v_pages, page_table, cu_seqlens, seq_lens, inv_freq=None,
                    interleaved=False, factor=1.0, q=None, q_out=None):
    """Write the batch's new rows k, v [T, heads, dim] into the paged cache, in
    place. With `inv_freq` (see `rope_frequencies`) k is rotated on the way by the
    position that its token takes in its sequence, and so is q
    [T, q_heads, dim], whose rotation is returned (in `q_out`, which may be q; by
    default a new tensor, whose rows of no sequence are undefined).
    Two new tokens that share a cache row leave either's values there."""
    n = _tokens(k, "k")
    dev, cache, batch = _paged(k_pages, v_pages, page_table, cu_seqlens, seq_lens, n)
    dt, heads, dim = k_pages.dtype, cache.heads, cache.dim
    _rows(k, "k", dt, dev, (n, heads, dim))
    _rows(v, "v", dt, dev, (n, heads, dim))
    if inv_freq is None:
        if q is not None or q_out is not None:
            raise ValueError("q is only rotated: it needs inv_freq")
        freq, pairs = None, 0
    else:
        freq, pairs = _frequencies(inv_freq, dev, dim).data_ptr(), inv_freq.shape[0]
    if not math.isfinite(factor):
        raise ValueError("factor must be finite")
    q_args = (None, None, None, None, 0)
    if q is not None:
        hq = q.shape[1] if _tokens(q, "q") == n else -1
        if hq <= 0:
            raise ValueError(f"q must be [{n}, heads, {dim}], got {tuple(q.shape)}")
        _rows(q, "q", dt, dev, (n, hq, dim))
        if q_out is None:
            q_out = torch.empty(n, hq, dim, dtype=dt, device=dev)
        else:
            _rows(q_out, "q_out", dt, dev, q.shape)
            if q_out.data_ptr() == q.data_ptr() and q_out.stride() != q.stride():
                raise ValueError("q_out may be q itself, not another view of its memory")
        q_args = (q.data_ptr(), _LL2(*q.stride()[:2]), q_out.data_ptr(), _LL2(*q_out.stride()[:2]), hq)
    elif q_out is not None:
        raise ValueError("q_out without q")
    check(_call(dev, lib().pkb200_paged_kv_append, ctypes.byref(cache), ctypes.byref(batch),
                k.data_ptr(), _LL2(*k.stride()[:2]), v.data_ptr(), _LL2(*v.stride()[:2]), *q_args,
                freq, pairs, float(factor), int(bool(interleaved))), "paged_kv_append")
    return q_out


def _aligned(t, name):
    """16-byte rows: what the copies of attention start on."""
    if t.data_ptr() % 16 or any(s % 8 for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
        raise ValueError(f"{name} must start on 16 bytes, with strides that are multiples of 8 values")
    return t


def _strides(t, make):
    """Strides without the last axis's; those of axes of one are never taken."""
    return make(*(s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)))


def paged_attention(q, k_pages, v_pages, page_table, cu_seqlens, seq_lens, max_q_len=None, causal=True,
                    window=None, scale=None, return_lse=False, out=None, lse=None, workspace=None):
    """Attention of the new tokens q [T, q_heads, dim] over the pages of their
    sequences (whose new keys are appended first: `paged_kv_append`). Query head h
    reads key head h // (q_heads / heads). With `causal` a token sees the keys up to
    its own position, with `window` the last `window` of those. A row that sees no
    key gives zeros (and -inf). Returns out, or (out, lse) with return_lse, the
    fp32 [T, q_heads] logarithms of the sums of exponentials; both can be passed in.
    Rows of no sequence keep what `out` and `lse` held.

    dim and the page size are multiples of 8, dim at most 256. max_q_len, the most
    new tokens of any sequence, selects kernels and changes no result: pass it for
    speed (by default 1 for as many tokens as sequences, T otherwise).
    `workspace`: a uint8 tensor to use instead of a new one, if it is large enough;
    calls that may overlap need their own."""
    n = _tokens(q, "q")
    dev, cache, batch = _paged(k_pages, v_pages, page_table, cu_seqlens, seq_lens, n)
    dim, hq = cache.dim, q.shape[1]
    _rows(q, "q", k_pages.dtype, dev, (n, hq, dim))
    if hq == 0 or hq % cache.heads:
        raise ValueError(f"{hq} query heads do not divide among {cache.heads} key heads")
    if dim % 8 or dim > 256:
        raise ValueError(f"dim must be a multiple of 8 up to 256, got {dim}")
    if cache.page_size % 8:
        raise ValueError(f"the page size must be a multiple of 8, got {cache.page_size}")
    if cache.num_pages == 0:
        raise ValueError("k_pages has no pages")
    if n * hq // cache.heads >= 2 ** 31 - 1:
        raise ValueError("too many tokens for one call")
    if window is not None and (window < 1 or not causal):
        raise ValueError("window must be at least 1, and needs causal")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    if max_q_len is None:
        max_q_len = 1 if n <= batch.num_seqs else n
    elif max_q_len < 0:
        raise ValueError("max_q_len must not be negative")
    for t, name in ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages")):
        _aligned(t, name)
    if out is None:
        out = torch.empty(n, hq, dim, dtype=q.dtype, device=dev)
    else:
        _aligned(_rows(out, "out", q.dtype, dev, (n, hq, dim)), "out")
    if lse is not None:
        _tensor(lse, "lse", (torch.float32,), 2, dev)
        if lse.shape != (n, hq) or not lse.is_contiguous():
            raise ValueError(f"lse must be contiguous, of shape {(n, hq)}")
    elif return_lse:
        lse = torch.empty(n, hq, dtype=torch.float32, device=dev)
    cache.k_stride, cache.v_stride = _strides(k_pages, _LL3), _strides(v_pages, _LL3)
    window = min(window or 0, 2 ** 30)
    max_q_len = min(max_q_len, n)

    def go(stream):
        nonlocal workspace
        c, b = ctypes.byref(cache), ctypes.byref(batch)
        need = lib().pkb200_paged_attention_workspace_size(c, b, hq, max_q_len, window)
        if workspace is None or workspace.numel() < need:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        return lib().pkb200_paged_attention(
            c, b, q.data_ptr(), _strides(q, _LL2), out.data_ptr(), _strides(out, _LL2),
            None if lse is None else lse.data_ptr(), hq, max_q_len, int(bool(causal)), window, scale,
            workspace.data_ptr(), workspace.numel(), stream)

    check(_call(dev, go), "paged_attention")
    return (out, lse) if return_lse else out
