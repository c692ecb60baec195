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
fused projection, with a contiguous last axis. `rope` is differentiable; through
a cache (`paged_kv_append`, `paged_attention`) no gradient flows.
"""
from __future__ import annotations

import importlib.machinery
import importlib.util
import math
import os
import sysconfig

import torch

from ._lib import LIB_PATH, lib

_module = None


def load_paged():
    """The compiled module (csrc/paged_binding.cpp), loaded once; raises if it is not built."""
    global _module
    if _module is None:
        lib()  # the library that it calls
        # (built per Python version: another one's module beside it is not this one's)
        path = os.path.join(os.path.dirname(LIB_PATH), "_paged" + sysconfig.get_config_var("EXT_SUFFIX"))
        if not os.path.exists(path):
            raise RuntimeError("pkb200: Python module of the paged operators not built; run "
                               "`python -c 'import __graft_entry__ as g; g.build()'`")
        loader = importlib.machinery.ExtensionFileLoader("_paged", path)
        spec = importlib.util.spec_from_file_location("_paged", path, loader=loader)
        module = importlib.util.module_from_spec(spec)
        loader.exec_module(module)
        _module = module
    return _module


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


class _Rope(torch.autograd.Function):
    """`rope` (or `rope_backward`) as a step of autograd. The map is linear, and
    each of the two is the other's gradient."""

    @staticmethod
    def forward(ctx, x, positions, inv_freq, interleaved, factor, backward):
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = interleaved, factor, backward
        return load_paged().rope(x, positions, inv_freq, interleaved, factor, None, backward)

    @staticmethod
    def backward(ctx, grad):
        interleaved, factor, backward = ctx.how
        if grad.stride(-1) != 1:  # a sum's gradient is expanded
            grad = grad.contiguous()
        return _Rope.apply(grad, *ctx.saved_tensors, interleaved, factor, not backward), None, None, None, None, None


def _rope(x, positions, inv_freq, interleaved, factor, out, backward):
    if torch.is_grad_enabled() and (getattr(x, "requires_grad", False) or getattr(inv_freq, "requires_grad", False)):
        if inv_freq.requires_grad:
            raise ValueError("inv_freq gets no gradient: pass inv_freq.detach()")
        if out is not None:
            raise ValueError("out is not taken for a tensor that requires a gradient")
        return _Rope.apply(x, positions, inv_freq, interleaved, factor, backward)
    return load_paged().rope(x, positions, inv_freq, interleaved, factor, out, backward)


def rope(x, positions, inv_freq, interleaved=False, factor=1.0, out=None):
    """Rotary positions. x is [T, H, D] (packed tokens) or [B, H, S, D] (what
    `qkv_projection` returns); positions int64 [T], [S] or [B, S]. The first
    2 * len(inv_freq) values of a head are rotated in pairs (i, half + i), or
    (2i, 2i + 1) if interleaved, by position * inv_freq[i], and scaled by factor;
    the others are copied. Angles are formed in 64 bits and are within
    2^-20 radians for |position * inv_freq| up to 2^31. `out` may be x, and otherwise shares no memory with it.
    Differentiable with respect to x (without `out`)."""
    return _rope(x, positions, inv_freq, interleaved, factor, out, False)


def rope_backward(grad, positions, inv_freq, interleaved=False, factor=1.0, out=None):
    """The gradient of `rope` with respect to x, from that of its result: the
    rotation by the negative angles (arguments as for `rope`)."""
    return _rope(grad, positions, inv_freq, interleaved, factor, out, True)


def paged_kv_append(k, v, k_pages, v_pages, page_table, cu_seqlens, seq_lens, inv_freq=None,
                    interleaved=False, factor=1.0, q=None, q_out=None):
    """Write the batch's new rows k, v [T, heads, dim] into the paged cache, in
    place. With `inv_freq` (see `rope_frequencies`) k is rotated on the way by the
    position that its token takes in its sequence, and so is q
    [T, q_heads, dim], whose rotation is returned (in `q_out`, which may be q; by
    default a new tensor, whose rows of no sequence are undefined).
    Two new tokens that share a cache row leave either's values there."""
    return load_paged().paged_kv_append(k, v, k_pages, v_pages, page_table, cu_seqlens, seq_lens, inv_freq,
                                  interleaved, factor, q, q_out)


def paged_attention(q, k_pages, v_pages, page_table, cu_seqlens, seq_lens, max_q_len=None, causal=True,
                    window=None, scale=None, return_lse=False, out=None, lse=None, workspace=None):
    """Attention of the new tokens q [T, q_heads, dim] over the pages of their
    sequences (whose new keys are appended first: `paged_kv_append`). Query head h
    reads key head h // (q_heads / heads). With `causal` a token sees the keys up to
    its own position, with `window` the last `window` of those. A row that sees no
    key gives zeros (and -inf). Returns out, or (out, lse) with return_lse, the
    fp32 [T, q_heads] logarithms of the sums of exponentials; both can be passed in
    (out may be q, and otherwise shares no memory with the inputs).
    Rows of no sequence keep what `out` and `lse` held.

    dim and the page size are multiples of 8, dim at most 256. max_q_len, the most
    new tokens of any sequence, selects kernels: pass it for speed (by default 1 for
    as many tokens as sequences, T otherwise). Any value is right for any batch, but
    the kernels round differently, so the last bits of a row depend on it and on the
    sizes of the batch. A call with the same arguments repeats itself.
    `workspace`: a uint8 tensor to use instead of a new one, if it is large enough;
    calls that may overlap need their own."""
    return load_paged().paged_attention(q, k_pages, v_pages, page_table, cu_seqlens, seq_lens, max_q_len, causal,
                                  window, scale, return_lse, out, lse, workspace)
