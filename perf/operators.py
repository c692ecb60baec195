"""Cases, plain forms and 64-bit definitions of the paged-cache operators.

Three operators of serving that are used one after the other for every new
token: rotary positions, the append of keys and values to a paged cache (with
the rotation applied on the way), and attention of the new tokens over the
cache.

  rope      x [T, H, D] or [B, H, S, D], one position per token; forward, and
            the gradient with respect to x.
  append    k, v [T, Hkv, D] of a ragged batch, written into pools of pages
            [pages, Hkv, page, D]; k (and q) rotated by the position that the
            token takes in its sequence.
  attend    q [T, Hq, D] of the same batch against every key of its sequence,
            causal, optionally within a window.

A ragged batch is (page_table [B, n], cu_seqlens [B + 1], seq_lens [B]): the
new tokens of sequence b are rows cu_seqlens[b]..cu_seqlens[b + 1] of the packed
tensors, they are the last ones of its seq_lens[b] tokens, and token p of the
sequence lives in row p % page of page page_table[b, p // page].
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # The rotation of one decode step's queries, half layout: a launch's
        # latency. [T, H, D] with one far position per sequence.
        {"name": "rope_step", "op": "rope", "batch": 0, "tokens": 64, "heads": 32, "dim": 128,
         "rot": 128, "interleaved": False, "grad": False, "type": "bf16", "base": 10000.0,
         "far": 131072, "factor": 1.0},
        # A prompt's queries as the QKV projection writes them, [4, 32, 2048, 128]
        # (this repository's prefill shape), adjacent pairs.
        {"name": "rope_prompt", "op": "rope", "batch": 4, "tokens": 2048, "heads": 32, "dim": 128,
         "rot": 128, "interleaved": True, "grad": False, "type": "bf16", "base": 10000.0,
         "far": 0, "factor": 1.0},
        # The gradient for a part of each head rotated with stretched
        # frequencies, in 32 bits, odd length, positions near a million.
        {"name": "rope_grad_far", "op": "rope", "batch": 0, "tokens": 5003, "heads": 24, "dim": 96,
         "rot": 64, "interleaved": False, "grad": True, "type": "fp32", "base": 500000.0,
         "far": 1000000, "factor": 1.1386},
        # One decode step of 96 sequences: every token lands in a page of its own;
        # k and q come out of one fused projection (strided rows).
        {"name": "append_step", "op": "append", "seqs": 96, "new": 1, "cached": 2047, "heads_kv": 8,
         "group": 4, "dim": 128, "rot": 128, "interleaved": False, "type": "bf16", "page": 16,
         "base": 10000.0, "fused": True, "pad": 32, "mix": 1},
        # Ragged prompt chunks, 64-token pages.
        {"name": "append_chunks", "op": "append", "seqs": 16, "new": 1531, "cached": 1000,
         "heads_kv": 8, "group": 4, "dim": 128, "rot": 128, "interleaved": False, "type": "bf16",
         "page": 64, "base": 500000.0, "fused": False, "pad": 0, "mix": 2},
        # One long prompt of a model with 64-wide heads, no rotation, fp16.
        {"name": "append_plain", "op": "append", "seqs": 1, "new": 16381, "cached": 0,
         "heads_kv": 16, "group": 1, "dim": 64, "rot": 0, "interleaved": False, "type": "fp16",
         "page": 32, "base": 10000.0, "fused": True, "pad": 0, "mix": 3},
        # One request's single token: latency.
        {"name": "attend_one", "op": "attend", "seqs": 1, "new": 1, "cached": 4095, "heads_kv": 8,
         "group": 4, "dim": 128, "type": "bf16", "page": 16, "window": 0, "lse": False, "pad": 0,
         "mix": 4},
        # A full decode batch of ragged contexts.
        {"name": "attend_batch", "op": "attend", "seqs": 64, "new": 1, "cached": 16384,
         "heads_kv": 8, "group": 4, "dim": 128, "type": "bf16", "page": 64, "window": 0,
         "lse": False, "pad": 0, "mix": 5},
        # Drafted tokens (several per sequence) verified at once, a sliding
        # window, 64-wide heads, fp16, with the log of the sums.
        {"name": "attend_drafts", "op": "attend", "seqs": 24, "new": 6, "cached": 20000,
         "heads_kv": 4, "group": 8, "dim": 64, "type": "fp16", "page": 32, "window": 4096,
         "lse": True, "pad": 5, "mix": 6},
        # A chunk of one long conversation: few rows, a very long cache.
        {"name": "attend_long", "op": "attend", "seqs": 1, "new": 509, "cached": 130000,
         "heads_kv": 4, "group": 7, "dim": 128, "type": "bf16", "page": 128, "window": 0,
         "lse": False, "pad": 0, "mix": 7},
        # This repository's prefill shape with a cache prefix: 4 sequences,
        # 32 heads of their own keys, 2048 new tokens after 2048 cached ones.
        {"name": "attend_prefill", "op": "attend", "seqs": 4, "new": -2048, "cached": -2048,
         "heads_kv": 32, "group": 1, "dim": 128, "type": "bf16", "page": 64, "window": 0,
         "lse": False, "pad": 0, "mix": 8},
        # One whole prompt, four query heads to a key head.
        {"name": "attend_prompt", "op": "attend", "seqs": 1, "new": -8190, "cached": 0,
         "heads_kv": 8, "group": 4, "dim": 128, "type": "bf16", "page": 64, "window": 0,
         "lse": True, "pad": 0, "mix": 9},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["rope", "append", "attend", "attend"])
        if op == "rope":
            dim = rng.choice([64, 72, 80, 96, 128, 192, 256])
            batch = rng.choice([0, 0, 1, 2, 3, 5])
            case = {"op": op, "batch": batch, "tokens": _log(rng, 1, 20000), "heads": rng.randint(1, 40),
                    "dim": dim, "rot": rng.choice([dim, dim, dim // 2, dim // 4 * 2]),
                    "interleaved": rng.random() < 0.5, "grad": rng.random() < 0.4,
                    "type": rng.choice(["bf16", "fp16", "fp32"]),
                    "base": rng.choice([10000.0, 500000.0, 1000000.0]),
                    "far": rng.choice([0, 5000, 1000000]), "factor": rng.choice([1.0, 1.25])}
        elif op == "append":
            dim = rng.choice([64, 80, 96, 128, 256])
            case = {"op": op, "seqs": _log(rng, 1, 200), "new": _log(rng, 1, 8192),
                    "cached": _log(rng, 1, 4096) - 1, "heads_kv": rng.choice([1, 2, 4, 8, 12]),
                    "group": rng.choice([1, 2, 4, 5, 8]), "dim": dim,
                    "rot": rng.choice([dim, dim, dim // 2, 0]), "interleaved": rng.random() < 0.5,
                    "type": rng.choice(["bf16", "fp16"]), "page": rng.choice([8, 16, 32, 64, 128]),
                    "base": rng.choice([10000.0, 500000.0]), "fused": rng.random() < 0.5,
                    "pad": rng.choice([0, 0, 3, 40]), "mix": rng.randrange(1 << 30)}
        else:
            kind = rng.choice(["step", "drafts", "chunk", "prompt"])
            group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
            case = {"op": op, "seqs": _log(rng, 1, 128) if kind != "prompt" else rng.randint(1, 6),
                    "new": {"step": 1, "drafts": rng.randint(2, max(2, 64 // group)),
                            "chunk": _log(rng, 16, 1024), "prompt": _log(rng, 100, 6000)}[kind],
                    "cached": _log(rng, 1, 60000) - 1 if kind != "prompt" else 0,
                    "heads_kv": rng.choice([1, 2, 4, 8, 16]), "group": group,
                    "dim": rng.choice([64, 96, 128] + ([256] if kind in ("step", "drafts") else [128])),
                    "type": rng.choice(["bf16", "bf16", "fp16"]),
                    "page": rng.choice([16, 32, 48, 64, 128]),
                    "window": rng.choice([0, 0, 0, 1000]), "lse": rng.random() < 0.4,
                    "pad": rng.choice([0, 0, 7]), "mix": rng.randrange(1 << 30)}
        if _fits(case):
            return case


def _fits(case):
    """No drawn case is larger than the largest listed one of its operator."""
    w = work(case)
    if case["op"] == "rope":
        return w["bytes"] <= 600e6
    if case["op"] == "append":
        pool = case["seqs"] * (abs(case["new"]) + case["cached"] + case["page"])
        return w["bytes"] <= 400e6 and pool * case["heads_kv"] * case["dim"] <= 1 << 28
    most = abs(case["new"]) + abs(case["cached"]) + case["page"]
    heads = case["heads_kv"] * case["group"]
    return (w["flops"] <= 0.5e12 and w["bytes"] <= 2e9
            and case["seqs"] * heads * abs(case["new"]) * most <= 32 * 8192 * 8192
            and case["seqs"] * case["heads_kv"] * most * case["dim"] <= 1 << 30)


def lengths(case):
    """(new, total) token counts of every sequence, from the case alone. A
    negative size in the case is every sequence's; a positive one is the
    largest, the first sequence's, and the others are spread below it."""
    r = random.Random(case["mix"])
    new, total = [], []
    for b in range(case["seqs"]):
        n, c = case["new"], case["cached"]
        n = -n if n < 0 else n if b == 0 else r.randint(max(1, n // 8), n)
        c = -c if c < 0 else c if b == 0 or c == 0 else r.randint(c // 8, c)
        new.append(n)
        total.append(n + c)
    return new, total


def _visible(case):
    """Per sequence: (keys that any new token sees, the sum over its new tokens of the keys seen)."""
    for n, s in zip(*lengths(case)):
        w = case["window"] or s
        first = s - n  # position of the first new token
        keys = s - max(0, first - w + 1)
        full = max(0, min(n, w - first))  # tokens whose window still starts at key 0
        yield keys, full * first + full * (full + 1) // 2 + (n - full) * w


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "rope":
        n = max(1, case["batch"]) * case["tokens"] * case["heads"]
        return {"bytes": 2.0 * n * case["dim"] * size + 8.0 * case["tokens"], "flops": 3.0 * n * case["rot"]}
    new, total = lengths(case)
    q_heads = case["heads_kv"] * case["group"]
    row = case["dim"] * size
    if case["op"] == "append":
        n = sum(new)
        moved = 2 * case["heads_kv"] + (q_heads if case["rot"] else 0)
        return {"bytes": 2.0 * n * moved * row + 4.0 * n,
                "flops": 3.0 * n * case["rot"] * (q_heads + case["heads_kv"])}
    seen = list(_visible(case))
    keys, pairs = sum(k for k, _ in seen), sum(p for _, p in seen)
    return {"bytes": 2.0 * keys * case["heads_kv"] * row + 2.0 * sum(new) * q_heads * row
            + 4.0 * keys / case["page"] + (4.0 * sum(new) * q_heads if case["lse"] else 0.0),
            "flops": 4.0 * pairs * q_heads * case["dim"]}


def _frequencies(case, device):
    """Radians per position of each rotated pair, as a program keeps them."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=device)
    return (case["base"] ** (-2.0 * i / max(1, case["rot"]))).float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(dt)

    state = {"case": case}
    if case["op"] == "rope":
        T, H, D = case["tokens"], case["heads"], case["dim"]
        state["inv_freq"] = _frequencies(case, "cuda")
        state["x"] = normal(case["batch"], H, T, D) if case["batch"] else normal(T, H, D)
        at = torch.randint(0, max(1, case["far"]), (1,), device="cuda", generator=g)
        state["positions"] = at + torch.arange(T, device="cuda")
        return state

    new, total = lengths(case)
    B, page, hkv, D = case["seqs"], case["page"], case["heads_kv"], case["dim"]
    hq = hkv * case["group"]
    need = [-(-s // page) for s in total]
    # a pool with a few pages that belong to nobody, handed out in no order
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    width = max(need)
    first = np.cumsum([0] + need[:-1])
    at = first[:, None] + np.arange(width)[None, :]
    at[np.arange(width)[None, :] >= np.array(need)[:, None]] = pages - 1  # past the end: any page
    state["page_table"] = order[torch.from_numpy(at).cuda()].contiguous()
    state["cu_seqlens"] = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device="cuda")
    state["seq_lens"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    state["n"], state["max_new"] = sum(new), max(new)
    rows = state["n"] + case["pad"]  # rows behind the last sequence: a batch padded to a fixed size
    if case["op"] == "append":
        state["inv_freq"] = _frequencies(case, "cuda") if case["rot"] else None
        if case["fused"]:  # one projection's rows, [q | k | v]
            both = normal(rows, (hq + 2 * hkv), D)
            state["q"], state["k"], state["v"] = both[:, :hq], both[:, hq:hq + hkv], both[:, hq + hkv:]
        else:
            state["q"], state["k"], state["v"] = normal(rows, hq, D), normal(rows, hkv, D), normal(rows, hkv, D)
        state["q_out"] = torch.zeros(rows, hq, D, dtype=dt, device="cuda")
        state["k_pages"] = torch.zeros(pages, hkv, page, D, dtype=dt, device="cuda")
        state["v_pages"] = torch.zeros(pages, hkv, page, D, dtype=dt, device="cuda")
    else:
        state["q"] = normal(rows, hq, D)
        state["k_pages"], state["v_pages"] = normal(pages, hkv, page, D), normal(pages, hkv, page, D)
        state["out"] = torch.zeros(rows, hq, D, dtype=dt, device="cuda")
        state["lse"] = torch.zeros(rows, hq, dtype=torch.float32, device="cuda") if case["lse"] else None
    return state


def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[state["case"]["op"]](state)


def _run_own(state):
    from polykernel_b200 import ops
    case = state["case"]
    if case["op"] == "rope":
        f = ops.rope_backward if case["grad"] else ops.rope
        return f(state["x"], state["positions"], state["inv_freq"], interleaved=case["interleaved"],
                 factor=case["factor"])
    if case["op"] == "append":
        if case["rot"]:
            ops.paged_kv_append(state["k"], state["v"], state["k_pages"], state["v_pages"],
                                state["page_table"], state["cu_seqlens"], state["seq_lens"],
                                inv_freq=state["inv_freq"], interleaved=case["interleaved"],
                                q=state["q"], q_out=state["q_out"])
        else:
            ops.paged_kv_append(state["k"], state["v"], state["k_pages"], state["v_pages"],
                                state["page_table"], state["cu_seqlens"], state["seq_lens"])
        return {"k": state["k_pages"], "v": state["v_pages"], "q": state["q_out"]}
    ops.paged_attention(state["q"], state["k_pages"], state["v_pages"], state["page_table"],
                        state["cu_seqlens"], state["seq_lens"], max_q_len=state["max_new"],
                        window=case["window"] or None, out=state["out"], lse=state["lse"])
    return {"out": state["out"], "lse": state["lse"]}


# ------------------------------------------------------------- plain forms --
def _rotated(x, positions, inv_freq, interleaved, factor=1.0, grad=False):
    """x [..., D] in 32 bits, its first 2 * len(inv_freq) values rotated by
    position * inv_freq; `positions` broadcasts against x's leading axes. The
    angles are formed in 64 bits: a far position's angle has none left in 32."""
    angle = positions.double()[..., None] * inv_freq.double()
    c, s = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    if grad:
        s = -s
    x = x.float()
    r = 2 * inv_freq.numel()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, x[..., r:]], dim=-1)


def _plain_rope(state):
    case, x, pos = state["case"], state["x"], state["positions"]
    at = pos if case["batch"] else pos[:, None]  # [B, H, S, D] or [T, H, D]
    return _rotated(x, at, state["inv_freq"], case["interleaved"], case["factor"], case["grad"]).to(x.dtype)


def _places(state):
    """(sequence, position in it) of every new token."""
    cu = state["cu_seqlens"].long()
    t = torch.arange(state["n"], device=cu.device)
    seq = torch.searchsorted(cu[1:], t, right=True)
    return seq, state["seq_lens"].long()[seq] - cu[seq + 1] + t


def _plain_append(state):
    case, n = state["case"], state["n"]
    seq, pos = _places(state)
    page = state["page_table"].long()[seq, pos // case["page"]]
    row = pos % case["page"]
    k = state["k"][:n]
    if case["rot"]:
        k = _rotated(k, pos[:, None], state["inv_freq"], case["interleaved"])
        q = _rotated(state["q"][:n], pos[:, None], state["inv_freq"], case["interleaved"])
        state["q_out"][:n] = q.to(state["q_out"].dtype)
    state["k_pages"][page, :, row] = k.to(state["k_pages"].dtype)
    state["v_pages"][page, :, row] = state["v"][:n]
    return {"k": state["k_pages"], "v": state["v_pages"], "q": state["q_out"]}


def _plain_attend(state):
    case, n, q = state["case"], state["n"], state["q"]
    B, hkv, G, D, page = case["seqs"], case["heads_kv"], case["group"], case["dim"], case["page"]
    dev = q.device
    cu, total = state["cu_seqlens"].long(), state["seq_lens"].long()
    most = state["max_new"]
    # every sequence's new tokens and keys as dense padded rows
    i = torch.arange(most, device=dev)
    rows = (cu[:-1, None] + i).clamp(max=n - 1)
    qd = q[rows].float().view(B, most, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * most, D)
    table = state["page_table"].long()
    keys = table.shape[1] * page
    kd = state["k_pages"][table].permute(0, 2, 1, 3, 4).reshape(B, hkv, keys, D).float()
    vd = state["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(B, hkv, keys, D).float()
    at = total[:, None] - (cu[1:] - cu[:-1])[:, None] + i  # [B, most] positions
    j = torch.arange(keys, device=dev)
    seen = (j <= at[..., None]) & (j < total[:, None, None])
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    s = torch.matmul(qd, kd.transpose(-1, -2)).view(B, hkv, G, most, keys)
    s = s.mul_(1.0 / math.sqrt(D)).masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp_(min=-3e38)
    p = s.sub_(top).exp_()
    mass = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, G * most, keys), vd).view(B, hkv, G, most, D) / mass
    seq, pos = _places(state)
    t = torch.arange(n, device=dev) - cu[seq]
    state["out"][:n] = o.permute(0, 3, 1, 2, 4)[seq, t].reshape(n, hkv * G, D).to(q.dtype)
    if case["lse"]:
        lse = (top + mass.log()).squeeze(-1)
        state["lse"][:n] = lse.permute(0, 3, 1, 2)[seq, t].reshape(n, hkv * G)
    return {"out": state["out"], "lse": state["lse"]}


# ------------------------------------------------------ 64-bit definitions --
def _exact_turn(x, positions, inv_freq, interleaved, factor, grad):
    """Each pair (a, b) of x as the complex number a + ib, times factor * e^(i angle)."""
    x = x.double().clone()
    half = inv_freq.numel()
    turn = torch.polar(torch.full_like(positions, factor, dtype=torch.float64)[..., None]
                       .expand(*positions.shape, half).contiguous(),
                       (-1.0 if grad else 1.0) * positions.double()[..., None] * inv_freq.double())
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rope":
        at = state["positions"] if case["batch"] else state["positions"][:, None]
        return _exact_turn(state["x"], at, state["inv_freq"], case["interleaved"], case["factor"], case["grad"])
    cu, total = state["cu_seqlens"].tolist(), state["seq_lens"].tolist()
    table, page = state["page_table"].long(), case["page"]
    if case["op"] == "append":
        k, v, q = (state[n].double() for n in ("k_pages", "v_pages", "q_out"))
        for b in range(case["seqs"]):
            rows = slice(cu[b], cu[b + 1])
            pos = torch.arange(total[b] - (cu[b + 1] - cu[b]), total[b], device=k.device)
            kb = state["k"][rows].double()
            if case["rot"]:
                args = (pos[:, None], state["inv_freq"], case["interleaved"], 1.0, False)
                kb, q[rows] = _exact_turn(kb, *args), _exact_turn(state["q"][rows], *args)
            k[table[b, pos // page], :, pos % page] = kb
            v[table[b, pos // page], :, pos % page] = state["v"][rows].double()
        return {"k": k, "v": v, "q": q}
    out, lse = state["out"].double(), None if state["lse"] is None else state["lse"].double()
    G, scale = case["group"], case["dim"] ** -0.5
    for b in range(case["seqs"]):
        rows, n, s = slice(cu[b], cu[b + 1]), cu[b + 1] - cu[b], total[b]
        used = table[b, :-(-s // page)]
        pos = torch.arange(s - n, s, device=out.device)[:, None]
        key = torch.arange(s, device=out.device)[None, :]
        hidden = (key > pos) | ((key <= pos - case["window"]) if case["window"] else (key < 0))
        for h in range(case["heads_kv"]):
            kb = state["k_pages"][used, h].reshape(-1, case["dim"])[:s].double()
            vb = state["v_pages"][used, h].reshape(-1, case["dim"])[:s].double()
            for g in range(h * G, h * G + G):
                score = (state["q"][rows, g].double() @ kb.T * scale).masked_fill(hidden, -math.inf)
                sums = torch.logsumexp(score, dim=-1, keepdim=True)
                out[rows, g] = torch.exp(score - sums) @ vb
                if lse is not None:
                    lse[rows, g] = sums[:, 0]
    return {"out": out, "lse": lse}
