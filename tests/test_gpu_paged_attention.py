"""GPU: attention over a paged cache against the definition in 64 bits.

Tolerance per output value, from the arithmetic, with p the exact weights of a row,
u = eps / 2 of the type and X = max_j sum_d |q_d k_jd| * scale over the row's keys:
* output rounding: u |o|;
* P rounded to the type once (tile kernel): u sum_j p_j |v_j|; in fp16 also half
  a step of its subnormals per key, 2^-25 sum_j |v_j| (the row's largest P is at least 1);
* scores: tensor-core fp32 sums lose at most 2^-22 of X per 16 products, below
  2^-18 X for 256 products; numerator and denominator move by that each: 2^-17 X sum_j p_j |v_j|;
* sums over n keys in steps of 16, 2^-22 each, the exponentials (2^-22) and the
  scaling of the joins: (n / 16 + 32) 2^-22 sum_j p_j |v_j|.
The log-sum: 2^-17 X + (n / 16 + 32) 2^-22 + 2^-22 |lse|.
"""
import math

import pytest

from tests.test_gpu_rope_append import batch, gen

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(cuda):
    import polykernel_b200 as pk
    pk.lib()
    pk.device_error()
    return pk.ops


@pytest.fixture(autouse=True)
def no_device_error(cuda):
    import polykernel_b200 as pk
    yield
    assert pk.device_error() == 0


def make(new, total, page, hkv, group, dim, dtype, seed=0, pad=2, token_major=False, width=None):
    """Random q and pools: rows of live tokens normal, everything else NaN."""
    g = gen(seed)
    table, cu, lens, pages = batch(new, total, page, seed=seed, width=width)
    n = sum(new)
    q = torch.randn(n + pad, hkv * group, dim, device="cuda", generator=g).to(dtype)
    pools = []
    for _ in range(2):
        shape = (pages, page, hkv, dim) if token_major else (pages, hkv, page, dim)
        pool = torch.full(shape, float("nan"), device="cuda", dtype=dtype)
        pool = pool.transpose(1, 2) if token_major else pool
        for b, t in enumerate(total):
            pos = torch.arange(t, device="cuda")
            pool[table[b].long()[pos // page], :, pos % page] = torch.randn(
                t, hkv, dim, device="cuda", generator=g).to(dtype)
        pools.append(pool)
    return q, *pools, table, cu, lens


def definition(q, kp, vp, table, cu, lens, causal=True, window=None, scale=None):
    """(out, lse, tolerance of out, tolerance of lse), 64 bits; masked keys take no part."""
    n, hq, dim = q.shape
    hkv, page = kp.shape[1:3]
    G = hq // hkv
    scale = dim ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out, tol = torch.zeros(n, hq, dim, dtype=torch.float64, device="cuda"), torch.zeros(n, hq, dim, device="cuda").double()
    lse, ltol = torch.zeros(n, hq, dtype=torch.float64, device="cuda"), torch.zeros(n, hq, device="cuda").double()
    cu, lens = cu.tolist(), lens.tolist()
    for b, s in enumerate(lens):
        rows = slice(cu[b], cu[b + 1])
        c = cu[b + 1] - cu[b]
        if c == 0:
            continue
        pos = torch.arange(s - c, s, device="cuda")[:, None]
        key = torch.arange(s, device="cuda")
        seen = (key <= pos) if causal else (key >= 0).expand(c, s)
        if window:
            seen = seen & (key > pos - window)
        at = (table[b].long()[key // page], slice(None), key % page)
        for h in range(hkv):
            k, v = kp[at][:, h].double(), vp[at][:, h].double()
            for g in range(G):
                qh = q[rows, h * G + g].double()
                sc = torch.where(seen, qh @ k.T * scale, -math.inf)
                L = torch.logsumexp(sc, -1)
                p = torch.where(seen, torch.exp(sc - L[:, None].clamp(min=-1e300)), 0.0)
                vs = torch.where(seen[..., None], v, 0.0) if not torch.isfinite(v).all() else v
                o = torch.einsum("ij,ijd->id", p, vs) if vs.dim() == 3 else p @ vs
                pv = torch.einsum("ij,ijd->id", p, vs.abs()) if vs.dim() == 3 else p @ vs.abs()
                X = torch.where(seen, qh.abs() @ k.abs().T * scale, 0.0).amax(-1, keepdim=True) if s else 0.0
                sums = (s / 16 + 32) * 2.0 ** -22
                t = u * o.abs() * (1 + 2.0 ** -9) + pv * (u * (1 + 2.0 ** -9) + 2.0 ** -17 * X + sums)
                if q.dtype == torch.float16:
                    sv = torch.where(seen[..., None], vs, 0.0).abs().sum(1) if vs.dim() == 3 else seen.double() @ v.abs()
                    t = t + 2.0 ** -25 * (sv + 1)
                out[rows, h * G + g], tol[rows, h * G + g] = o, t
                lse[rows, h * G + g] = L
                ltol[rows, h * G + g] = (2.0 ** -17 * X).squeeze(-1) + sums + 2.0 ** -22 * L.abs() if s else 0.0
    return out, lse, tol, ltol


def check(ops, args, max_q_len=None, **kw):
    """Run, compare with the definition, and check that rows of no sequence are left alone."""
    q, cu = args[0], args[4]
    n = int(cu[-1])
    out = torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    got = ops.paged_attention(*args, max_q_len=max_q_len, out=out, lse=lse, return_lse=True, **kw)
    assert got[0] is out and got[1] is lse
    want, wl, tol, ltol = definition(*args, **kw)
    far = (out.double() - want).abs()[:n] / tol[:n].clamp(min=1e-300)
    assert torch.equal(out[:n].isnan(), want[:n].isnan())
    assert bool((far.nan_to_num(0) <= 1).all()), float(far.nan_to_num(0).max())
    dead = wl[:n] == -math.inf
    assert torch.equal(lse[:n] == -math.inf, dead)
    assert bool(((lse.double() - wl).abs()[:n][~dead].nan_to_num(0) <= ltol[:n][~dead].nan_to_num(1)).all())
    assert bool((out[n:] == 7).all()) and bool((lse[n:] == 7).all())
    return out


ROWS = [  # new, total, page, key heads, group, dim: few rows per key head
    ([1], [1], 16, 1, 1, 64),
    ([1], [4096], 16, 8, 4, 128),
    ([1, 1, 1, 1], [1, 63, 64, 65], 16, 2, 4, 128),
    ([1, 0, 1], [1000, 77, 129], 64, 1, 16, 96),
    ([3, 5, 1], [3, 200, 513], 32, 2, 5, 64),
    ([4, 4], [700, 5], 8, 2, 8, 128),
    ([1, 1], [300, 40], 48, 3, 7, 80),
    ([2, 1], [130, 257], 16, 1, 3, 256),
    ([9, 1], [1030, 31], 64, 2, 7, 256),
    ([1, 2], [90, 333], 24, 2, 32, 72),
    ([1] * 70, [1 + 37 * i % 411 for i in range(70)], 16, 2, 2, 64),
    ([1], [20000], 128, 1, 8, 128),
    ([1, 1], [15, 1], 128, 4, 1, 8),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", ROWS, ids=str)
def test_few_rows(ops, case, dtype):
    check(ops, make(*case, dtype), max_q_len=max(case[0]))


TILES = [  # many rows per key head
    ([65], [65], 16, 1, 1, 64),
    ([128], [128], 64, 2, 1, 128),
    ([129], [400], 16, 1, 4, 128),
    ([257], [257], 32, 2, 1, 128),
    ([300, 1, 77], [300, 900, 1000], 64, 2, 4, 128),
    ([40, 200, 0, 33], [40, 1500, 10, 34], 16, 1, 3, 96),
    ([70], [5000], 128, 1, 7, 128),
    ([500], [1111], 8, 2, 5, 72),
    ([20, 31], [2000, 31], 48, 2, 16, 64),
    ([3, 2], [260, 129], 64, 1, 100, 128),
    ([2], [700], 64, 1, 128, 64),
    ([1000], [1000], 256, 1, 2, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", TILES, ids=str)
def test_many_rows(ops, case, dtype):
    check(ops, make(*case, dtype), max_q_len=max(case[0]))


@pytest.mark.parametrize("window", [1, 17, 128, 1000])
@pytest.mark.parametrize("case", [ROWS[2], ROWS[4], ROWS[5], ROWS[11], TILES[3], TILES[4], TILES[6]], ids=str)
def test_window(ops, case, window):
    check(ops, make(*case, torch.bfloat16), max_q_len=max(case[0]), window=window)


@pytest.mark.parametrize("case", [ROWS[2], ROWS[4], TILES[2], TILES[4]], ids=str)
def test_not_causal_and_scaled(ops, case):
    check(ops, make(*case, torch.float16), max_q_len=max(case[0]), causal=False, scale=0.3)


@pytest.mark.parametrize("case", [ROWS[4], ROWS[7], TILES[4], TILES[8]], ids=str)
@pytest.mark.parametrize("max_q_len", [None, 1, 10 ** 9])
def test_max_q_len_only_selects(ops, case, max_q_len):
    check(ops, make(*case, torch.bfloat16), max_q_len=max_q_len)


@pytest.mark.parametrize("case", [ROWS[4], TILES[4]], ids=str)
def test_token_major_pools_and_strided_q(ops, case):
    q, *rest = make(*case, torch.bfloat16, token_major=True)
    wide = torch.randn(q.shape[0], q.shape[1] + 3, q.shape[2] + 8, device="cuda").bfloat16()
    wide[:, 2:-1, 8:] = q
    check(ops, (wide[:, 2:-1, 8:], *rest), max_q_len=max(case[0]))


@pytest.mark.parametrize("case", [ROWS[1], ROWS[4], ROWS[5], ROWS[9], TILES[2], TILES[4], TILES[10]], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite(ops, case, bad):
    """A key's value that is not finite reaches the rows that see the key, and no
    other; a score that is not finite likewise."""
    args = make(*case, torch.bfloat16)
    q, kp, vp, table, cu, lens = args
    page = case[2]
    for b, (c, t) in enumerate(zip(case[0], case[1])):
        if c > 1:  # the middle one of the new tokens
            at = t - c // 2
            vp[table[b, at // page], :, at % page, ::3] = bad
            if bad != bad:
                kp[table[b, at // page], 0, at % page] = bad
    # only rows before the bad keys are compared with the definition's finite
    # values; behind them both are not finite
    n = int(cu[-1])
    out, lse = ops.paged_attention(*args, max_q_len=max(case[0]), return_lse=True)
    want, wl, tol, ltol = definition(*args)
    fine = torch.isfinite(want[:n])
    assert torch.equal(torch.isfinite(out[:n]), fine)
    assert bool(((out[:n].double() - want[:n]).abs()[fine] <= tol[:n][fine]).all())


@pytest.mark.parametrize("rows", ["few", "many"])
def test_large_and_equal_scores(ops, rows):
    """Scores in the thousands (one key takes all the weight), and all equal."""
    case = ([2, 1], [300, 64], 16, 2, 4, 128) if rows == "few" else ([200], [500], 32, 2, 2, 128)
    q, kp, vp, table, cu, lens = make(*case, torch.bfloat16)
    check(ops, (q * 60, kp, vp, table, cu, lens), max_q_len=max(case[0]))
    check(ops, (torch.zeros_like(q), kp, vp, table, cu, lens), max_q_len=max(case[0]))


@pytest.mark.parametrize("case", [ROWS[2], ROWS[10], TILES[4], TILES[6]], ids=str)
def test_repeatable(ops, case):
    """The order of every sum is fixed: runs agree to the bit."""
    args = make(*case, torch.bfloat16)
    first = ops.paged_attention(*args, max_q_len=max(case[0]))[:sum(case[0])].clone()
    for _ in range(5):
        again = ops.paged_attention(*args, max_q_len=max(case[0]))[:sum(case[0])]
        assert torch.equal(first, again)


def test_shared_pages(ops):
    """Two sequences that share their first pages."""
    new, total, page = [1, 1], [70, 90], 16
    q, kp, vp, table, cu, lens = make(new, total, page, 2, 4, 128, torch.bfloat16)
    table[1, :4] = table[0, :4]
    check(ops, (q, kp, vp, table, cu, lens), max_q_len=1)


def test_captured_and_replayed(ops):
    """Captured graphs follow the lengths; two graphs with workspaces of their own
    replay side by side."""
    cases = [([1, 1, 1], [40, 700, 9], 16, 2, 4, 128), ([100, 30], [400, 30], 16, 2, 4, 128)]
    runs = []
    for case in cases:
        q, kp, vp, table, cu, lens = make(*case, torch.bfloat16, width=60)
        kp.nan_to_num_(0.1)
        vp.nan_to_num_(0.1)
        table.clamp_(min=0)  # pages past the present end, for the lengths to grow into
        args = (q, kp, vp, table, cu, lens)
        out = torch.zeros_like(q)
        ops.paged_attention(*args, max_q_len=max(case[0]), out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(*args, max_q_len=max(case[0]), out=out)
        runs.append((graph, args, out, torch.cuda.Stream()))
    for grow in (0, 5, 130):
        for graph, args, out, stream in runs:
            args[5].add_(grow)
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, args, out, stream in runs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for graph, args, out, stream in runs:
            n = int(args[4][-1])
            want, _, tol, _ = definition(*args)
            assert bool(((out.double() - want).abs() <= tol)[:n].all())


def test_other_stream_and_own_workspace(ops):
    case = ROWS[10]
    args = make(*case, torch.bfloat16)
    stream = torch.cuda.Stream()
    workspace = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        out = ops.paged_attention(*args, max_q_len=1, workspace=workspace)
    stream.synchronize()
    want, _, tol, _ = definition(*args)
    n = sum(case[0])
    assert bool(((out.double() - want).abs() <= tol)[:n].all())


def test_far_pages(ops):
    """Pool offsets that pass 2^31 values."""
    page, hkv, dim = 128, 8, 128
    pages = (1 << 31) // (page * hkv * dim) + 40
    kp, vp = (torch.zeros(pages, hkv, page, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    for new, max_q_len in (([1, 1], 1), ([90, 70], 90)):
        total = [300, 129]
        table = torch.arange(pages - 6, pages, device="cuda", dtype=torch.int32).view(2, 3).flip(0).contiguous()
        g = gen(3)
        n = sum(new)
        q = torch.randn(n, hkv * 2, dim, device="cuda", generator=g).bfloat16()
        k, v = (torch.randn(n, hkv, dim, device="cuda", generator=g).bfloat16() for _ in range(2))
        kp[-6:], vp[-6:] = (torch.randn(6, hkv, page, dim, device="cuda", generator=g).bfloat16() for _ in range(2))
        cu = torch.tensor([0] + new, device="cuda").cumsum(0).int()
        lens = torch.tensor(total, device="cuda", dtype=torch.int32)
        ops.paged_kv_append(k, v, kp, vp, table, cu, lens)
        last = total[0] - 1
        assert torch.equal(kp[table[0, last // page].long(), :, last % page], k[new[0] - 1])
        check(ops, (q, kp, vp, table, cu, lens), max_q_len=max_q_len)


def test_window_past_two_to_the_30(ops):
    """A window of more than 2^30 keys is kept exactly: its first key, among 2^30 + 1024
    of one shared page, is the one that decides the output."""
    page, n, window = 1024, 2 ** 30 + 1024, 2 ** 30 + 5
    kp = torch.zeros(2, 1, page, 8, device="cuda", dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    table = torch.zeros(1, n // page, dtype=torch.int32, device="cuda")
    first = n - window
    table[0, first // page] = 1
    kp[1, 0, first % page] = 8.0  # a score of 8 * 8 = 64 natural units above all others
    vp[1, 0, first % page] = 3.0
    q = torch.ones(1, 1, 8, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    # the others' weight, 2^30.1 exp(-64), is below a half step of 3 by far
    got = ops.paged_attention(q, kp, vp, table, cu, lens, window=window, scale=1.0)
    assert bool((got == 3.0).all())
    assert bool((ops.paged_attention(q, kp, vp, table, cu, lens, window=window - 1, scale=1.0) == 0.0).all())


def test_prompt_then_tokens(ops):
    """The operators as a program uses them: a projection, its split, the rotated
    append and attention, for a ragged prompt and then token by token, against
    the same in 64 bits over the whole contexts."""
    hq, hkv, dim, page = 8, 2, 64, 16
    g = gen(11)
    freq, factor = ops.rope_frequencies(dim, 10000.0, {"type": "linear", "factor": 2.0})
    model = hq * dim
    w = (torch.randn(model, (hq + 2 * hkv) * dim, device="cuda", generator=g) / model ** 0.5).bfloat16()
    prompts = [37, 5, 130]
    steps = 4
    table, _, _, pages = batch(prompts, [p + steps for p in prompts], page)
    kp, vp = (torch.full((pages, hkv, page, dim), float("nan"), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    seen = [[] for _ in prompts]  # projected rows of each sequence
    for step in range(steps + 1):
        new = prompts if step == 0 else [1, 1, 1]
        n = sum(new)
        cu = torch.tensor([0] + new, device="cuda").cumsum(0).int()
        lens += torch.tensor(new, device="cuda", dtype=torch.int32)
        x = torch.randn(n, model, device="cuda", generator=g).bfloat16()
        qkv = ops.matmul(x, w).view(n, hq + 2 * hkv, dim)
        q, k, v = qkv.split([hq, hkv, hkv], dim=1)
        qr = ops.paged_kv_append(k, v, kp, vp, table, cu, lens, inv_freq=freq, factor=factor, q=q)
        out = ops.paged_attention(qr, kp, vp, table, cu, lens, max_q_len=max(new))
        want, _, tol, _ = definition(qr, kp, vp, table, cu, lens)
        assert bool(((out.double() - want).abs() <= tol).all())
        # and the cache holds the rotated keys of the whole context
        t = 0
        for b, c in enumerate(new):
            seen[b].append((k[t:t + c].clone(), v[t:t + c].clone()))
            t += c
            kb, vb = (torch.cat([s[i] for s in seen[b]]) for i in (0, 1))
            pos = torch.arange(kb.shape[0], device="cuda")
            at = table[b].long()[pos // page], slice(None), pos % page
            assert torch.equal(vp[at], vb)
            assert torch.equal(kp[at], ops.rope(kb, pos, freq, factor=factor))


def test_refusals(ops):
    q, kp, vp, table, cu, lens = make([2, 1], [20, 9], 16, 2, 2, 64, torch.bfloat16)

    def refuses(error, f, *a, **kw):
        with pytest.raises(error):
            f(*a, **kw)

    at = ops.paged_attention
    rest = (table, cu, lens)
    refuses(TypeError, at, q.float(), kp, vp, *rest)
    refuses(TypeError, at, q.half(), kp, vp, *rest)
    refuses(TypeError, at, q, kp, vp.half(), *rest)
    refuses(TypeError, at, q, kp, vp, table.long(), cu, lens)
    refuses(TypeError, at, q, kp, vp, table, cu.long(), lens)
    refuses(ValueError, at, q, kp, vp, table, cu, lens[:1])
    refuses(ValueError, at, q, kp, vp, table, cu[:2], lens)
    refuses(ValueError, at, q, kp, vp, table.cpu(), cu, lens)
    refuses(ValueError, at, q[:, :3], kp, vp, *rest)
    refuses(ValueError, at, q, kp, vp[:, :, :8], *rest)
    refuses(ValueError, at, q, kp[:, :, :12], vp[:, :, :12], *rest)
    refuses(ValueError, at, q[..., :60], kp[..., :60], vp[..., :60], *rest)
    refuses(ValueError, at, q, kp[:0], vp[:0], *rest)
    refuses(ValueError, at, q, kp, vp, *rest, window=0)
    refuses(ValueError, at, q, kp, vp, *rest, window=4, causal=False)
    refuses(ValueError, at, q, kp, vp, *rest, scale=0.0)
    refuses(ValueError, at, q, kp, vp, *rest, scale=float("nan"))
    refuses(ValueError, at, q, kp, vp, *rest, max_q_len=-1)
    refuses(ValueError, at, q, kp, vp, *rest, out=torch.empty_like(q)[:2])
    refuses(ValueError, at, q, kp, vp, *rest, lse=torch.empty(2, 2, device="cuda"))
    refuses(ValueError, at, torch.empty(q.numel() + 4, device="cuda").bfloat16()[4:].view_as(q), kp, vp, *rest)
    refuses(ValueError, at, q.transpose(1, 2), kp, vp, *rest)
    ap = ops.paged_kv_append
    k = q[:, :2]
    refuses(ValueError, ap, k[:, :1], k, kp, vp, *rest)
    refuses(ValueError, ap, k, k[:2], kp, vp, *rest)
    refuses(ValueError, ap, k, k, kp, vp, *rest, q=q)
    refuses(TypeError, ap, k, k, kp, vp, *rest, inv_freq=torch.ones(8, device="cuda", dtype=torch.float64))
    refuses(ValueError, ap, k, k, kp, vp, *rest, inv_freq=torch.ones(33, device="cuda"))
    refuses(ValueError, ap, k, k, kp, vp, *rest, inv_freq=torch.ones(8, device="cuda"), q_out=q)
    refuses(ValueError, ap, k, k, kp, vp, *rest, inv_freq=torch.ones(8, device="cuda"), q=q, q_out=q.flip(0)[:2])
    rp, pos, f = ops.rope, torch.zeros(5, dtype=torch.int64, device="cuda"), torch.ones(32, device="cuda")
    assert rp(q, pos, f).shape == q.shape
    refuses(TypeError, rp, q, pos.int(), f)
    refuses(ValueError, rp, q, pos[:2], f)
    refuses(ValueError, rp, q, pos.cpu(), f)
    refuses(ValueError, rp, q, pos, torch.ones(33, device="cuda"))
    refuses(ValueError, rp, q.transpose(1, 2), pos[:4], f)
    refuses(ValueError, rp, q, pos, f, factor=float("inf"))
    refuses(TypeError, rp, q, pos, f, out=q.half())


def device_error():
    import polykernel_b200 as pk
    return pk.device_error()


@pytest.mark.parametrize("case", [([1, 2, 1], [200, 70, 33], 16, 2, 4, 128),
                                  ([100, 2, 140], [200, 70, 333], 32, 2, 4, 128)], ids=str)
def test_wrong_batches(ops, case):
    """Descriptions that lead out of range (tests/cpp/paged_index_test.cpp walks the
    same arithmetic) are cut off there, and reported; other sequences are served."""
    most = max(case[0])
    new, page = case[0], case[2]
    args = make(*case, torch.bfloat16)
    q, kp, vp, table, cu, lens = args
    n = sum(new)
    want, wl, tol, ltol = definition(*args)
    zeros = torch.zeros_like

    def others(out, b):
        rows = torch.ones(n, dtype=torch.bool, device="cuda")
        rows[int(cu[b]):int(cu[b + 1])] = False
        return bool(((out[:n].double() - want[:n]).abs() <= tol[:n])[rows].all())

    for page_index in (-1, kp.shape[0], 2 ** 31 - 1, -(2 ** 31)):
        t = table.clone()
        t[1, 1] = page_index
        out = ops.paged_attention(q, kp, vp, t, cu, lens, max_q_len=most)
        assert device_error() == 8 and others(out, 1)
        # the page's keys read as zeros
        t[1, 1] = kp.shape[0]
        more = [torch.cat([x, zeros(x[:1])]) for x in (kp, vp)]
        w, _, tl, _ = definition(q, *more, t, cu, lens)
        assert bool(((out.double() - w).abs() <= tl)[:n].all())
        # and the append drops its tokens
        k, v = (torch.ones(q.shape[0], kp.shape[1], kp.shape[3], device="cuda").bfloat16() for _ in range(2))
        t[1] = page_index
        kc, vc = kp.clone(), vp.clone()
        ops.paged_kv_append(k, v, kc, vc, t, cu, lens)
        assert device_error() == 8
        changed = (kc.nan_to_num(9.0) != kp.nan_to_num(9.0)).any(-1).any(1)
        assert int(changed.sum()) == n - new[1]
    # fewer tokens than new ones: those before position 0 see nothing
    short = lens.clone()
    short[1] = new[1] - 1
    out, lse = ops.paged_attention(q, kp, vp, table, cu, short, max_q_len=most, return_lse=True)
    assert device_error() == 8 and others(out, 1)
    first = int(cu[1])
    assert bool((out[first] == 0).all()) and bool((lse[first] == -math.inf).all())
    # a length past the table, a negative one, offsets out of order or past the rows
    for bad in (table.shape[1] * page + 1, 2 ** 31 - 1, -5, -(2 ** 31)):
        wrong = lens.clone()
        wrong[1] = bad
        safe = table.clamp(min=0)
        out = ops.paged_attention(q, kp, vp, safe, cu, wrong, max_q_len=most)
        assert device_error() == 8 and others(out, 1)
    for bad in (-3, 2 ** 31 - 1, n + 50):
        wrong = cu.clone()
        wrong[3] = bad
        out = ops.paged_attention(q, kp, vp, table, wrong, lens, max_q_len=most)
        assert device_error() == 8 and others(out, 2)


@pytest.mark.parametrize("case", [([1, 3], [9, 300], 16, 2, 4, 8), ([200, 1], [200, 77], 16, 1, 4, 8),
                                  ([90], [700], 16, 1, 2, 40)], ids=str)
def test_narrow_heads_and_sliced_table(ops, case):
    q, kp, vp, table, cu, lens = make(*case, torch.bfloat16)
    wide = torch.full((table.shape[0], table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:-3] = table
    check(ops, (q, kp, vp, wide[:, 2:-3], cu, lens), max_q_len=max(case[0]))


@pytest.mark.parametrize("max_q_len", [None, 1, 300])
def test_many_sequences(ops, max_q_len):
    """Single tokens, drafts and prompts in one batch of several hundred."""
    B = 300
    new = [1 if b % 7 else (300 if b == 140 else 1 + b % 40) for b in range(B)]
    new[3] = new[200] = 0
    total = [n + (b * 37) % 200 for b, n in enumerate(new)]
    check(ops, make(new, total, 16, 1, 4, 64, torch.bfloat16), max_q_len=max_q_len)


def test_overlapping_sequences_are_safe(ops):
    """Offsets that run backwards make sequences overlap, more rows than the tensors
    have: nothing is written out of range, and the error is reported."""
    new, total, page = [400, 30, 400], [400, 30, 400], 16
    q, kp, vp, table, cu, lens = make(new, total, page, 2, 2, 128, torch.bfloat16, pad=0)
    n = q.shape[0]
    cu.copy_(torch.tensor([0, n, 0, n], dtype=torch.int32))
    lens.fill_(int(table.shape[1]) * page)
    table.clamp_(min=0)
    room = torch.full((n + 64, *q.shape[1:]), 7.0, device="cuda", dtype=q.dtype)
    ops.paged_attention(q, kp, vp, table, cu, lens, max_q_len=n, out=room[32:32 + n])
    assert device_error() == 8
    assert bool((room[:32] == 7).all()) and bool((room[32 + n:] == 7).all())


@pytest.mark.parametrize("max_q_len", [None, 1, 2])
@pytest.mark.parametrize("new, group, dim", [([0, 1], 40, 128), ([1, 0, 0, 1], 64, 128), ([0, 1], 33, 72),
                                             ([0, 2], 33, 128), ([0, 1], 70, 64), ([0, 1, 0], 128, 128)], ids=str)
def test_fewer_tokens_than_sequences_and_wide_groups(ops, new, group, dim, max_q_len):
    """Single tokens whose group alone is too many rows for the kernel of few rows."""
    total = [40 + 300 * i for i in range(len(new))]
    check(ops, make(new, total, 16, 1, group, dim, torch.bfloat16, pad=0), max_q_len=max_q_len)


def test_expanded_outputs_are_refused(ops):
    q, kp, vp, table, cu, lens = make([2, 1], [20, 9], 16, 2, 2, 64, torch.bfloat16)
    f = torch.ones(8, device="cuda")
    pos = torch.zeros(q.shape[0], dtype=torch.int64, device="cuda")
    same = torch.zeros_like(q[:, :1]).expand_as(q)
    with pytest.raises(ValueError):
        ops.rope(q, pos, f, out=same)
    with pytest.raises(ValueError):
        ops.paged_attention(q, kp, vp, table, cu, lens, out=same)
    with pytest.raises(ValueError):
        ops.paged_kv_append(q[:, :2], q[:, :2], kp[:1].expand_as(kp), vp, table, cu, lens)
    # expanded inputs are fine
    one = q[:, :1].expand_as(q)
    assert torch.equal(ops.rope(one, pos + 3, f), ops.rope(one.contiguous(), pos + 3, f))
    n, used = int(cu[-1]), table[0, :1].long()
    shared = kp[used].nan_to_num(0.5).expand_as(kp)  # one page under every index
    for most in (2, 100):
        got = ops.paged_attention(one, shared, vp, table, cu, lens, max_q_len=most)[:n]
        want = ops.paged_attention(one.contiguous(), shared.contiguous(), vp, table, cu, lens, max_q_len=most)[:n]
        assert torch.equal(got, want)


def test_two_threads_at_once(ops):
    """Calls from several host threads, each on a stream of its own."""
    import threading
    cases = [ROWS[3], TILES[4], ROWS[4], TILES[3]]
    made = [make(*c, torch.bfloat16, seed=i) for i, c in enumerate(cases)]
    want = [ops.paged_attention(*a, max_q_len=max(c[0]))[:sum(c[0])].clone() for a, c in zip(made, cases)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = ops.paged_attention(*made[i], max_q_len=max(cases[i][0]))[:sum(cases[i][0])]
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
