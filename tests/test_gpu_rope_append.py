"""GPU: rotary positions and the append to a paged cache, against plain
implementations in 64 bits.

Tolerances, derived from the arithmetic: the result of a pair is
f (a cos - b sin) with |value| <= 1.0 * f * (|a| + |b|). In fp32, cos and sin are
within 2 ulp (2^-22 relative to 1) of exact, the angle's reduced fraction is rounded to
2^-25 of a turn at most (2 pi 2^-25 < 2^-22 radians), the scaling by f and the
products and their sum add 2^-24 each: below 2^-20 f (|a| + |b|) together. Then one
rounding to the type, half a step: eps / 2 of the value.
"""
import numpy as np
import pytest

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


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rotate64(x, angle, interleaved, factor):
    """(rotated x in 64 bits, |a| + |b| of each value's pair); angle [..., pairs]."""
    x = x.double()
    r = 2 * angle.shape[-1]
    out, size = x.clone(), torch.zeros_like(x)
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[..., first], x[..., second]
    out[..., first] = factor * (a * angle.cos() - b * angle.sin())
    out[..., second] = factor * (b * angle.cos() + a * angle.sin())
    size[..., first] = size[..., second] = abs(factor) * (a.abs() + b.abs())
    return out, size


def check_rotated(got, x, angle, interleaved, factor):
    want, size = rotate64(x, angle, interleaved, factor)
    room = torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -20 * size
    if x.dtype == torch.float16:
        room += 2.0 ** -25  # half a step of its subnormals
    assert bool(((got.double() - want).abs() <= room).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 64, 64), (7, 5, 128, 128), (33, 3, 80, 40), (5, 9, 72, 36),
                                       (3, 2, 10, 6), (4, 1, 256, 64), (2, 2, 7, 2), (129, 24, 96, 48),
                                       (6, 4, 64, 0)])
def test_rope_packed(ops, dtype, interleaved, T, H, D, rot):
    g = gen(T * 1000 + D)
    x = torch.randn(T, H, D, device="cuda", generator=g).to(dtype)
    pos = torch.randint(-5, 1 << 20, (T,), device="cuda", generator=g)
    freq, _ = ops.rope_frequencies(rot, 10000.0)
    for factor in (1.0, 1.25):
        for f, sign in ((ops.rope, 1.0), (ops.rope_backward, -1.0)):
            y = f(x, pos, freq, interleaved=interleaved, factor=factor)
            angle = sign * pos.double()[:, None, None] * freq.double()
            check_rotated(y, x, angle, interleaved, factor)
            assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("per_batch", [False, True])
def test_rope_attention_layout_and_views(ops, interleaved, per_batch):
    B, H, S, D = 3, 5, 37, 128
    g = gen(2)
    wide = torch.randn(B, S, 2 * H * D, device="cuda", generator=g).bfloat16()
    x = wide[..., H * D:].view(B, S, H, D).transpose(1, 2)  # strided, 256-byte offset
    pos = torch.randint(0, 5000, (B, S) if per_batch else (S,), device="cuda", generator=g)
    freq, _ = ops.rope_frequencies(64)
    y = ops.rope(x, pos, freq, interleaved=interleaved)
    angle = (pos if per_batch else pos.expand(B, S)).double()[:, None, :, None] * freq.double()
    check_rotated(y, x, angle, interleaved, 1.0)
    before = wide.clone()
    assert ops.rope(x, pos, freq, interleaved=interleaved, out=x) is x  # in place
    assert torch.equal(x, y)
    assert torch.equal(wide[..., :H * D], before[..., :H * D])


def test_rope_unaligned_rows(ops):
    """Row strides and a base address that allow no wide access."""
    flat = torch.randn(7 * 3 * 67 + 1, device="cuda", generator=gen(3)).bfloat16()
    x = flat[1:].view(7, 3, 67)[..., :64]
    pos = torch.arange(7, device="cuda") * 999
    freq, _ = ops.rope_frequencies(64)
    check_rotated(ops.rope(x, pos, freq), x, pos.double()[:, None, None] * freq.double(), False, 1.0)


@pytest.mark.parametrize("far", [1 << 20, (1 << 31) - 1, -(1 << 31)])
def test_rope_far_positions(ops, far):
    """Angles keep their fraction at the far end of the documented range. The
    64-bit products round twice at 2^-53 of up to 2^31 radians: 2^-21."""
    x = torch.randn(4, 2, 64, device="cuda", generator=gen(4))
    pos = torch.full((4,), far, device="cuda") - torch.arange(4, device="cuda") * (1 if far > 0 else -1)
    freq, _ = ops.rope_frequencies(64, 1e6)
    y = ops.rope(x, pos, freq)
    rad = np.zeros((4, 32))
    two_pi = np.longdouble("6.28318530717958647692528676655900576")
    for i, p in enumerate(pos.tolist()):
        for j, f in enumerate(freq.double().tolist()):
            a = np.longdouble(p) * np.longdouble(f)  # 24 x 31 bits: exact in 64
            rad[i, j] = float(a - np.rint(a / two_pi) * two_pi)
    angle = torch.tensor(rad, device="cuda")[:, None, :]
    want, size = rotate64(x, angle, False, 1.0)
    assert bool(((y.double() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -19 * size).all())


def test_rope_gradient_against_differences(ops):
    """<g, rope(x + e d) - rope(x - e d)> / 2e = <rope_backward(g), d>: the map is
    linear, so differences have no truncation error."""
    g = gen(5)
    x, d, up = (torch.randn(9, 4, 48, device="cuda", generator=g) for _ in range(3))
    pos = torch.randint(0, 3000, (9,), device="cuda", generator=g)
    freq, factor = ops.rope_frequencies(32, scaling={"type": "yarn", "factor": 4.0, "original_length": 512})
    assert factor > 1
    kw = dict(interleaved=True, factor=factor)
    diff = (ops.rope(x + d, pos, freq, **kw).double() - ops.rope(x - d, pos, freq, **kw).double()) / 2
    left = (up.double() * diff).sum()
    right = (ops.rope_backward(up, pos, freq, **kw).double() * d.double()).sum()
    scale = (up.double().abs() * (x.abs() + d.abs()).double()).sum() * 2 * factor
    assert abs(float(left - right)) <= 2.0 ** -19 * float(scale)


def test_rope_empty(ops):
    freq, _ = ops.rope_frequencies(64)
    x = torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16)
    assert ops.rope(x, torch.empty(0, dtype=torch.int64, device="cuda"), freq).shape == x.shape


# ------------------------------------------------------------------ append --
def batch(new, total, page, spare=2, seed=0, width=None):
    """Page table (a random order of the pool's pages, -1 past each end), offsets, lengths, pool size."""
    need = [-(-t // page) for t in total]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(new), width or max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    cu = torch.tensor([0] + new).cumsum(0).int()
    return table.cuda(), cu.cuda(), torch.tensor(total, dtype=torch.int32).cuda(), sum(need) + spare


APPENDS = [
    # new, total, page, heads, q_heads, dim, rot
    ([1], [1], 16, 1, 1, 64, 64),
    ([1, 1, 1], [17, 1, 16], 16, 8, 32, 128, 128),
    ([5, 0, 33, 1], [5, 9, 40, 64], 8, 2, 6, 96, 48),
    ([130], [131], 64, 3, 3, 80, 80),
    ([3, 4], [30, 4], 7, 2, 2, 40, 20),     # a page size of no power of two
    ([2, 2], [3, 2], 1, 1, 5, 256, 64),     # pages of one row
    ([300, 7], [300, 2000], 128, 4, 4, 64, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", APPENDS)
def test_append(ops, dtype, interleaved, case):
    new, total, page, heads, q_heads, dim, rot = case
    g = gen(sum(total))
    table, cu, lens, pages = batch(new, total, page)
    n, pad = sum(new), 3
    both = torch.randn(n + pad, q_heads + 2 * heads, dim, device="cuda", generator=g).to(dtype)
    q, k, v = both.split([q_heads, heads, heads], dim=1)
    mark = float("nan")
    # token-major pools, passed as a transposed view
    kp = torch.full((pages, page, heads, dim), mark, device="cuda", dtype=dtype).transpose(1, 2)
    vp = torch.full((pages, heads, page, dim), mark, device="cuda", dtype=dtype)
    freq = ops.rope_frequencies(rot)[0] if rot else None
    q_out = torch.full_like(q, mark) if rot else None
    got = ops.paged_kv_append(k, v, kp, vp, table, cu, lens, inv_freq=freq, interleaved=interleaved,
                              q=q if rot else None, q_out=q_out)
    assert got is q_out
    kref, vref = torch.full_like(kp, mark), torch.full_like(vp, mark)
    t = 0
    for b, c in enumerate(new):
        pos = torch.arange(total[b] - c, total[b], device="cuda")
        at = table[b].long()[pos // page], slice(None), pos % page
        if rot:
            angle = pos.double()[:, None, None] * freq.double()
            check_rotated(kp[at], k[t:t + c], angle, interleaved, 1.0)
            check_rotated(q_out[t:t + c], q[t:t + c], angle, interleaved, 1.0)
            kref[at] = kp[at]
        else:
            kref[at] = k[t:t + c]
        vref[at] = v[t:t + c]
        t += c
    # every other row of the pools, and the rows of no sequence, as they were
    assert torch.equal(kp.contiguous().view(torch.int16), kref.contiguous().view(torch.int16))
    assert torch.equal(vp.view(torch.int16), vref.view(torch.int16))
    if rot:
        assert bool(q_out[n:].isnan().all())


def test_append_in_place_and_replayed(ops):
    """q rotated in place; a captured append follows the lengths it is replayed with."""
    new, total, page = [1, 1], [5, 40], 16
    table, cu, lens, pages = batch(new, [64, 64], page)
    lens.copy_(torch.tensor(total))
    g = gen(9)
    q0, k, v = (torch.randn(2, 4, 64, device="cuda", generator=g).bfloat16() for _ in range(3))
    kp, vp = (torch.zeros(pages, 4, page, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    freq, _ = ops.rope_frequencies(64)
    q = q0.clone()
    ops.paged_kv_append(k, v, kp, vp, table, cu, lens, inv_freq=freq, q=q, q_out=q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_kv_append(k, v, kp, vp, table, cu, lens, inv_freq=freq, q=q, q_out=q)
    for step in range(1, 4):
        lens += 1
        q.copy_(q0)
        graph.replay()
        for b in range(2):
            p = total[b] + step - 1
            angle = torch.tensor([[p]], device="cuda").double() * freq.double()
            check_rotated(q[b], q0[b], angle, False, 1.0)
            check_rotated(kp[table[b, p // page], :, p % page], k[b], angle, False, 1.0)


def test_append_many_sequences(ops):
    """More sequences than one block keeps the offsets of."""
    B, page = 2500, 8
    total = [1 + b % 9 for b in range(B)]
    table, cu, lens, pages = batch([1] * B, total, page)
    k, v = (torch.randn(B, 1, 8, device="cuda", generator=gen(i)).bfloat16() for i in (1, 2))
    kp, vp = (torch.zeros(pages, 1, page, 8, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    ops.paged_kv_append(k, v, kp, vp, table, cu, lens)
    pos = lens.long() - 1
    at = table.long()[torch.arange(B, device="cuda"), pos // page]
    assert torch.equal(kp[at, :, pos % page], k) and torch.equal(vp[at, :, pos % page], v)
