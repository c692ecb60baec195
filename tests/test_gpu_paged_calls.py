"""GPU: what the calls of the paged operators take and refuse, beyond shapes and types."""
import pytest

from tests.test_gpu_paged_attention import ROWS, TILES, make
from tests.test_gpu_rope_append import batch, check_rotated, gen

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


def bf16(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=gen(seed)).bfloat16()


def test_outputs_that_overlap_inputs_are_refused(ops):
    """Threads read rows that others write: an output is the input itself, or apart from it."""
    f, _ = ops.rope_frequencies(64)
    pos = torch.arange(9, device="cuda")
    buf = bf16(10 * 4 * 64)
    x = buf[:9 * 256].view(9, 4, 64)
    with pytest.raises(ValueError, match="overlaps"):
        ops.rope(x, pos, f, out=buf[256:].view(9, 4, 64))  # one row further
    with pytest.raises(ValueError, match="overlaps"):
        ops.rope(x, pos, f, out=buf[8:8 + 9 * 256].view(9, 4, 64))
    with pytest.raises(ValueError, match="overlaps"):
        ops.rope(x, pos, f, out=buf[:9 * 256].view(4, 9, 64).transpose(0, 1))
    new, total, page = [2, 1], [20, 9], 16
    table, cu, lens, pages = batch(new, total, page)
    both = bf16(3, 8 + 4, 64)
    q, k, v = both.split([8, 2, 2], dim=1)
    kp, vp = bf16(pages, 2, page, 64, seed=1), bf16(pages, 2, page, 64, seed=2)
    append = (k, v, kp, vp, table, cu, lens)
    for q_out in (both[:, 1:9], both[:, 2:10], both[:, 4:]):
        with pytest.raises(ValueError, match="overlaps"):
            ops.paged_kv_append(*append, inv_freq=f, q=q, q_out=q_out)
    with pytest.raises(ValueError, match="overlaps"):
        ops.paged_kv_append(k, v, kp, kp, table, cu, lens)
    with pytest.raises(ValueError, match="overlaps"):
        ops.paged_kv_append(kp.view(-1, 2, 64)[:3], v, kp, vp, table, cu, lens)
    qc = q.contiguous()
    more = bf16(4, 8, 64)
    for out in (more[1:], kp.view(-1, 8, 64)[:3]):
        with pytest.raises(ValueError, match="overlaps"):
            ops.paged_attention(more[:3] if out.data_ptr() != kp.data_ptr() else qc, kp, vp, table, cu, lens, out=out)


def test_outputs_in_the_gaps_of_inputs(ops):
    """Slices of one buffer that share no value are taken."""
    f, _ = ops.rope_frequencies(64)
    pos = torch.arange(9, device="cuda")
    buf = bf16(9, 8, 128)
    want = ops.rope(buf[:, :4, :64], pos, f)
    got = ops.rope(buf[:, :4, :64], pos, f, out=buf[:, 4:, 64:])
    assert torch.equal(got, want)
    # pools that alternate in one tensor, and q rotated in place beside k and v
    new, total, page = [2, 1], [20, 9], 16
    table, cu, lens, pages = batch(new, total, page)
    both = bf16(3, 8 + 4, 64)
    q, k, v = both.split([8, 2, 2], dim=1)
    apart = [torch.zeros(pages, 2, page, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    want = ops.paged_kv_append(k, v, *apart, table, cu, lens, inv_freq=f, q=q).clone()
    pool = torch.zeros(pages, 2, 2, page, 64, device="cuda", dtype=torch.bfloat16)
    got = ops.paged_kv_append(k, v, pool[:, 0], pool[:, 1], table, cu, lens, inv_freq=f, q=q, q_out=q)
    assert got is q and torch.equal(q, want)
    assert torch.equal(pool[:, 0], apart[0]) and torch.equal(pool[:, 1], apart[1])


@pytest.mark.parametrize("case", [ROWS[4], ROWS[11], TILES[4], TILES[6]], ids=str)
def test_attention_in_place_of_q(ops, case):
    q, *rest = make(*case, torch.bfloat16)
    n = sum(case[0])
    want = ops.paged_attention(q, *rest, max_q_len=max(case[0]))[:n].clone()
    assert ops.paged_attention(q, *rest, max_q_len=max(case[0]), out=q) is q
    assert torch.equal(q[:n], want)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_with_a_factor(ops, dtype, interleaved):
    """The factor on cos and sin reaches k and q in the cache's append."""
    new, total, page = [3, 1], [20, 70], 16
    table, cu, lens, pages = batch(new, total, page)
    g = gen(8)
    q, k, v = (torch.randn(4, h, 96, device="cuda", generator=g).to(dtype) for h in (6, 2, 2))
    kp, vp = (torch.zeros(pages, 2, page, 96, device="cuda", dtype=dtype) for _ in range(2))
    freq, factor = ops.rope_frequencies(64, scaling={"type": "yarn", "factor": 8.0, "original_length": 64})
    assert factor > 1.2
    got = ops.paged_kv_append(k, v, kp, vp, table, cu, lens, inv_freq=freq, interleaved=interleaved, factor=factor, q=q)
    pos = torch.tensor([17, 18, 19, 69], device="cuda")
    at = table[[0, 0, 0, 1], pos // page].long(), slice(None), pos % page
    angle = pos.double()[:, None, None] * freq.double()
    check_rotated(got, q, angle, interleaved, factor)
    check_rotated(kp[at], k, angle, interleaved, factor)
    assert torch.equal(got[..., 64:], q[..., 64:]) and torch.equal(kp[at][..., 64:], k[..., 64:])
    assert torch.equal(vp[at], v)
