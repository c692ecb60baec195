"""GPU: `ops.rope` as a step of autograd. The map is linear, so its gradient is the
map of the opposite angles: compared with the 64-bit formula under the tolerance of
test_gpu_rope_append.py, and with `ops.rope_backward` to the bit."""
import pytest

from tests.test_gpu_rope_append import check_rotated, gen

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops(cuda):
    from polykernel_b200 import ops
    return ops


def inputs(ops, shape, dtype, rot=48):
    g = gen(sum(shape))
    x, up = (torch.randn(*shape, device="cuda", generator=g).to(dtype) for _ in range(2))
    S = shape[0] if len(shape) == 3 else shape[2]
    pos = torch.randint(0, 9000, (S,), device="cuda", generator=g)
    return x, up, pos, ops.rope_frequencies(rot)[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", [(9, 4, 64), (1, 1, 48), (2, 3, 17, 96)])
def test_gradient(ops, dtype, interleaved, shape):
    x, up, pos, freq = inputs(ops, shape, dtype)
    kw = dict(interleaved=interleaved, factor=1.25)
    leaf = x.clone().requires_grad_()
    y = ops.rope(leaf, pos, freq, **kw)
    assert torch.equal(y, ops.rope(x, pos, freq, **kw))
    y.backward(up)
    at = pos if len(shape) == 4 else pos[:, None]
    check_rotated(leaf.grad, up, -at.double()[..., None] * freq.double(), interleaved, 1.25)
    assert torch.equal(leaf.grad, ops.rope_backward(up, pos, freq, **kw))


def test_gradient_of_a_sum_and_of_views(ops):
    """Gradients arrive expanded from a sum, and strided through a transpose."""
    x, up, pos, freq = inputs(ops, (2, 17, 3, 96), torch.float32)
    pos = pos[:1].expand(17)
    leaf = x.clone().requires_grad_()
    with pytest.raises(ValueError):  # positions are one per token, side by side
        ops.rope(leaf.transpose(1, 2), pos, freq)
    pos = pos.contiguous()
    y = ops.rope(leaf.transpose(1, 2), pos, freq)
    (y.sum() + (y.transpose(1, 2) * up).sum()).backward()
    want = ops.rope_backward((up + 1).transpose(1, 2), pos, freq).transpose(1, 2)
    assert torch.equal(leaf.grad, want)


def test_second_gradient(ops):
    x, up, pos, freq = inputs(ops, (9, 4, 64), torch.float32)
    leaf, weight = x.clone().requires_grad_(), up.clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.rope(leaf, pos, freq), leaf, weight, create_graph=True)
    (back,) = torch.autograd.grad(g, weight, x)
    assert torch.equal(back, ops.rope(x, pos, freq))


def test_without_gradients_and_refusals(ops):
    x, up, pos, freq = inputs(ops, (9, 4, 64), torch.bfloat16)
    leaf = x.clone().requires_grad_()
    with torch.no_grad():
        assert not ops.rope(leaf, pos, freq).requires_grad
    with pytest.raises(ValueError):
        ops.rope(leaf, pos, freq, out=torch.empty_like(x))
    with pytest.raises(ValueError):
        ops.rope(x, pos, freq.clone().requires_grad_())
    y = ops.rope(leaf, pos, freq)
    pos += 1  # what the gradient needs is not to change before it is taken
    with pytest.raises(RuntimeError):
        y.backward(up)


def test_captured_step(ops):
    """Forward and gradient on another stream, captured and replayed with new inputs."""
    x, up, pos, freq = inputs(ops, (9, 4, 64), torch.bfloat16)
    leaf = x.clone().requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(ops.rope(leaf, pos, freq), leaf, up)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (g,) = torch.autograd.grad(ops.rope(leaf, pos, freq), leaf, up)
    up.mul_(2)
    pos.add_(5)
    graph.replay()
    assert torch.equal(g, ops.rope_backward(up, pos, freq))
