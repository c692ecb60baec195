"""CPU: the argument checks of the rotary and paged-append entry points, and the frequencies."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from polykernel_b200 import ops
    return ops


def test_frequencies(ops):
    f, factor = ops.rope_frequencies(8, 10000.0, device="cpu")
    assert factor == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001]))
    linear, _ = ops.rope_frequencies(8, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(linear, f / 4)
    # ntk: the fastest pair is kept, the slowest divided by the factor
    ntk, _ = ops.rope_frequencies(8, scaling={"type": "ntk", "factor": 4.0}, device="cpu")
    assert ntk[0] == 1.0 and math.isclose(ntk[-1].item(), 0.001 / 4, rel_tol=1e-6)
    for kind in ({"type": "yarn", "factor": 8.0, "original_length": 2048},
                 {"type": "bands", "factor": 8.0, "original_length": 2048, "low": 1.0, "high": 4.0}):
        full, _ = ops.rope_frequencies(64, device="cpu")
        g, factor = ops.rope_frequencies(64, scaling=kind, device="cpu")
        ratio = full / g
        assert ratio[0] == 1.0 and math.isclose(ratio[-1].item(), 8.0, rel_tol=1e-5)
        assert bool((ratio.diff() >= -1e-5).all())
        assert math.isclose(factor, 0.1 * math.log(8.0) + 1 if kind["type"] == "yarn" else 1.0)
    # bands: 2 turns within the length is a third of the way from 1 to 4
    b, _ = ops.rope_frequencies(2, scaling={"type": "bands", "factor": 8.0, "original_length": 4 * math.pi,
                                            "low": 1.0, "high": 4.0}, device="cpu")
    assert math.isclose(b.item(), 1 / 3 + (2 / 3) / 8, rel_tol=1e-6)


@pytest.mark.parametrize("args", [(7, 1e4, None), (8, -1.0, None), (8, 1e4, {"type": "other"}),
                                  (8, 1e4, {"type": "linear", "factor": 0.0}),
                                  (2, 1e4, {"type": "ntk", "factor": 2.0}),
                                  (8, 1e4, {"type": "linear", "factor": 2.0, "beta": 1}),
                                  (8, 1e4, {"type": "bands", "factor": 2.0, "original_length": 8,
                                            "low": 4.0, "high": 4.0})])
def test_frequency_refusals(ops, args):
    with pytest.raises(ValueError):
        ops.rope_frequencies(*args, device="cpu")


def test_cpu_tensors_are_refused(ops):
    x = torch.zeros(2, 1, 8)
    f, _ = ops.rope_frequencies(8, device="cpu")
    with pytest.raises(ValueError):
        ops.rope(x, torch.zeros(2, dtype=torch.int64), f)
    with pytest.raises(ValueError):
        ops.rope(torch.zeros(8), torch.zeros(2, dtype=torch.int64), f)
    pool = torch.zeros(1, 1, 8, 8, dtype=torch.bfloat16)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_kv_append(x.bfloat16(), x.bfloat16(), pool, pool, i32[None], i32, i32)


def test_c_entry_refusals_without_a_device():
    """Rejected before any device work: cudaErrorInvalidValue (1); empty calls return 0."""
    from polykernel_b200 import _lib
    L = _lib.lib()
    one = ctypes.c_longlong * 3
    st = one(8, 8, 8)
    buf = ctypes.create_string_buffer(64)
    p = ctypes.addressof(buf)

    def rope(dtype=0, pairs=4, B=1, tokens=1, H=1, D=8, x=p, factor=1.0, strides=st):
        return L.pkb200_rope(x, p, dtype, p, 0, p, pairs, B, tokens, H, D, strides, strides,
                             ctypes.c_float(factor), 0, 0, None)

    assert [rope(B=0), rope(tokens=0), rope(H=0), rope(D=0, pairs=0)] == [0, 0, 0, 0]
    assert [rope(dtype=3), rope(pairs=5), rope(pairs=-1), rope(B=-1), rope(tokens=-1), rope(H=-1),
            rope(x=None), rope(factor=math.nan), rope(strides=None), rope(B=70000)] == [1] * 10

    def append(tokens=1, seqs=1, k=p, pairs=0, q_heads=0, factor=1.0, cu=p, **cache):
        c = dict(k=p, v=p, k_stride=st, v_stride=st, num_pages=1, heads=1, page_size=1, dim=8, dtype=0)
        c.update(cache)
        c = _lib.PagedCache(**c)
        b = _lib.PagedBatch(p, cu, p, 1, 1, seqs, tokens)
        return L.pkb200_paged_kv_append(ctypes.byref(c), ctypes.byref(b), k, st, p, st, None, None, None,
                                        None, q_heads, None, pairs, ctypes.c_float(factor), 0, None)

    assert [append(tokens=0), append(seqs=0)] == [0, 0]
    assert [append(tokens=-1), append(seqs=-1), append(k=None), append(pairs=2), append(pairs=5),
            append(q_heads=1), append(q_heads=-1), append(factor=math.inf), append(cu=None),
            append(dtype=2), append(heads=0), append(page_size=0), append(dim=0),
            append(num_pages=-1), append(k=None)] == [1] * 15
    assert L.pkb200_paged_kv_append(None, None, p, st, p, st, None, None, None, None, 0, None, 0,
                                    ctypes.c_float(1.0), 0, None) == 1


def test_wrong_batches_stay_in_range(tmp_path):
    """The kernels' index arithmetic over random, mostly wrong, batch descriptions."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = tmp_path / "paged_index_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-o", str(exe),
                    os.path.join(root, "tests", "cpp", "paged_index_test.cpp")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.startswith("ok"), out.stdout + out.stderr


def test_attention_c_entry_refusals_without_a_device():
    from polykernel_b200 import _lib
    L = _lib.lib()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    st3, st2 = (ctypes.c_longlong * 3)(64, 64, 64), (ctypes.c_longlong * 2)(64, 64)

    def run(q=p, out=p, hq=1, most=1, causal=1, window=0, scale=1.0, tokens=1, seqs=1, ws=p, q_st=st2,
            out_st=st2, width=1, **cache):
        c = dict(k=p, v=p, k_stride=st3, v_stride=st3, num_pages=1, heads=1, page_size=8, dim=64, dtype=0)
        c.update(cache)
        c = _lib.PagedCache(**c)
        b = _lib.PagedBatch(p, p, p, width, width, seqs, tokens)
        return L.pkb200_paged_attention(ctypes.byref(c), ctypes.byref(b), q, q_st, out, out_st, None, hq, most,
                                        causal, window, ctypes.c_float(scale), ws, 0, None)

    odd = (ctypes.c_longlong * 2)(64, 60)
    odd3 = (ctypes.c_longlong * 3)(64, 64, 63)
    assert [run(tokens=0), run(seqs=0)] == [0, 0]
    refused = [run(q=None), run(out=None), run(hq=0), run(hq=3, heads=2), run(most=-1), run(window=-1),
               run(window=5, causal=0), run(scale=0.0), run(scale=-1.0), run(scale=math.nan),
               run(scale=math.inf), run(tokens=-1), run(dim=60), run(dim=264), run(page_size=12),
               run(page_size=0), run(num_pages=0), run(dtype=2), run(q=p + 8), run(out=p + 2), run(k=p + 4),
               run(q_st=odd), run(out_st=odd), run(k_stride=odd3), run(v_stride=odd3), run(k=None),
               run(tokens=2 ** 30, hq=4, heads=1)]
    assert refused == [1] * len(refused)


def test_attention_python_checks(ops):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(1, 1, 8, 64, dtype=torch.bfloat16)
    i32 = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):  # CPU tensors
        ops.paged_attention(q, pool, pool, i32[None], torch.zeros(2, dtype=torch.int32), i32)
    with pytest.raises(ValueError):
        ops.paged_attention(q[0], pool, pool, i32[None], i32, i32)
