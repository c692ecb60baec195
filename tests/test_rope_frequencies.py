"""CPU: the frequencies between the ends of the stretched ranges."""
import math

import pytest

torch = pytest.importorskip("torch")


def test_yarn_between_its_ends():
    """64 values, base 10^4, trained on 2048 tokens: pair 8.06 turns 32 times within
    them and pair 20.1 once, so the ramp over the index goes from 8 to 21."""
    from polykernel_b200 import ops
    full, _ = ops.rope_frequencies(64, 1e4, device="cpu")
    f, factor = ops.rope_frequencies(64, 1e4, {"type": "yarn", "factor": 8.0, "original_length": 2048}, device="cpu")
    for i in range(32):
        ramp = min(max((i - 8) / 13, 0.0), 1.0)
        want = 1e4 ** (-i / 32) * ((1 - ramp) + ramp / 8)
        assert math.isclose(f[i].item(), want, rel_tol=2.0 ** -23), i
    assert torch.equal(f[:9], full[:9]) and not torch.equal(f[9:10], full[9:10])
    assert math.isclose(factor, 1.2079441541679836)
    # other turns and a factor of one's own
    f, factor = ops.rope_frequencies(64, 1e4, {"type": "yarn", "factor": 4.0, "original_length": 4096, "beta_fast": 16,
                                               "beta_slow": 2, "attention_factor": 0.9}, device="cpu")
    low = math.floor(32 * math.log(4096 / (2 * math.pi * 16)) / math.log(1e4))
    high = math.ceil(32 * math.log(4096 / (2 * math.pi * 2)) / math.log(1e4))
    assert (low, high, factor) == (12, 21, 0.9)
    i = 16
    ramp = (i - low) / (high - low)
    assert math.isclose(f[i].item(), 1e4 ** (-i / 32) * ((1 - ramp) + ramp / 4), rel_tol=2.0 ** -23)
