"""Failure detection of attention over a paged cache, without faulting a GPU: tiles
that arrive later than the blocks wait end the call with a status. The warps of
a block do not give up at one time (a tile can land between two warps' looks at
it), and none may be left behind at a barrier that another one never reaches."""
import pytest

from tests.test_gpu_paged_attention import ROWS, make

torch = pytest.importorskip("torch")


def test_limits_are_checked():
    from polykernel_b200._lib import lib
    for bad in ((-1, 0), (0, -1), (10 ** 12, 0), (0, 10 ** 12)):
        assert lib().pkb200_selftest_paged_limits(*bad) != 0
    assert lib().pkb200_selftest_paged_limits(0, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("case", [ROWS[1], ROWS[4], ROWS[5], ROWS[10]], ids=str)
def test_late_tiles_end_the_call(cuda, case):
    import polykernel_b200 as pk
    lib = pk.lib()
    args = make(*case, torch.bfloat16)
    n, most = sum(case[0]), max(case[0])
    want = pk.ops.paged_attention(*args, max_q_len=most)[:n].clone()
    torch.cuda.synchronize()
    assert pk.device_error() == 0
    limit = 100_000  # ~50 us
    codes = []
    try:
        # far later (a look at a barrier may itself last a millisecond), and
        # nearer the limit, where some warps still get their tile
        for hold in [400 * limit] * 3 + [int(limit / 2 * 1.1 ** i) for i in range(60)]:
            assert lib.pkb200_selftest_paged_limits(limit, hold) == 0
            got = pk.ops.paged_attention(*args, max_q_len=most)[:n]
            torch.cuda.synchronize()
            codes.append(pk.device_error())
            assert codes[-1] in (0, 1, 4)
            if codes[-1] == 0:
                assert torch.equal(got, want)
    finally:
        lib.pkb200_selftest_paged_limits(0, 0)
    assert codes[:3] == [4] * 3
    assert torch.equal(pk.ops.paged_attention(*args, max_q_len=most)[:n], want)
    assert pk.device_error() == 0


@pytest.mark.gpu
def test_going_over_values_again_is_no_late_tile(cuda):
    """Where values are not finite, blocks go over a run's values once more, for
    longer than a wait may last: the fetching warp's limit runs anew meanwhile."""
    import math

    import polykernel_b200 as pk
    lib = pk.lib()
    B, total, page = 40, 8000, 64
    q, kp, vp, table, cu, lens = args = make([1] * B, [total] * B, page, 4, 4, 128, torch.bfloat16)
    vp[table[:, 0].long(), :, 5, 3] = math.inf
    vp[table[:, 90].long(), :, 0, 70] = -math.inf
    want = pk.ops.paged_attention(*args, max_q_len=1)[:B].clone()
    assert bool((want[..., 3] == math.inf).all()) and bool((want[..., 70] == -math.inf).all())
    assert int((~torch.isfinite(want)).sum()) == 2 * want.shape[0] * want.shape[1]
    try:
        assert lib.pkb200_selftest_paged_limits(200_000, 0) == 0  # ~0.1 ms
        for _ in range(3):
            got = pk.ops.paged_attention(*args, max_q_len=1)[:B]
            torch.cuda.synchronize()
            assert pk.device_error() == 0 and torch.equal(got, want)
    finally:
        lib.pkb200_selftest_paged_limits(0, 0)
