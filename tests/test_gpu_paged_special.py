"""GPU: attention over a paged cache whose values are not finite, against the
definition in 64 bits (tolerances: test_gpu_paged_attention.py). Weights of visible keys
are positive, however small, so an infinite value gives an infinity of its sign,
infinities of both signs NaN, and log-sums do not depend on values."""
import math

import pytest

from tests.test_gpu_paged_attention import ROWS, TILES, definition, make

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


def compare(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isposinf(), want.isposinf())
    assert torch.equal(got.isneginf(), want.isneginf())
    fine = torch.isfinite(want)
    far = (got.double() - want).abs()[fine] / tol[fine].clamp(min=1e-300)
    assert bool((far <= 1).all()), float(far.max())


def spoil(vp, table, new, total, page, places):
    """Values that are not finite at those fractions of each sequence's keys, in columns of their own and shared ones."""
    inf = math.inf
    for b, t in enumerate(total):
        for place in places:
            for step, (bad, columns) in enumerate([(inf, slice(0, None, 3)), (-inf, slice(1, None, 5)),
                                                   (float("nan"), slice(2, 3))]):
                key = min(t - 1, int(place * t) + step)
                if new[b] and t > 4:
                    vp[table[b, key // page], :, key % page, columns] = bad


@pytest.mark.parametrize("places", [[0.0], [0.4], [0.97], [0.1, 0.5, 0.999]], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", [ROWS[1], ROWS[2], ROWS[4], ROWS[5], ROWS[7], ROWS[8], ROWS[9], ROWS[11],
                                  TILES[1], TILES[2], TILES[4], TILES[5], TILES[6], TILES[8], TILES[9]], ids=str)
def test_infinite_values(ops, case, dtype, places):
    q, kp, vp, table, cu, lens = args = make(*case, dtype)
    spoil(vp, table, case[0], case[1], case[2], places)
    n = sum(case[0])
    # scores that differ by up to hundreds: weights that 16 bits, and 32, round to 0
    for scale in (None, 1.0, 4.0):
        want, wl, tol, ltol = definition(*args, scale=scale)
        out, lse = ops.paged_attention(*args, max_q_len=max(case[0]), scale=scale, return_lse=True)
        compare(out[:n], want[:n], tol[:n])
        compare(lse[:n], wl[:n], ltol[:n])


@pytest.mark.parametrize("max_q_len", [None, 1])
@pytest.mark.parametrize("case", [ROWS[4], ROWS[5], ROWS[11], TILES[4]], ids=str)
def test_infinite_values_windows_and_any_kernel(ops, case, max_q_len):
    q, kp, vp, table, cu, lens = args = make(*case, torch.bfloat16)
    spoil(vp, table, case[0], case[1], case[2], [0.0, 0.93, 0.98])
    n = sum(case[0])
    for kw in (dict(window=40), dict(window=300), dict(causal=False)):
        want, wl, tol, ltol = definition(*args, **kw)
        out, lse = ops.paged_attention(*args, max_q_len=max_q_len, return_lse=True, **kw)
        compare(out[:n], want[:n], tol[:n])
        compare(lse[:n], wl[:n], ltol[:n])


@pytest.mark.parametrize("case", [ROWS[1], ROWS[4], ROWS[11], TILES[2], TILES[4]], ids=str)
def test_infinite_keys_and_values(ops, case):
    """A key that scores -inf has weight 0, and 0 * inf is NaN; one that scores
    inf leaves its rows NaN."""
    q, kp, vp, table, cu, lens = args = make(*case, torch.bfloat16)
    for b, (c, t) in enumerate(zip(case[0], case[1])):
        for key in ({t // 3, t - 1 - c // 2} if c else ()):
            at = table[b, key // case[2]], slice(None), key % case[2]
            kp[at] = 0.0
            kp[(*at, 0)] = math.inf  # a score of the sign of the query's first value
            vp[(*at, slice(0, 7))] = math.inf
    n = sum(case[0])
    out = ops.paged_attention(*args, max_q_len=max(case[0]))[:n]
    want = definition(*args)[0][:n]
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.isinf(), want.isinf())


def test_queries_that_are_not_finite(ops):
    """A row whose scores are NaN is NaN, and no other."""
    for case in (ROWS[4], TILES[4]):
        args = make(*case, torch.bfloat16)
        args[0][1] = float("nan")
        n = sum(case[0])
        want, wl, tol, ltol = definition(*args)
        out, lse = ops.paged_attention(*args, max_q_len=max(case[0]), return_lse=True)
        compare(out[:n], want[:n], tol[:n])
        compare(lse[:n], wl[:n], ltol[:n])


def test_one_infinite_value_in_a_long_context(ops):
    """The last of many new tokens has an infinite value: its column is infinite
    for that token alone, and finding that out takes no more than going over the
    values again (a row formed key by key would take hundreds of times the call's own time)."""
    case = ([256], [30000], 64, 32, 1, 128)
    q, kp, vp, table, cu, lens = args = make(*case, torch.bfloat16, pad=0)
    last = 29999
    at = table[0, last // 64], 3, last % 64, 17

    def run():
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        out = ops.paged_attention(*args, max_q_len=256)
        end.record()
        end.synchronize()
        return out, start.elapsed_time(end)

    clean, _ = run()
    usual = min(run()[1] for _ in range(3))
    vp[at] = math.inf
    out, _ = run()
    longer = min(run()[1] for _ in range(3))
    want = clean.clone()
    want[255, 3, 17] = math.inf
    # (in that tile the value was part of no sum, so all others are as they were but
    # for the clean value's own share)
    same = out == want
    same[255, 3, 17] = bool(out[255, 3, 17] == math.inf)
    assert bool(same.all())
    assert longer < 20 * usual, (longer, usual)


@pytest.mark.parametrize("gone", [-1, 2 ** 31 - 1])
@pytest.mark.parametrize("window", [1, 40, 200])
@pytest.mark.parametrize("case", [ROWS[1], ROWS[4], ROWS[5], ROWS[8], ROWS[10], ROWS[11], TILES[4], TILES[5],
                                  TILES[6], TILES[8]], ids=str)
def test_pages_behind_the_window_may_be_gone(ops, case, window, gone):
    """A server that frees pages which no new token's window reaches marks them in
    the table: that is no error, and changes nothing (the fixture checks the error word)."""
    q, kp, vp, table, cu, lens = args = make(*case, torch.bfloat16)
    n, page = sum(case[0]), case[2]
    freed = table.clone()
    for b, (c, t) in enumerate(zip(case[0], case[1])):
        freed[b, :max(0, t - c - window + 1) // page] = gone
    kw = dict(max_q_len=max(case[0]), window=window, return_lse=True)
    out, lse = ops.paged_attention(q, kp, vp, freed, cu, lens, **kw)
    want, wl, tol, ltol = definition(*args, window=window)
    compare(out[:n], want[:n], tol[:n])
    compare(lse[:n], wl[:n], ltol[:n])


@pytest.mark.parametrize("case", [ROWS[4], TILES[4]], ids=str)
def test_pages_that_the_window_reaches_may_not(ops, case):
    import polykernel_b200 as pk
    q, kp, vp, table, cu, lens = make(*case, torch.bfloat16)
    c, t, page = case[0][2], case[1][2], case[2]
    table[2, max(0, t - c - 100 + 1) // page] = -1
    ops.paged_attention(q, kp, vp, table, cu, lens, max_q_len=max(case[0]), window=100)
    assert pk.device_error() == 8


@pytest.mark.parametrize("case", ROWS + TILES, ids=str)
def test_log_sums(ops, case):
    """Log-sums are finite where the definition's are (a NaN would pass a
    comparison that leaves NaN out), for every shape."""
    args = make(*case, torch.bfloat16)
    n = sum(case[0])
    want, wl, tol, ltol = definition(*args)
    out, lse = ops.paged_attention(*args, max_q_len=max(case[0]), return_lse=True)
    compare(lse[:n], wl[:n], ltol[:n])
    compare(out[:n], want[:n], tol[:n])
