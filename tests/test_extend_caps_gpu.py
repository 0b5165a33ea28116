"""Capped scores of ft_extend far from the usual scales and caps, against the 64-bit oracle."""
import pytest
import torch

import extend_cases
from test_extend_gpu import DTYPES, Step

pytestmark = pytest.mark.gpu
FORMS = [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 64)]


def filled(scale, cap, d, part=0.3):
    """The queries' factor for which the scores' standard deviation is `part` of the cap (keys are N(0, 1))."""
    return part * cap / (scale * d ** 0.5)


def tight(dtype, out, absv, size, cap, d):
    """extend_cases.bounds with a tanh that is off by at most 2^-20 of its value, not of the cap.

    Up to |x| = 1 the fit is within 2^-24 of the value, and roundings of x (two), x^2, the sum (weighted with at most 0.3 each)
    and the last product make it less than 8 half steps, 2^-21.  Beyond, 2 / (1 + e^2x) is at most 0.24 and off by 2^-21 (the
    exponent function, its argument, the reciprocal) of itself, its difference from 1 >= 0.76 by another half step: 2^-22.  The
    factor cap log2(e) and the sum with the row's offset round twice more, which the rest of 2^-20 holds."""
    u = 2.0 ** -24 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    x = 2 * (d + 8) * 2.0 ** -24 * size + 2.0 ** -20 * size.clamp(max=cap)
    rel = torch.expm1(2 * x) + 2.0 ** -15
    return (u + rel)[..., None] * absv + u * (out.abs() + rel[..., None] * absv) + 1e-30, x + 2.0 ** -15


def near(s, scale, cap, bounds, path="auto"):
    o, lse = s.run(path, cap, scale)
    out, want, absv, size = extend_cases.oracle(s.q, s.k, s.v, s.table, s.seq, s.ext, scale, cap, s.window)
    tol, tol_lse = bounds(s.dtype, out, absv, size, cap, s.d)
    n = sum(s.ext)
    err, err_lse = (o[:n].double().cpu() - out[:n]).abs(), (lse[:n].double().cpu() - want[:n]).abs()
    assert bool((err <= tol[:n]).all()), (err / tol[:n]).max().item()
    assert bool((err_lse <= tol_lse[:n]).all()), (err_lse / tol_lse[:n]).max().item()


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("scale,cap", [(1 / 128, 30.0), (1 / 256, 50.0), (None, 200.0), (None, 500.0), (1 / 16, 1000.0), (1.0, 1e-3)])
def test_scores_that_fill_the_cap(dtype, d, scale, cap):
    scale = scale or d ** -0.5
    s = Step([400, 90, 290], [60, 90, 1], [([0, 2], 250)], 8, 2, d, DTYPES[dtype], q_scale=filled(scale, cap, d))
    near(s, scale, cap, extend_cases.bounds)


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("cap,part", [(1e4, 1e-4), (1e4, 0.05), (3e5, 1e-3), (1e30, 1e-30), (3e38, 1e-38)])
def test_caps_far_above_the_scores(dtype, d, cap, part):
    """As good as no cap, and as exact: the error goes by the scores, not by the cap."""
    s = Step([400, 90, 290], [60, 90, 1], [([0, 2], 250)], 8, 2, d, DTYPES[dtype], q_scale=filled(d ** -0.5, cap, d, part))
    near(s, d ** -0.5, cap, tight)


@pytest.mark.parametrize("dtype,d", FORMS)
def test_a_tiny_cap_and_zero_scores(dtype, d):
    """Every score is the cap, its negative, or 0: plain averages."""
    s = Step([200, 90], [30, 90], [], 8, 2, d, DTYPES[dtype])
    s.q[3], s.gq[3] = 0, 0
    near(s, d ** -0.5, 1e-20, extend_cases.bounds)
    near(s, d ** -0.5, 1e-42, extend_cases.bounds)


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("cap,part", [(30.0, 0.1), (30.0, 0.6), (1e4, 1e-4)])
def test_scores_out_of_sight_change_no_bit(dtype, d, cap, part):
    """Keys that a query does not see, beside keys that it sees: whatever they hold, its output stays the same bit by bit."""
    s = Step([400, 90, 290], [60, 90, 1], [([0, 2], 250)], 8, 2, d, DTYPES[dtype], q_scale=filled(d ** -0.5, cap, d, part))
    want, want_lse = s.run(cap=cap)
    keys = s.gk.clone()
    for value in (1000.0, float("inf"), float("nan"), -float("inf")):
        for hit in ([380], [381], [380, 381, 385]):
            s.gk.copy_(keys)
            rows = s.table[0, hit].long()
            s.gk[rows] = s.gk[rows] * value if abs(value) < 1e4 else value
            o, lse = s.run(cap=cap)
            seen_from = 60 - (400 - hit[0])                      # request 0's queries from here on see it
            n = sum(s.ext)
            same = [i for i in range(n) if not seen_from <= i < 60]
            assert torch.equal(o[same], want[same]) and torch.equal(lse[same], want_lse[same])


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("cap", [30.0, 1e4])
def test_what_other_kernels_leave_behind_changes_no_bit(dtype, d, cap):
    """Tiles of K are not filled behind their last token: a call repeats itself after kernels that left other bytes there."""
    s = Step([300, 311, 77], [60, 3, 77], [], 8, 2, d, DTYPES[dtype])
    n = sum(s.ext)
    want, want_lse = s.run(cap=cap)
    for other, fill in ((torch.float32, 1e30), (torch.float32, -0.007), (torch.bfloat16, 1e4), (torch.float16, 6e4)):
        left = Step([1500] * 8, [200] * 8, [], 8, 2, 128, other)
        left.gk.fill_(fill), left.gv.fill_(fill)
        left.gq.zero_()
        left.run()
        o, lse = s.run(cap=cap)
        assert torch.equal(o[:n], want[:n]) and torch.equal(lse[:n], want_lse[:n])
