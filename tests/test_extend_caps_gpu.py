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
def test_a_tiny_cap_and_zero_scores(dtype, d):
    """Every score is the cap, its negative, or 0: plain averages."""
    s = Step([200, 90], [30, 90], [], 8, 2, d, DTYPES[dtype])
    s.q[3], s.gq[3] = 0, 0
    near(s, d ** -0.5, 1e-20, extend_cases.bounds)
    near(s, d ** -0.5, 1e-42, extend_cases.bounds)
