"""Beams whose scores are the largest and lowest that fp32 holds."""
import math

import pytest
import torch

from beam_cases import check, inputs

gpu = pytest.mark.gpu


@gpu
def test_a_beam_whose_score_is_the_lowest_is_live():
    logits, scores, _ = inputs(3, 2, 500, torch.float32, seed=1)
    scores[0, 0] = scores[1, 0] = torch.finfo(torch.float32).min
    scores[2, 0] = torch.finfo(torch.float32).max
    logits[1, 1, 2:] = -math.inf
    check(logits, scores, 8)


@gpu
def test_beams_of_the_lowest_score_alone():
    # fp32 rounds all of these scores to one value; the lowest beam comes first, and of its tokens the larger logit
    logits, scores, _ = inputs(2, 8, 3001, torch.bfloat16, seed=4)
    scores[:] = torch.finfo(torch.float32).min
    scores[1, 3:] = -math.inf
    for best in (5, 64):
        check(logits, scores, best)
    check(logits[..., :30], scores, 64)         # some beams list fewer tokens than results
    check(logits[..., :5], scores, 64)          # all of them together do


@gpu
@pytest.mark.parametrize("far", [1e9, 1e20, 3e38])
def test_scores_far_from_one_another(far):
    logits, scores, _ = inputs(4, 6, 900, torch.float32, seed=5)
    scores[0, ::2], scores[1, ::2], scores[2] = -far, far, -far
    scores[3] = torch.linspace(-far, far, 6)
    for best in (3, 40):
        check(logits, scores, best)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sums_below_all_of_fp32(dtype):
    # logit and score are fp32's own, their sum is not: such a token comes last, and its score rounds to -inf
    logits, scores, _ = inputs(2, 3, 8, dtype, seed=7)
    logits[:, :, 1::4] = -2e38
    scores[0, 0] = -2e38
    scores[1] = -2e38
    for best in (20, 64):
        check(logits, scores, best)
