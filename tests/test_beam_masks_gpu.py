"""Beam selection of logits of any size against the definition in 64 bits: masks of a type's lowest value and of other large values, rows of
nothing else, single large logits."""
import math

import pytest
import torch

from beam_cases import check, inputs

gpu = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
MASKS = [(name, mask) for name in ("bf16", "fp32") for mask in ("min", -1e9, -1e10, -1e20, -1e30)] + [("fp16", "min"), ("fp16", -6e4)]


def value(name, mask):
    return torch.finfo(DTYPES[name]).min if mask == "min" else mask


@gpu
@pytest.mark.parametrize("name,mask", MASKS)
@pytest.mark.parametrize("vocab,best", [(61, 8), (6001, 8), (70000, 4), (70000, 40)])
@pytest.mark.parametrize("kept", [1, 5, 1000])
def test_all_tokens_but_a_few_are_masked(name, mask, vocab, best, kept):
    logits, scores, g = inputs(3, 3, vocab, DTYPES[name], seed=vocab + kept)
    for r in range(3):
        for b in range(3):
            banned = torch.ones(vocab, dtype=torch.bool)
            banned[torch.randperm(vocab, generator=g)[:kept]] = False
            logits[r, b, banned] = value(name, mask)
    check(logits, scores, best)


@gpu
@pytest.mark.parametrize("name,mask", MASKS)
@pytest.mark.parametrize("best", [4, 24])
def test_stretches_and_whole_rows_are_masked(name, mask, best):
    vocab = 50021
    logits, scores, _ = inputs(5, 4, vocab, DTYPES[name], seed=best)
    masked = value(name, mask)
    logits[0, :, :vocab // 2] = masked          # nothing else in the first chunks
    logits[1, :, vocab // 2:] = masked          # nothing else in the last ones
    logits[2, 1], logits[2, 3] = masked, masked  # beams of nothing else
    logits[3] = masked                          # a request of nothing else
    logits[4, 0, 300:900], logits[4, 1, 7:], logits[4, 2, :-2], logits[4, 3] = masked, masked, masked, -math.inf
    check(logits, scores, best)


@gpu
@pytest.mark.parametrize("name", sorted(DTYPES))
def test_fewer_tokens_than_results_are_left(name):
    # three ordinary logits; masked tokens follow them among the results, banned ones do not
    lowest = torch.finfo(DTYPES[name]).min
    for rest in (lowest, -math.inf):
        for vocab in (9, 3001):
            logits, scores = torch.full((2, 1, vocab), rest, dtype=DTYPES[name]), torch.tensor([[-3.0], [0.0]])
            logits[:, 0, [1, 5, vocab - 1]] = torch.tensor([0.5, -1.0, 2.0], dtype=DTYPES[name])
            check(logits, scores, 8)
    # more equal results than the merge lists
    check(torch.full((1, 64, 70), lowest, dtype=DTYPES[name]), torch.zeros(1, 64) - 1, 64)


@gpu
@pytest.mark.parametrize("name,big", [(n, b) for n in ("bf16", "fp32") for b in (2e6, 3e8, 1.2e9, 3e9, 1e12, 1e30, "max")] + [("fp16", "max")])
@pytest.mark.parametrize("beams", [1, 3])
def test_single_large_logits(name, big, beams):
    big = torch.finfo(DTYPES[name]).max if big == "max" else big
    for vocab in (50, 6007):
        logits, scores, _ = inputs(4, beams, vocab, DTYPES[name], seed=vocab)
        scores[:, 0] = 4.0
        logits[0, 0, 7] = big
        logits[1, 0, vocab - 1] = big
        logits[1, 0, 3] = -big
        logits[2, 0] = big
        logits[3, :, 5:9] = big
        check(logits, scores, 6)


@gpu
@pytest.mark.parametrize("spread", [1e3, 1e6, 1e9, 1e18])
def test_widely_spread_logits(spread):
    logits, scores, _ = inputs(3, 4, 20011, torch.float32, seed=2)
    check(logits * spread, scores, 10)
    check((logits * spread).bfloat16(), scores, 10)
    check(logits * spread - 5 * spread, scores, 10)


@gpu
@pytest.mark.parametrize("name", sorted(DTYPES))
def test_scores_of_rising_logits_and_of_lists_that_overflow(name):
    vocab = 90001
    rising = torch.linspace(-20, 20, vocab).to(DTYPES[name])
    plateau = torch.where(torch.arange(vocab) % 3 == 0, torch.tensor(4.0), torch.tensor(-3.0)).to(DTYPES[name])
    logits = torch.stack([rising, plateau, rising.flip(0)]).repeat(2, 1).view(2, 3, vocab)
    scores = torch.linspace(-3, 0, 6).view(2, 3)
    for best in (1, 8, 64):
        check(logits, scores, best)


@gpu
def test_nan_and_infinities_stay_with_their_beam():
    for dtype in DTYPES.values():
        logits, scores, _ = inputs(3, 3, 9001, dtype, seed=3)
        logits[0, 0, 17], logits[0, 1] = math.inf, torch.finfo(dtype).min
        logits[1, 0, 8000], logits[1, 2, :8500] = float("nan"), torch.finfo(dtype).min
        logits[2, 1, 4], logits[2, 1, 9000] = torch.finfo(dtype).min, math.inf
        check(logits, scores, 12)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_below_all_of_fp32(dtype):
    # logit and score are fp32's own, their sum is not: such a token comes last, and its score rounds to -inf
    logits, scores, _ = inputs(2, 3, 40, dtype, seed=6)
    logits[:, :, 3:] = -2e38
    scores[:, 0] = -2e38
    scores[1] = -2e38
    for best in (8, 64):
        check(logits, scores, best)
