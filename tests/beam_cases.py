"""The 64-bit oracle of beam selection for logits and scores of any size, and a call held to it."""
import math

import numpy as np
import torch

import fasttree
from ft_b200 import lib


def want(logits, scores, best):
    """Scores in 64 bits (from the largest logit, which may dwarf a logarithm), beams and tokens: of equal scores the lowest beam,
    then the larger logit, then the lowest token."""
    x, s = logits.double().cpu(), scores.double().cpu()
    top = x.amax(-1, keepdim=True)
    score = s[..., None] + ((x - top) - (x - top).exp().sum(-1, keepdim=True).log())
    score = torch.where(torch.isfinite(score) & (x > -math.inf), score, torch.full_like(score, -math.inf))
    batch, beams, vocab = x.shape
    out, ob, ot = torch.full((batch, best), -math.inf, dtype=torch.float64), torch.full((batch, best), -1), torch.full((batch, best), -1)
    beam, token = np.divmod(np.arange(beams * vocab), vocab)
    for r in range(batch):
        flat = score[r].flatten()
        order = np.lexsort((token, -x[r].flatten().numpy(), beam, -flat.numpy()))[:best]
        order = torch.from_numpy(order)
        order = order[flat[order] > -math.inf]
        n = order.numel()
        out[r, :n], ob[r, :n], ot[r, :n] = flat[order], order // vocab, order % vocab
    return out, ob, ot


def check(logits, scores, best):
    batch = logits.shape[0]
    out = torch.full((batch, best), float("nan"), device="cuda")
    ob, ot = (torch.full((batch, best), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    fasttree.fasttree_beam_select(logits.cuda(), scores.cuda(), out, ob, ot)
    torch.cuda.synchronize()
    assert lib.read_device_status() == 0
    ws, wb, wt = want(logits, scores, best)
    assert torch.equal(ob.cpu().long(), wb) and torch.equal(ot.cpu().long(), wt)
    # a sum of exponentials, each within 2^-21, in chains of fp32 sums of at most 128; one rounding of the score, which may be beyond fp32
    got, rounded = out.cpu().double(), ws.float().double()
    assert torch.equal(got.isinf(), rounded.isinf()) and not got.isnan().any()
    live = ~rounded.isinf()
    assert bool(((got - ws)[live].abs() <= 2.0 ** -24 * ws[live].abs() + 2.0 ** -17).all())


def inputs(batch, beams, vocab, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(batch, beams, vocab, generator=g) * 2.5).to(dtype), torch.randn(batch, beams, generator=g) - 5, g
