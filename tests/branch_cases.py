"""Trees of drafted tokens and the 64-bit oracle of their attention (plain torch, no code of the product)."""
import math
import random

import torch


def tree(rng, n, pads=0, chain=0.4, roots=0.0):
    """Parents of ``n`` tokens, the last ``pads`` of them padding (-2)."""
    kept = max(1, n - pads)
    out = [-1]
    for i in range(1, kept):
        out.append(-1 if rng.random() < roots else i - 1 if rng.random() < chain else rng.randrange(i))
    return out + [-2] * (n - kept)


def paths(parents):
    """Per token the numbers that it sees among its request's, and its depth; children of padding are padding."""
    sees, depth, pad = [], [], []
    for i, p in enumerate(parents):
        bad = p < -1 or p >= i or (p >= 0 and pad[p])        # -2, what is no earlier token, what hangs on padding
        pad.append(bad)
        sees.append([] if bad else [i] if p == -1 else sees[p] + [i])
        depth.append(depth[p] + 1 if p >= 0 and not bad else 0)
    return sees, depth


def in_sight(cached, parents, window):
    """Per token the offsets behind its request's start that it sees, and its position."""
    sees, depth = paths(parents)
    out = []
    for i in range(len(parents)):
        first = cached + depth[i] - window + 1 if window else 0
        out.append(list(range(max(0, first), cached)) + [cached + j for j in sees[i] if not window or depth[i] - depth[j] < window])
    return out, [cached + d for d in depth]


def oracle(q, k, v, table, cached, trees, scale, cap, window):
    """Output, LSE, sum of weight x |v| and the largest sum of |q k| x scale of every query row and head, in 64 bits, as
    extend_cases.oracle gives them; a row that sees nothing is 0 with an LSE of -inf."""
    hq, hkv = q.shape[1], k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, absv = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    lse, size = torch.full(q.shape[:2], -math.inf, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    at = 0
    for r, (c, parents) in enumerate(zip(cached, trees)):
        sight, _ = in_sight(c, parents, window)
        for i, offsets in enumerate(sight):
            if offsets:
                sel = table[r, offsets].long()
                kk, vv = k[sel].repeat_interleave(hq // hkv, 1), v[sel].repeat_interleave(hq // hkv, 1)
                products = kk * q[at + i]
                s = products.sum(-1) * scale
                size[at + i] = products.abs().sum(-1).amax(0) * abs(scale)
                if cap > 0:
                    s = cap * torch.tanh(s / cap)
                lse[at + i] = torch.logsumexp(s, 0)
                w = torch.exp(s - lse[at + i])
                out[at + i], absv[at + i] = (w[..., None] * vv).sum(0), (w[..., None] * vv.abs()).sum(0)
        at += len(parents)
    return out, lse, absv, size


def random_step(rng):
    """Cached and drafted lengths, shared prefixes and a window of a small step."""
    n = rng.randint(1, 7)
    cached = [rng.choice((0, 1, rng.randint(1, 400))) for _ in range(n)]
    nodes = [rng.choice((0, 1, rng.randint(1, 20), rng.randint(1, 150))) for _ in range(n)]
    shared = []
    if n > 1 and rng.random() < 0.6:
        members = sorted(rng.sample(range(n), rng.randint(2, n)))
        length = rng.randint(0, min(cached[m] for m in members))
        if length:
            shared.append((members, length))
    return cached, nodes, shared, rng.choice((0, 0, rng.randint(1, 60), rng.randint(1, 500)))


def make_trees(rng, nodes):
    return [tree(rng, n, rng.choice((0, 0, min(2, n - 1))), rng.choice((0.0, 0.4, 1.0)), rng.choice((0.0, 0.2))) if n else [] for n in nodes]


def rng_of(seed):
    return random.Random(seed)
