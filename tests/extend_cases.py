"""Inputs and the 64-bit oracle of the extend-attention and append tests (plain torch, no code of the product)."""
import math

import torch


def pool(seq, ext, shared, rows_extra=7, layout="scattered", seed=0):
    """``(table [requests, width], pool rows)`` of requests with ``seq`` tokens; ``shared``: (members, length) pairs, of which
    a member takes the pool rows of the first member for its first ``length`` tokens (longer pairs last)."""
    g = torch.Generator().manual_seed(seed)
    width = max(seq, default=0) + 3
    rows = sum(seq) + rows_extra
    order = torch.arange(rows) if layout == "prefill" else torch.randperm(rows, generator=g)
    table = torch.full((len(seq), width), -7, dtype=torch.int32)
    at = 0
    for r, n in enumerate(seq):
        table[r, :n] = order[at:at + n].to(torch.int32)
        at += n
    for members, length in sorted(shared, key=lambda s: s[1]):
        for m in members[1:]:
            table[m, :length] = table[members[0], :length]
    return table, rows


def oracle(q, k, v, table, seq, ext, scale, cap, window):
    """Output, LSE, sum of weight x |v| and the largest sum of |q k| x scale of every query row and head, in 64 bits."""
    hq, hkv = q.shape[1], k.shape[1]
    g = hq // hkv
    q, k, v = q.double(), k.double(), v.double()
    out, lse, absv = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -math.inf, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape[:2], dtype=torch.float64)
    at = 0
    for r, (n, e) in enumerate(zip(seq, ext)):
        rows = table[r, :n].long()
        for i in range(e):
            pos = n - e + i
            first = max(0, pos - window + 1) if window else 0
            sel = rows[first:pos + 1]
            kk, vv = k[sel].repeat_interleave(g, 1), v[sel].repeat_interleave(g, 1)        # [keys, heads, d]
            s = (kk * q[at + i]).sum(-1) * scale
            size[at + i] = (kk * q[at + i]).abs().sum(-1).amax(0) * abs(scale)
            if cap > 0:
                s = cap * torch.tanh(s / cap)
            lse[at + i] = torch.logsumexp(s, 0)
            w = torch.exp(s - lse[at + i])
            out[at + i] = (w[..., None] * vv).sum(0)
            absv[at + i] = (w[..., None] * vv.abs()).sum(0)
        at += e
    return out, lse, absv, size


def bounds(dtype, out, absv, size, cap, d):
    """How far a kernel's outputs and LSEs may be off, per element.

    The storage type's half step u counts twice: on each probability before the product with V (relative to the sum of weight
    x |v|) and on the output.  In fp32 a score is a sum of d products: off by at most (d + 8) half steps of the sum of |q k|
    scale - the 8 for the scalings, and tensor cores that cut instead of rounding count double -, a tanh by 2^-21 of the cap.
    The exponent function, its argument (up to 160 in the power of two) and the sums of a row are within 2^-15 together.  An
    error x in the scores moves every weight by at most e^2x - 1."""
    u = torch.finfo(dtype).eps / 2
    if dtype == torch.float32:
        u = 2.0 ** -24
    x = 2 * (d + 8) * 2.0 ** -24 * size + (cap * 2.0 ** -21 if cap > 0 else 0.0)
    rel = torch.expm1(2 * x) + 2.0 ** -15
    return (u + rel)[..., None] * absv + u * (out.abs() + rel[..., None] * absv) + 1e-30, x + 2.0 ** -15
