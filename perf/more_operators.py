"""The work that the operators for branching continuations are measured on, with their plain forms.

* ``draft``   attention of a step's drafted tokens, which form a tree per request, over the paged cache that holds their
              prefixes and themselves: a token sees the cached tokens, its ancestors and itself (scores capped or not,
              everything or the newest ``window`` positions in sight).  A pass also turns the trees' parents, new in every
              step, into the tokens' positions;
* ``accept``  the drafted tokens that the model agrees with, from its logits: from a request's first token on, the child that
              holds the largest logit's token, as long as there is one; the accepted tokens' cache rows come first in the
              request's row table;
* ``beam``    a step of beam search: the best of beams x vocabulary by summed log-probability, and the row table's rows of
              the beams that go on.

``listed()`` are fixed cases from the repository's own head layouts and batches; ``draw(rng)`` gives more of the same
ranges.  Inputs are N(0, 1) tensors made from the seed on the GPU, queries larger where scores are capped, logits with a
spread of a few units.
"""
import math
import os
import random
import sys

import torch

own = False      # True: the framework's operators; False: the same in elementary torch operations

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _framework():
    package = os.path.abspath("fasttree-artifact_b200")      # the working folder is the repository's root
    for p in (package, os.path.join(package, "kernel_bench")):
        if p not in sys.path:
            sys.path.insert(0, p)
    import fasttree
    return fasttree


def _draft(name, reqs, shared, private, nodes, hq, hkv, d, dtype, cap=0.0, window=0, layout="prefill", pads=0, shape_seed=0):
    return {"name": name, "op": "draft", "reqs": reqs, "shared": shared, "private_lo": private[0], "private_hi": private[1],
            "nodes_lo": nodes[0], "nodes_hi": nodes[1], "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "cap": cap,
            "window": window, "layout": layout, "pads": pads, "shape_seed": shape_seed}


def _accept(name, reqs, nodes, vocab, dtype, depth, shape_seed=0):
    return {"name": name, "op": "accept", "reqs": reqs, "nodes_lo": nodes[0], "nodes_hi": nodes[1], "vocab": vocab,
            "dtype": dtype, "depth": depth, "shape_seed": shape_seed}


def _beam(name, reqs, beams, best, vocab, dtype, length, shape_seed=0):
    return {"name": name, "op": "beam", "reqs": reqs, "beams": beams, "best": best, "vocab": vocab, "dtype": dtype,
            "length_lo": length[0], "length_hi": length[1], "shape_seed": shape_seed}


def listed():
    return [
        # four requests with a few drafted tokens each, fp32 storage: the smallest configuration
        _draft("draft_small_fp32", 4, 512, (64, 64), (5, 13), 8, 2, 128, "fp32", shape_seed=1),
        # one conversation, 32 drafted tokens: the call's latency
        _draft("draft_one", 1, 0, (2500, 2500), (32, 32), 32, 8, 128, "fp16"),
        # a batch of conversations of many lengths, cache rows in no order, trees padded to one size
        _draft("draft_batch_64", 64, 0, (300, 4000), (16, 16), 32, 8, 128, "bf16", layout="scattered", pads=4, shape_seed=2),
        # questions on one document: ragged trees behind a prefix that all share
        _draft("draft_shared_64", 64, 4096, (20, 300), (9, 61), 32, 8, 128, "fp16", shape_seed=3),
        # a model that caps its scores and looks 4096 tokens back, heads of 256
        _draft("draft_window_256", 16, 0, (300, 9000), (24, 24), 16, 8, 256, "bf16", cap=50.0, window=4096, shape_seed=4),
        # long contexts, large trees: the largest
        _draft("draft_long_8", 8, 0, (12000, 20000), (64, 64), 64, 8, 128, "bf16", shape_seed=5),
        # one conversation's drafts against the model's logits: latency
        _accept("accept_one", 1, (32, 32), 32000, "fp16", 4),
        # a batch, ragged trees, a large vocabulary
        _accept("accept_batch_64", 64, (12, 33), 131072, "bf16", 6, shape_seed=6),
        # logits in fp32, an odd vocabulary, every drafted token of short chains in question
        _accept("accept_odd_fp32", 33, (5, 6), 100003, "fp32", 5, shape_seed=7),
        # one request of four beams: latency
        _beam("beam_one", 1, 4, 8, 32000, "fp16", (300, 300)),
        # a batch of four beams each, a large vocabulary, twice as many candidates as beams
        _beam("beam_batch_64", 64, 4, 8, 131072, "bf16", (100, 6000), shape_seed=8),
        # wide beams, an odd vocabulary, fp32
        _beam("beam_wide_fp32", 12, 16, 32, 50021, "fp32", (500, 9000), shape_seed=9),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.2:
        while True:
            lo = _log_int(rng, 1, 64)
            case = _accept("", _log_int(rng, 1, 128), (lo, lo + rng.choice((0, rng.randrange(1 + lo)))),
                           _log_int(rng, 1000, 131072), rng.choice(("fp16", "bf16", "fp32")), _log_int(rng, 1, 10),
                           rng.randrange(1 << 20))
            if case["reqs"] * case["nodes_hi"] * case["vocab"] * BYTES[case["dtype"]] <= 64 * 33 * 131072 * 2:
                break
    elif kind < 0.45:
        while True:
            beams = rng.choice((1, 2, 3, 4, 5, 8, 16))
            lo = _log_int(rng, 10, 8000)
            case = _beam("", _log_int(rng, 1, 128), beams, rng.choice((beams, 2 * beams)), _log_int(rng, 1000, 131072),
                         rng.choice(("fp16", "bf16", "bf16", "fp32")), (lo, lo + rng.randrange(1 + lo)), rng.randrange(1 << 20))
            if case["reqs"] * beams * case["vocab"] * BYTES[case["dtype"]] <= 64 * 4 * 131072 * 2:
                break
    else:
        while True:
            dtype = rng.choice(("fp16", "bf16", "bf16", "fp16", "fp32"))
            hq, hkv = rng.choice(((32, 8), (28, 4), (16, 16), (64, 8), (16, 8), (16, 1), (8, 2)))
            lo = _log_int(rng, 1, 128)
            private = rng.choice((0, _log_int(rng, 1, 20000)))
            case = _draft("", _log_int(rng, 1, 128), rng.choice((0, _log_int(rng, 16, 8192))),
                          (private, private + rng.choice((0, _log_int(rng, 1, 4096)))), (lo, lo + rng.choice((0, rng.randrange(1 + lo)))),
                          hq, hkv, rng.choice((64, 128, 128, 256)), dtype, rng.choice((0.0, 0.0, 30.0)),
                          rng.choice((0, 0, _log_int(rng, 64, 8192))), rng.choice(("prefill", "scattered")),
                          rng.choice((0, 0, 3)), rng.randrange(1 << 20))
            cost = work(case)
            # at most the largest listed case's work; less in fp32, which no tensor core takes unrounded
            most = (6e8, 2.5e11) if dtype != "fp32" else (6e7, 8e9)
            if cost["bytes"] <= most[0] and cost["flops"] <= most[1]:
                break
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------------ shapes
def _draft_shape(case):
    """Per request its cached private tokens and its drafted tokens."""
    rng = random.Random(case["shape_seed"])
    private = [rng.randint(case["private_lo"], case["private_hi"]) for _ in range(case["reqs"])]
    return private, [rng.randint(case["nodes_lo"], case["nodes_hi"]) for _ in range(case["reqs"])]


def _accept_shape(case):
    """Per request its drafted tokens, how many of them the model agrees with, and its cached tokens."""
    rng = random.Random(case["shape_seed"])
    nodes = [rng.randint(case["nodes_lo"], case["nodes_hi"]) for _ in range(case["reqs"])]
    return nodes, [rng.randint(1, min(n, case["depth"])) for n in nodes], [rng.randint(10, 3000) for _ in nodes]


def _beam_shape(case):
    """Per request its tokens so far, and how many leading ones all of its beams share."""
    rng = random.Random(case["shape_seed"])
    length = [rng.randint(case["length_lo"], case["length_hi"]) for _ in range(case["reqs"])]
    return length, [rng.randint(0, n // 2) for n in length]


def work(case):
    if case["op"] == "accept":
        nodes, agreed, _ = _accept_shape(case)
        # the logits along the accepted path, the trees with their tokens and rows, the results
        return {"bytes": sum(agreed) * case["vocab"] * BYTES[case["dtype"]] + 20 * sum(nodes) + 8 * len(nodes), "flops": sum(agreed) * case["vocab"]}
    if case["op"] == "beam":
        length, shared = _beam_shape(case)
        logits = case["reqs"] * case["beams"] * case["vocab"]
        rows = sum(n - s for n, s in zip(length, shared)) * case["beams"]
        return {"bytes": logits * BYTES[case["dtype"]] + 8 * rows + case["reqs"] * (4 * case["beams"] + 12 * case["best"]), "flops": 4 * logits}
    e, hq, hkv, d, w = BYTES[case["dtype"]], case["hq"], case["hkv"], case["d"], case["window"]
    private, nodes = _draft_shape(case)
    rows, pairs, low = 0, 0, case["shared"]
    for p, n in zip(private, nodes):
        cached = case["shared"] + p
        begin = max(0, cached - w + 1) if w else 0
        pairs += n * (cached - begin + 1)                     # at least: the cached tokens and itself
        low = min(low, begin)
        rows += cached + n - max(case["shared"], begin)
    rows += case["shared"] - low
    return {"bytes": 2 * e * d * (rows * hkv + sum(nodes) * hq) + 8 * sum(nodes), "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------------ inputs
def _randn(gen, *shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dtype)


def _tree(rng, n, pads=0):
    """Parents of n drafted tokens: the first is the root, every other one hangs on the token before it or on any earlier one;
    the last ``pads`` are padding (-2)."""
    kept = max(1, n - pads)
    return [-1] + [i - 1 if rng.random() < 0.4 else rng.randrange(i) for i in range(1, kept)] + [-2] * (n - kept)


def _draft_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    private, nodes = _draft_shape(case)
    hq, hkv, d, dtype, shared = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]], case["shared"]
    seq = [shared + p + n for p, n in zip(private, nodes)]
    rows = shared + sum(private) + sum(nodes) + 64
    order = torch.arange(rows) if case["layout"] == "prefill" else torch.randperm(rows, generator=torch.Generator().manual_seed(seed))
    order = order.to(torch.int32)
    table = torch.zeros(len(seq), max(seq) + 5, dtype=torch.int32)
    at = shared
    for r, length in enumerate(seq):
        table[r, :shared] = order[:shared]
        table[r, shared:length] = order[at:at + length - shared]
        at += length - shared
    k, v = _randn(gen, rows, hkv, d, dtype=dtype), _randn(gen, rows, hkv, d, dtype=dtype)
    q = _randn(gen, sum(nodes), hq, d, dtype=dtype, scale=4.0 if case["cap"] else 1.0)
    parents = [x for n in nodes for x in _tree(rng, n, min(case["pads"], n - 1))]
    return {"q": q, "k": k, "v": v, "table": table.cuda(), "seq": seq, "nodes": nodes, "scale": d ** -0.5,
            "parents": torch.tensor(parents, dtype=torch.int32, device="cuda")}


def _accept_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    nodes, agreed, cached = _accept_shape(case)
    total, vocab = sum(nodes), case["vocab"]
    logits = _randn(gen, total, vocab, dtype=DTYPES[case["dtype"]], scale=2.5)
    parents, tokens, peaks = [], [], []
    for n, path in zip(nodes, agreed):
        # a path of accepted tokens through the tree; siblings never hold the same token
        on = sorted(rng.sample(range(1, n), path - 1)) if path > 1 else []
        on = [0] + on
        tree = _tree(rng, n)
        for a, b in zip(on, on[1:]):
            tree[b] = a
        base, ids = len(tokens), rng.sample(range(vocab), n + 1)
        parents += tree
        tokens += ids[:n]
        for a, b in zip(on, on[1:] + [n]):
            peaks.append((base + a, ids[b]))              # behind the last one the model wants a token that nobody drafted
    where = torch.tensor(peaks, device="cuda")
    logits[where[:, 0], where[:, 1]] = 24.0
    rows = sum(cached) + total + 64
    slots = torch.randperm(rows, generator=gen, device="cuda")[:total].to(torch.int32)
    table = torch.zeros(len(nodes), max(c + n for c, n in zip(cached, nodes)) + 3, dtype=torch.int32, device="cuda")
    return {"logits": logits, "parents": torch.tensor(parents, dtype=torch.int32, device="cuda"),
            "tokens": torch.tensor(tokens, device="cuda"), "nodes": nodes, "cached": cached, "slots": slots, "table": table}


def _beam_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    reqs, beams = case["reqs"], case["beams"]
    length, shared = _beam_shape(case)
    logits = _randn(gen, reqs, beams, case["vocab"], dtype=DTYPES[case["dtype"]], scale=2.5)
    scores = torch.randn(reqs, beams, generator=gen, device="cuda") - 10.0
    width = max(length) + 3
    # two rows of the table per beam: one that it has, one for what goes on from it
    table = torch.randint(0, 1 << 24, (2 * reqs * beams, width), generator=gen, device="cuda", dtype=torch.int32)
    rows = torch.randperm(2 * reqs * beams, generator=gen, device="cuda").to(torch.int32).view(2, reqs, beams)
    return {"logits": logits, "scores": scores, "table": table, "rows": rows[0], "next_rows": rows[1],
            "starts": torch.tensor(shared, dtype=torch.int32, device="cuda"), "ends": torch.tensor(length, dtype=torch.int32, device="cuda")}


def _inputs(case, seed):
    return {"draft": _draft_inputs, "accept": _accept_inputs, "beam": _beam_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    dev = {"device": "cuda"}
    if case["op"] == "draft":
        s["o"] = torch.empty_like(s["q"])
        s["positions"] = torch.empty(s["q"].shape[0], dtype=torch.int32, **dev)
        if own:
            n = len(s["seq"])
            prefixes = [(range(n), case["shared"])] if n > 1 and case["shared"] else None
            s["plan"] = _framework().fasttree_extend_preparation(
                s["seq"], s["nodes"], [r * s["table"].shape[1] for r in range(n)], case["hq"], case["hkv"], case["d"], s["q"].dtype,
                shared_prefixes=prefixes, window=case["window"], draft=True, device="cuda")
    elif case["op"] == "accept":
        n = len(s["nodes"])
        s["accepted"] = torch.empty(n, max(s["nodes"]), dtype=torch.int32, **dev)
        s["counts"], s["next"] = torch.empty(n, dtype=torch.int32, **dev), torch.empty(n, dtype=torch.int64, **dev)
        if own:
            s["plan"] = _framework().fasttree_extend_preparation(
                [c + m for c, m in zip(s["cached"], s["nodes"])], s["nodes"], [r * s["table"].shape[1] for r in range(n)], 8, 2, 128,
                torch.float16, draft=True, device="cuda")
    else:
        shape = (case["reqs"], case["best"])
        s["best_scores"] = torch.empty(shape, dtype=torch.float32, **dev)
        s["best_beams"], s["best_tokens"] = torch.empty(shape, dtype=torch.int32, **dev), torch.empty(shape, dtype=torch.int32, **dev)
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"draft": _draft_own, "accept": _accept_own, "beam": _beam_own}[op](s)
    return {"draft": _draft_plain, "accept": _accept_plain, "beam": _beam_plain}[op](s)


def _draft_own(s):
    ft = _framework()
    ft.fasttree_draft_tree(s["parents"], s["plan"], s["positions"])
    ft.fasttree_extend(s["q"], s["k"], s["v"], s["o"], s["table"], s["plan"], s["scale"], logit_cap=s["case"]["cap"] or -1)
    return s["o"], s["positions"]


def _accept_own(s):
    _framework().fasttree_draft_accept(s["logits"], s["tokens"], s["parents"], s["plan"], s["accepted"], s["counts"], s["next"],
                                       slots=s["slots"], kv_entries=s["table"])
    return s["accepted"], s["counts"], s["next"], s["table"]


def _beam_own(s):
    ft, beams = _framework(), s["case"]["beams"]
    ft.fasttree_beam_select(s["logits"], s["scores"], s["best_scores"], s["best_beams"], s["best_tokens"])
    ft.fasttree_beam_reorder(s["table"], s["rows"], s["best_beams"][:, :beams], s["starts"], s["ends"], out_rows=s["next_rows"])
    return s["best_scores"], s["best_beams"], s["best_tokens"], s["table"]


def _ancestors(parents):
    """Which tokens of one tree each of them sees among themselves, and the tokens' depths: [n, n], [n]."""
    n = parents.shape[0]
    index = torch.arange(n, device=parents.device)
    at = torch.where(parents == -2, torch.full_like(index, -1), index)
    depth = torch.zeros_like(index)
    seen = torch.zeros(n, n, dtype=torch.bool, device=parents.device)
    for _ in range(n):                                       # all tokens climb one step at a time
        seen |= at[:, None] == index
        up = torch.where(at >= 0, parents.long()[at.clamp(min=0)], torch.full_like(at, -1))
        depth += up >= 0
        at = up
    return seen, depth


def _draft_plain(s):
    c = s["case"]
    hq, hkv, w = c["hq"], c["hkv"], c["window"]
    at = 0
    for r, (length, n) in enumerate(zip(s["seq"], s["nodes"])):
        cached = length - n
        seen, depth = _ancestors(s["parents"][at:at + n])
        s["positions"][at:at + n] = (cached + depth).to(torch.int32)
        sight = torch.cat([torch.ones(n, cached, dtype=torch.bool, device="cuda"), seen], 1)
        if w:
            where = torch.cat([torch.arange(cached, device="cuda"), cached + depth])
            sight &= where[None] > (cached + depth - w)[:, None]
        slots = s["table"][r, :length].long()
        k = s["k"][slots].float().permute(1, 2, 0)[:, None]       # [kv heads, 1, d, keys]
        v = s["v"][slots].float().transpose(0, 1)[:, None]        # [kv heads, 1, keys, d]
        q = s["q"][at:at + n].float().transpose(0, 1).unflatten(0, (hkv, hq // hkv))
        scores = (q @ k) * s["scale"]
        if c["cap"]:
            scores = torch.tanh(scores / c["cap"]) * c["cap"]
        scores = scores.masked_fill(~sight, -math.inf)
        top = scores.amax(-1, keepdim=True)
        weights = (scores - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
        total = weights.sum(-1, keepdim=True)
        out = (weights @ v) / torch.where(total == 0, torch.ones_like(total), total)
        s["o"][at:at + n] = out.flatten(0, 1).transpose(0, 1).to(s["o"].dtype)
        at += n
    return s["o"], s["positions"]


def _accept_plain(s):
    n, device = len(s["nodes"]), s["logits"].device
    # the largest logit, of equal ones the first
    top = s["logits"].amax(1, keepdim=True)
    ids = torch.arange(s["logits"].shape[1], device=device)
    target = torch.where(s["logits"] == top, ids, ids.shape[0]).amin(1)
    nodes = torch.tensor(s["nodes"], device=device)
    first = nodes.cumsum(0) - nodes
    width = max(s["nodes"])
    inside = torch.arange(width, device=device) < nodes[:, None]
    where = torch.where(inside, first[:, None] + torch.arange(width, device=device), 0)
    parents, tokens = torch.where(inside, s["parents"].long()[where], -2), s["tokens"][where]
    at, alive = torch.zeros(n, dtype=torch.long, device=device), parents[:, 0] == -1
    s["accepted"].fill_(-1)
    s["counts"].zero_()
    s["next"].fill_(-1)
    index = torch.arange(width, device=device)
    for step in range(width):
        s["accepted"][:, step] = torch.where(alive, at, -1).to(torch.int32)
        s["counts"].add_(alive.to(torch.int32))
        want = target[first + at]
        s["next"].copy_(torch.where(alive, want, s["next"]))
        child = torch.where((parents == at[:, None]) & (tokens == want[:, None]) & (index > at[:, None]), index, width).amin(1)
        alive = alive & (child < width)
        at = torch.where(alive, child, at)
    # accepted tokens first, the others behind them, both in order
    taken = torch.zeros(n, width + 1, dtype=torch.bool, device=device)
    taken.scatter_(1, torch.where(s["accepted"] >= 0, s["accepted"].long(), width), True)
    group = torch.where(inside, torch.where(taken[:, :width], 0, 1), 2)
    order = torch.sort(group, dim=1, stable=True).indices
    cached = torch.tensor(s["cached"], device=device)
    row = torch.arange(n, device=device)[:, None].expand(n, width)
    s["table"][row[inside], (cached[:, None] + index)[inside]] = s["slots"][(first[:, None] + order)[inside]]
    return s["accepted"], s["counts"], s["next"], s["table"]


def _beam_plain(s):
    c = s["case"]
    reqs, beams, best, vocab = c["reqs"], c["beams"], c["best"], c["vocab"]
    x = s["logits"].float()
    # scores next to one another: the logarithm of the sum and what follows in 64 bits
    top = x.amax(-1, keepdim=True)
    lse = top.double() + (x - top).exp().sum(-1, dtype=torch.float64, keepdim=True).log()
    # per beam its best by (logit, lowest token): one whole number each
    bits = (x + 0.0).view(torch.int32)
    rank = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    keys = rank * (1 << 32) + (0xffffffff - torch.arange(vocab, device=x.device))
    keys = torch.topk(keys, min(best, vocab), dim=-1).values
    tokens = 0xffffffff - (keys & 0xffffffff)
    score = s["scores"].double()[..., None] + (torch.gather(x, 2, tokens).double() - lse)
    # of equal scores the lowest beam's first
    score, at = torch.sort(score.flatten(1), dim=1, descending=True, stable=True)
    s["best_scores"].copy_(score[:, :best])
    s["best_beams"].copy_(at[:, :best] // keys.shape[-1])
    s["best_tokens"].copy_(torch.gather(tokens.flatten(1), 1, at[:, :best]))
    # the rows of the beams that go on
    go_on = torch.gather(s["rows"].long(), 1, s["best_beams"][:, :beams].long())
    column = torch.arange(s["table"].shape[1], device=x.device)
    moved = ((column >= s["starts"][:, None]) & (column < s["ends"][:, None]))[:, None]
    s["table"][s["next_rows"].long()] = torch.where(moved, s["table"][go_on], s["table"][s["next_rows"].long()])
    return s["best_scores"], s["best_beams"], s["best_tokens"], s["table"]


# ------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    return {"draft": _draft_exact, "accept": _accept_exact, "beam": _beam_exact}[case["op"]](case, seed)


def _draft_exact(case, seed):
    s = _draft_inputs(case, seed)
    parents, hq, hkv = s["parents"].tolist(), case["hq"], case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    positions, at = [], 0
    for r, (length, n) in enumerate(zip(s["seq"], s["nodes"])):
        cached, tree = length - n, parents[at:at + n]
        reach, depth = [], []                       # per token the set of drafted tokens that it sees
        for i, p in enumerate(tree):
            reach.append(set() if p == -2 else {i} if p == -1 else reach[p] | {i})
            depth.append(depth[p] + 1 if p >= 0 else 0)
        positions += [cached + x for x in depth]
        seen = torch.zeros(n, length, dtype=torch.bool)
        for i in range(n):
            far = case["window"] or length + n
            seen[i, max(0, cached + depth[i] - far + 1):cached] = True
            for j in reach[i]:
                seen[i, cached + j] = depth[i] - depth[j] < far
        seen = seen.cuda()
        some = seen.any(1)
        slots = s["table"][r, :length].long()
        for h in range(hq):
            k, v = s["k"][slots, h // (hq // hkv)].double(), s["v"][slots, h // (hq // hkv)].double()
            z = torch.einsum("qd,kd->qk", s["q"][at:at + n, h].double(), k) * s["scale"]
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            z = torch.where(seen, z, torch.full_like(z, -math.inf))[some]
            out[at:at + n, h][some] = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)) @ v
        at += n
    return out, torch.tensor(positions, dtype=torch.int32, device="cuda")


def _accept_exact(case, seed):
    s = _accept_inputs(case, seed)
    parents, tokens, table = s["parents"].tolist(), s["tokens"].tolist(), s["table"].clone()
    n, width = len(s["nodes"]), max(s["nodes"])
    accepted, counts, following = torch.full((n, width), -1, dtype=torch.int32), torch.zeros(n, dtype=torch.int32), torch.full((n,), -1)
    base = 0
    for r, m in enumerate(s["nodes"]):
        path, at = [], 0
        while at is not None:
            path.append(at)
            row = s["logits"][base + at].double()
            want = int(torch.nonzero(row == row.max())[0])
            at = next((i for i in range(at + 1, m) if parents[base + i] == path[-1] and tokens[base + i] == want), None)
        accepted[r, :len(path)] = torch.tensor(path, dtype=torch.int32)
        counts[r], following[r] = len(path), want
        order = path + [i for i in range(m) if i not in path]
        table[r, s["cached"][r]:s["cached"][r] + m] = s["slots"][base:base + m][torch.tensor(order, device="cuda")]
        base += m
    return accepted.cuda(), counts.cuda(), following.cuda(), table


def _beam_exact(case, seed):
    s = _beam_inputs(case, seed)
    best, vocab, beams = case["best"], case["vocab"], case["beams"]
    scores, table = [], s["table"].clone()
    from_beam, from_token = [], []
    for r in range(case["reqs"]):
        all_scores = (s["scores"][r].double()[:, None] + torch.log_softmax(s["logits"][r].double(), -1)).flatten()
        border = torch.topk(all_scores, best).values[-1]
        some = torch.nonzero(all_scores >= border)[:, 0]     # in the order of beams and tokens
        order = torch.sort(all_scores[some], descending=True, stable=True).indices[:best]
        scores.append(all_scores[some][order])
        from_beam.append(some[order] // vocab)
        from_token.append(some[order] % vocab)
        lo, hi = int(s["starts"][r]), int(s["ends"][r])
        table[s["next_rows"][r].long(), lo:hi] = s["table"][s["rows"][r][from_beam[-1][:beams]].long(), lo:hi]
    return torch.stack(scores), torch.stack(from_beam).to(torch.int32), torch.stack(from_token).to(torch.int32), table
