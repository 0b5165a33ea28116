"""The work that the serving operators beside tree decode are measured on, with their plain forms.

* ``append``  a step's keys and values go into the paged cache; keys and queries are turned by their positions on the
              way (a position per token, or one each along time, height and width);
* ``extend``  causal attention of several new tokens per request - one of them, a question, a whole prompt - over the
              paged cache that holds their prefixes and themselves, the prefixes shared between requests or not, the
              scores capped by a tanh or not, everything or the newest ``window`` positions in sight.

``listed()`` are fixed cases from the repository's own head layouts and batches; ``draw(rng)`` gives more of the same
ranges.  Inputs are N(0, 1) tensors made from the seed on the GPU, queries larger where scores are capped.
"""
import math
import os
import random
import sys

import torch

own = False      # True: the framework's operators; False: the same in elementary torch operations

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _framework():
    package = os.path.abspath("fasttree-artifact_b200")      # the working folder is the repository's root
    for p in (package, os.path.join(package, "kernel_bench")):
        if p not in sys.path:
            sys.path.insert(0, p)
    import fasttree
    return fasttree


def _append(name, tokens, hq, hkv, d, dtype, axes=1, rot=None, interleaved=False, padded=0, layout="scattered"):
    return {"name": name, "op": "append", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype, "axes": axes,
            "rot": rot or d, "interleaved": interleaved, "padded": padded, "layout": layout}


def _extend(name, groups, shared, reqs, private, new, hq, hkv, d, dtype, cap=0.0, window=0, layout="prefill", shape_seed=0):
    return {"name": name, "op": "extend", "groups": groups, "shared": shared, "reqs": reqs, "private_lo": private[0],
            "private_hi": private[1], "new_lo": new[0], "new_hi": new[1], "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
            "cap": cap, "window": window, "layout": layout, "shape_seed": shape_seed}


def listed():
    return [
        # one decode step's tokens of 64 requests: the call's latency
        _append("append_step_64", 64, 32, 8, 128, "fp16"),
        # a prefill chunk: every token's keys and values to consecutive slots
        _append("append_chunk", 8192, 32, 8, 128, "bf16", layout="prefill"),
        # images in the prompt: positions along time, height and width; an odd number of tokens, the batch padded
        _append("append_images", 5037, 28, 4, 128, "bf16", axes=3, padded=11),
        # half of each head turned, in adjacent pairs; fp32 storage
        _append("append_pairs_fp32", 777, 8, 2, 128, "fp32", rot=64, interleaved=True),
        # the smallest configuration in fp32: a few new tokens of four requests
        _extend("extend_small_fp32", 1, 512, 4, (64, 64), (3, 17), 8, 2, 128, "fp32"),
        # one decode step: 64 single tokens under a system prompt, every request with turns of its own
        _extend("step_prefix_64", 1, 4096, 64, (256, 256), (1, 1), 32, 8, 128, "fp16"),
        # one decode step of a model that caps its scores and looks 4096 tokens back, heads of 256, ragged lengths
        _extend("step_window_256", 16, 0, 16, (300, 9000), (1, 1), 16, 8, 256, "bf16", cap=50.0, window=4096),
        # a burst of questions on one document: short new turns on a long prefix that all share
        _extend("questions_64", 1, 4096, 64, (0, 0), (20, 60), 32, 8, 128, "bf16", shape_seed=1),
        # sixteen documents with eight questions each, heads of 64, slots in no order
        _extend("documents_64", 16, 1500, 128, (0, 40), (12, 40), 32, 8, 64, "fp16", layout="scattered", shape_seed=2),
        # ragged prompts without a cached prefix, slots in no order
        _extend("prompts_16", 16, 0, 16, (0, 0), (200, 2000), 32, 8, 128, "fp16", layout="scattered", shape_seed=3),
        # prompts of a model that caps its scores, seven query heads per KV head
        _extend("prompts_capped", 8, 0, 8, (0, 2000), (700, 2500), 28, 4, 128, "bf16", cap=30.0, shape_seed=4),
        # a chunk of one long prompt behind what is cached of it: the largest
        _extend("chunk_long", 1, 0, 1, (12288, 12288), (4096, 4096), 64, 8, 128, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.3:
        hq, hkv = rng.choice(((32, 8), (28, 4), (16, 16), (64, 8), (8, 2), (5, 1)))
        d = rng.choice((64, 128, 256))
        axes = rng.choice((1, 1, 3))
        tokens = _log_int(rng, 1, 8192)
        case = _append("", tokens, hq, hkv, d, rng.choice(("fp16", "bf16", "fp32")), axes,
                       d if axes == 3 else rng.choice((d, d // 2, 32)), rng.random() < 0.3,
                       rng.randrange(0, 1 + min(16, tokens // 4)), rng.choice(("scattered", "prefill")))
        if case["dtype"] == "fp32" and hq * tokens > 32 * 4096:
            case["tokens"] = 1 + 32 * 4096 // hq
        del case["name"]
        return case
    while True:
        dtype = rng.choice(("fp16", "bf16", "bf16", "fp16", "fp32"))
        hq, hkv = rng.choice(((32, 8), (28, 4), (16, 16), (64, 8), (16, 8), (16, 1), (8, 2)))
        d = rng.choice((64, 128, 128, 256))
        reqs = _log_int(rng, 1, 256)
        groups = rng.choice((1, reqs, 1 + rng.randrange(reqs)))
        shared = rng.choice((0, _log_int(rng, 16, 16384)))
        private_lo = rng.choice((0, 0, _log_int(rng, 1, 4096)))
        private_hi = private_lo + rng.choice((0, _log_int(rng, 1, 4096)))
        new_lo = rng.choice((1, _log_int(rng, 1, 4096)))
        new_hi = new_lo + rng.choice((0, 0 if new_lo == 1 else _log_int(rng, 1, 1000)))
        case = _extend("", groups, shared, reqs, (private_lo, private_hi), (new_lo, new_hi), hq, hkv, d, dtype,
                       rng.choice((0.0, 0.0, 30.0, 50.0)), rng.choice((0, 0, _log_int(rng, 64, 8192))),
                       rng.choice(("prefill", "scattered")), rng.randrange(1 << 20))
        del case["name"]
        cost = work(case)
        # at most the largest listed case's work; less in fp32, which no tensor core takes unrounded
        most = (6e8, 1.9e12) if dtype != "fp32" else (6e7, 8e9)
        if cost["bytes"] <= most[0] and cost["flops"] <= most[1]:
            return case


# ------------------------------------------------------------------------------------------------------ shapes
def _shape(case):
    """Per request: its group, its cached private tokens and its new tokens (requests of a group stand together)."""
    rng = random.Random(case["shape_seed"])
    n = case["reqs"]
    group = sorted(r % case["groups"] for r in range(n))
    private = [rng.randint(case["private_lo"], case["private_hi"]) for _ in range(n)]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(n)]
    return group, private, new


def _in_sight(case, first, count):
    """Pairs of a query at positions first .. first + count - 1 and a key that it sees."""
    w = case["window"]
    if not w:
        return count * first + count * (count + 1) // 2
    ramp = max(0, min(count, w - 1 - first))      # positions that still see everything
    return ramp * first + ramp * (ramp + 1) // 2 + (count - ramp) * w


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        kept = case["tokens"] - case["padded"]
        table = 4 * case["rot"] * case["tokens"]
        return {"bytes": 2 * e * d * (hq * case["tokens"] + 2 * hkv * kept) + table + 4 * case["tokens"] * (1 + case["axes"]),
                "flops": 3 * case["rot"] * (hq + hkv) * case["tokens"]}
    group, private, new = _shape(case)
    rows, pairs, w = 0, 0, case["window"]
    low = {}      # per group: the first shared position that any of its queries sees
    for g, p, n in zip(group, private, new):
        cached = case["shared"] + p
        pairs += _in_sight(case, cached, n)
        begin = max(0, cached - w + 1) if w else 0
        low[g] = min(low.get(g, case["shared"]), begin)
        rows += cached + n - max(case["shared"], begin)
    rows += sum(case["shared"] - b for b in low.values())
    return {"bytes": 2 * e * d * (rows * hkv + sum(new) * hq), "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------------ inputs
def _randn(gen, *shape, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(scale).to(dtype)


def _sections(case):
    half = case["rot"] // 2
    if case["axes"] == 1:
        return [half]
    return [half - 2 * (3 * half // 8), 3 * half // 8, 3 * half // 8]      # 16, 24, 24 of 64


def _append_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t, hq, hkv, d, dtype = case["tokens"], case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    qkv = _randn(gen, t, (hq + 2 * hkv) * d, dtype=dtype)      # as one projection leaves them
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
    rows = t + 64
    # one row more than the pool has: where the plain form puts the padding tokens (slot -1)
    k_rows, v_rows = _randn(gen, rows + 1, hkv, d, dtype=dtype), _randn(gen, rows + 1, hkv, d, dtype=dtype)
    if case["layout"] == "prefill":
        slots = torch.arange(17, 17 + t, device="cuda")
    else:
        slots = torch.randperm(rows, generator=gen, device="cuda")[:t]
    slots = slots.to(torch.int32)
    if case["padded"]:
        slots[t - case["padded"]:] = -1
    length = 16384
    positions = torch.randint(0, length, (case["axes"], t), generator=gen, device="cuda")
    half = case["rot"] // 2
    angles = torch.outer(torch.arange(length, dtype=torch.float64, device="cuda"),
                         torch.arange(half, dtype=torch.float64, device="cuda").div_(-half).mul_(math.log(1e4)).exp_())
    table = torch.cat([angles.cos(), angles.sin()], dim=1).float()      # what a model keeps for all of its layers
    return {"q": q, "k": k, "v": v, "k_rows": k_rows, "v_rows": v_rows, "k_buffer": k_rows[:-1], "v_buffer": v_rows[:-1],
            "slots": slots, "positions": positions if case["axes"] > 1 else positions[0], "table": table}


def _extend_inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    group, private, new = _shape(case)
    hq, hkv, d, dtype, shared = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]], case["shared"]
    groups = max(group) + 1
    seq = [shared + p + n for p, n in zip(private, new)]
    rows = groups * shared + sum(private) + sum(new) + 64
    order = torch.arange(rows) if case["layout"] == "prefill" else torch.randperm(rows, generator=torch.Generator().manual_seed(seed))
    order = order.to(torch.int32)
    width = max(seq) + 5
    table = torch.zeros(len(seq), width, dtype=torch.int32)
    at = groups * shared
    for r, length in enumerate(seq):
        table[r, :shared] = order[group[r] * shared:(group[r] + 1) * shared]
        table[r, shared:length] = order[at:at + length - shared]
        at += length - shared
    k, v = _randn(gen, rows, hkv, d, dtype=dtype), _randn(gen, rows, hkv, d, dtype=dtype)
    scale = 4.0 if case["cap"] else 1.0
    q = _randn(gen, sum(new), hq, d, dtype=dtype, scale=scale)
    return {"q": q, "k": k, "v": v, "table": table.cuda(), "seq": seq, "new": new, "group": group, "scale": d ** -0.5}


def prepare(case, seed):
    s = _append_inputs(case, seed) if case["op"] == "append" else _extend_inputs(case, seed)
    s["case"] = case
    if case["op"] == "append":
        s["q_out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    else:
        s["o"] = torch.empty_like(s["q"])
        if own:
            members = {}
            for r, g in enumerate(s["group"]):
                members.setdefault(g, []).append(r)
            prefixes = [(m, case["shared"]) for m in members.values() if len(m) > 1 and case["shared"]]
            s["plan"] = _framework().fasttree_extend_preparation(
                s["seq"], s["new"], [r * s["table"].shape[1] for r in range(len(s["seq"]))], case["hq"], case["hkv"], case["d"],
                s["q"].dtype, shared_prefixes=prefixes, window=case["window"], device="cuda")
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _append_own(s) if s["case"]["op"] == "append" else _extend_own(s)
    return _append_plain(s) if s["case"]["op"] == "append" else _extend_plain(s)


def _append_own(s):
    c = s["case"]
    _framework().fasttree_append(s["q"], s["k"], s["v"], s["k_buffer"], s["v_buffer"], s["slots"], q_out=s["q_out"],
                                 positions=s["positions"], cos_sin=s["table"], sections=_sections(c) if c["axes"] > 1 else None,
                                 interleaved=c["interleaved"])
    return s["q_out"], s["k_buffer"], s["v_buffer"]


def _extend_own(s):
    _framework().fasttree_extend(s["q"], s["k"], s["v"], s["o"], s["table"], s["plan"], s["scale"],
                                 logit_cap=s["case"]["cap"] or -1)
    return s["o"]


def _turn(x, cos, sin, rot, interleaved):
    x = x.float()
    head, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
    a, b = a * cos - b * sin, b * cos + a * sin
    head = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([head, rest], dim=-1)


def _append_plain(s):
    c, rot = s["case"], s["case"]["rot"]
    pos = s["positions"] if c["axes"] > 1 else s["positions"][None]
    turns = s["table"][pos]                                       # [axes, tokens, rot]
    cos, sin = [], []
    at = 0
    for axis, n in enumerate(_sections(c)):
        cos.append(turns[axis, :, at:at + n])
        sin.append(turns[axis, :, rot // 2 + at:rot // 2 + at + n])
        at += n
    cos, sin = torch.cat(cos, 1)[:, None], torch.cat(sin, 1)[:, None]
    s["q_out"].copy_(_turn(s["q"], cos, sin, rot, c["interleaved"]))
    slots = s["slots"].long()                                     # -1: the row behind the pool's last
    s["k_rows"][slots] = _turn(s["k"], cos, sin, rot, c["interleaved"]).to(s["k"].dtype)
    s["v_rows"][slots] = s["v"]
    return s["q_out"], s["k_buffer"], s["v_buffer"]


def _extend_plain(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    at = 0
    for r, (length, n) in enumerate(zip(s["seq"], s["new"])):
        slots = s["table"][r, :length].long()
        k = s["k"][slots].float().permute(1, 2, 0)[:, None]       # [kv heads, 1, d, keys]
        v = s["v"][slots].float().transpose(0, 1)[:, None]        # [kv heads, 1, keys, d]
        keys = torch.arange(length, device="cuda")
        step = max(1, (1 << 28) // (hq * length))
        for b in range(0, n, step):
            e = min(n, b + step)
            q = s["q"][at + b:at + e].float().transpose(0, 1).unflatten(0, (hkv, hq // hkv))
            scores = (q @ k) * s["scale"]
            if c["cap"]:
                scores = torch.tanh(scores / c["cap"]) * c["cap"]
            pos = torch.arange(length - n + b, length - n + e, device="cuda")[:, None]
            hidden = keys > pos
            if c["window"]:
                hidden = hidden | (keys <= pos - c["window"])
            scores = scores.masked_fill(hidden, -math.inf)
            weights = (scores - scores.amax(-1, keepdim=True)).exp()
            out = (weights @ v) / weights.sum(-1, keepdim=True)
            s["o"][at + b:at + e] = out.flatten(0, 1).transpose(0, 1).to(s["o"].dtype)
        at += n
    return s["o"]


# ------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    return _append_exact(case, seed) if case["op"] == "append" else _extend_exact(case, seed)


def _append_exact(case, seed):
    s = _append_inputs(case, seed)
    half = case["rot"] // 2
    axis_of = torch.tensor([a for a, n in enumerate(_sections(case)) for _ in range(n)], device="cuda")
    pos = s["positions"].reshape(case["axes"], -1)
    pair = torch.arange(half, device="cuda")
    where = pos[axis_of].t()                                      # [tokens, pairs]
    unit = torch.complex(s["table"].double()[where, pair], s["table"].double()[where, pair + half])[:, None]
    first = 2 * pair if case["interleaved"] else pair
    second = first + (1 if case["interleaved"] else half)

    def turned(x):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * unit
        y[..., first], y[..., second] = z.real, z.imag
        return y

    k, v = s["k_buffer"].double(), s["v_buffer"].double()
    kept = s["slots"] >= 0
    k[s["slots"][kept].long()] = turned(s["k"])[kept]
    v[s["slots"][kept].long()] = s["v"].double()[kept]
    return turned(s["q"]), k, v


def _extend_exact(case, seed):
    s = _extend_inputs(case, seed)
    hq, hkv = case["hq"], case["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    end = 0
    for r, (length, n) in enumerate(zip(s["seq"], s["new"])):
        end += n
        slots = s["table"][r, :length].long()
        age = torch.arange(length - n, length, device="cuda")[:, None] - torch.arange(length, device="cuda")
        seen = (age >= 0) & (age < (case["window"] or length))
        for h in range(hq):
            k, v = s["k"][slots, h // (hq // hkv)].double(), s["v"][slots, h // (hq // hkv)].double()
            z = torch.einsum("qd,kd->qk", s["q"][end - n:end, h].double(), k) * s["scale"]
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            z = torch.where(seen, z, torch.full_like(z, -math.inf))
            out[end - n:end, h] = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)) @ v
    return out
