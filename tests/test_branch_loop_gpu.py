"""The operators for branching continuations together, as a serving loop runs them: greedy decoding from drafted trees, and beam search,
of a one-layer model with random weights over the paged cache, against the same model in 64 bits over whole sequences."""
import math

import pytest
import torch

import branch_cases
import fasttree
from ft_b200 import lib

pytestmark = pytest.mark.gpu
VOCAB, HIDDEN, HQ, HKV, D = 89, 48, 4, 2, 64


class Model:
    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        w = lambda *s: torch.randn(*s, generator=g) / s[0] ** 0.5
        self.embed, self.out = torch.randn(VOCAB, HIDDEN, generator=g), w(HIDDEN, VOCAB) * 3
        self.wq, self.wk, self.wv, self.wo = w(HIDDEN, HQ * D), w(HIDDEN, HKV * D), w(HIDDEN, HKV * D), w(HQ * D, HIDDEN) * 2
        angle = torch.outer(torch.arange(512.0), 10000.0 ** (-torch.arange(D // 2) / (D // 2)))
        self.table = torch.cat([angle.cos(), angle.sin()], 1)
        self.gpu = {n: getattr(self, n).cuda() for n in ("embed", "out", "wq", "wk", "wv", "wo", "table")}

    def exact(self, tokens):
        """Logits behind the last token, in 64 bits."""
        n = len(tokens)
        x = self.embed[tokens].double()
        c, s = self.table[:n, :D // 2].double()[:, None], self.table[:n, D // 2:].double()[:, None]
        turn = lambda y: torch.cat([y[..., :D // 2] * c - y[..., D // 2:] * s, y[..., D // 2:] * c + y[..., :D // 2] * s], -1)
        q, k, v = (turn((x @ self.wq.double()).view(n, HQ, D))[-1], turn((x @ self.wk.double()).view(n, HKV, D)), (x @ self.wv.double()).view(n, HKV, D))
        k, v = k.repeat_interleave(HQ // HKV, 1), v.repeat_interleave(HQ // HKV, 1)
        p = torch.softmax(torch.einsum("hd,khd->hk", q, k) * D ** -0.5, -1)
        return (x[-1] + torch.einsum("hk,khd->hd", p, v).reshape(-1) @ self.wo.double()) @ self.out.double()

    def step(self, cache, tokens, slots, positions, table, plan):
        """Logits behind each of the step's tokens, whose keys and values enter the cache."""
        w = self.gpu
        x = w["embed"][tokens]
        q, k, v = (x @ w["wq"]).view(-1, HQ, D), (x @ w["wk"]).view(-1, HKV, D), (x @ w["wv"]).view(-1, HKV, D)
        fasttree.fasttree_append(q, k, v, *cache, slots, positions=positions, cos_sin=w["table"])
        o = torch.empty_like(q)
        fasttree.fasttree_extend(q, *cache, o, table, plan, D ** -0.5)
        return (x + o.flatten(1) @ w["wo"]) @ w["out"]

    def prefill(self, cache, prompts, table, shared):
        """All tokens but the last of each prompt into the cache, the shared ones once."""
        slot = 0
        for r, prompt in enumerate(prompts):
            n = len(prompt) - 1
            own = list(range(slot, slot + (n if r == 0 else n - shared)))
            slot += len(own)
            table[r, :n] = torch.tensor(own if r == 0 else table[0, :shared].tolist() + own, dtype=torch.int32)
            start = 0 if r == 0 else shared
            plan = fasttree.fasttree_extend_preparation([n], [n - start], [r * table.shape[1]], HQ, HKV, D, torch.float32)
            self.step(cache, torch.tensor(prompt[start:n], device="cuda"), torch.tensor(own, device="cuda"), torch.arange(start, n, device="cuda"), table, plan)
        return slot


def test_greedy_decoding_from_drafted_trees():
    torch.backends.cuda.matmul.allow_tf32 = False
    model, rng = Model(1), branch_cases.rng_of(2)
    shared, wanted = 21, 14
    common = [rng.randrange(VOCAB) for _ in range(shared)]
    prompts = [common + [rng.randrange(VOCAB) for _ in range(n)] for n in (2, 5, 9)]
    greedy = []
    for p in prompts:
        seq = list(p)
        for _ in range(wanted + 8):
            top = torch.topk(model.exact(seq), 2)
            assert top.values[0] - top.values[1] > 1e-3        # what follows does not hang on a rounding
            seq.append(int(top.indices[0]))
        greedy.append(seq[len(p):])
    table = torch.zeros(3, 200, dtype=torch.int32, device="cuda")
    cache = [torch.zeros(400, HKV, D, device="cuda") for _ in range(2)]
    slot = model.prefill(cache, prompts, table, shared)
    cached, certain, done, steps = [len(p) - 1 for p in prompts], [p[-1] for p in prompts], [[], [], []], 0
    while min(len(d) for d in done) < wanted:
        # drafts: what the model will say for some steps, with wrong tokens beside and behind
        trees, tokens = [], []
        for r in range(3):
            ahead = greedy[r][len(done[r]):]
            tree, ids, at = [-1], [certain[r]], 0
            for t in ahead[:rng.randrange(4)]:
                if rng.random() < 0.5:
                    tree.append(at)
                    ids.append((t + 1) % VOCAB)
                tree.append(at)
                ids.append(t)
                at = len(tree) - 1
            for _ in range(rng.randrange(3)):
                tree.append(rng.randrange(len(tree)))
                ids.append(rng.randrange(VOCAB))
            trees.append(tree + [-2] * rng.randrange(2))
            tokens.append(ids + [0] * (len(trees[-1]) - len(ids)))
        nodes = [len(t) for t in trees]
        total = sum(nodes)
        slots = torch.arange(slot, slot + total, device="cuda")
        slot += total
        at = 0
        for r, n in enumerate(nodes):
            table[r, cached[r]:cached[r] + n] = slots[at:at + n].int()
            at += n
        plan = fasttree.fasttree_extend_preparation([c + n for c, n in zip(cached, nodes)], nodes, [r * 200 for r in range(3)], HQ, HKV, D,
                                                    torch.float32, shared_prefixes=[([0, 1, 2], shared)], draft=True)
        parents = torch.tensor([p for t in trees for p in t], device="cuda")
        ids = torch.tensor([x for t in tokens for x in t], device="cuda")
        positions = torch.empty(total, dtype=torch.int64, device="cuda")
        fasttree.fasttree_draft_tree(parents, plan, positions)
        logits = model.step(cache, ids, slots, positions, table, plan)
        accepted = torch.empty(3, max(nodes), dtype=torch.int32, device="cuda")
        counts, following = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda")
        fasttree.fasttree_draft_accept(logits, ids, parents, plan, accepted, counts, following, slots=slots, kv_entries=table)
        for r in range(3):
            path = accepted[r, :int(counts[r])].tolist()
            done[r] += [tokens[r][i] for i in path[1:]] + [int(following[r])]
            cached[r] += len(path)
            certain[r] = int(following[r])
        steps += 1
    assert lib.read_device_status() == 0
    for r in range(3):
        assert done[r][:wanted] == greedy[r][:wanted]
    assert steps < wanted                                       # some drafts were accepted


def test_beam_search():
    torch.backends.cuda.matmul.allow_tf32 = False
    model, rng = Model(3), branch_cases.rng_of(4)
    beams, length, shared = 3, 7, 11
    common = [rng.randrange(VOCAB) for _ in range(shared)]
    prompts = [common + [rng.randrange(VOCAB) for _ in range(n)] for n in (3, 6)]
    expect = []
    for p in prompts:
        live = [(0.0, list(p))]
        for _ in range(length):
            options = sorted(((s + x, b, t) for b, (s, seq) in enumerate(live) for t, x in enumerate(torch.log_softmax(model.exact(seq), -1).tolist())),
                             key=lambda o: (-o[0], o[1], o[2]))
            assert options[beams - 1][0] - options[beams][0] > 1e-4
            live = [(s, live[b][1] + [t]) for s, b, t in options[:beams]]
        expect.append(live)
    rows = torch.arange(2 * beams, device="cuda").view(2, beams)
    table = torch.zeros(2 * beams, 64, dtype=torch.int32, device="cuda")
    history = torch.zeros(2 * beams, length, dtype=torch.int64, device="cuda")
    cache = [torch.zeros(300, HKV, D, device="cuda") for _ in range(2)]
    first = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    slot = model.prefill(cache, prompts, first, shared)
    table.copy_(first.repeat_interleave(beams, 0))             # the beams' rows share what is cached
    cached = [len(p) - 1 for p in prompts for _ in range(beams)]
    tokens = torch.tensor([p[-1] for p in prompts for _ in range(beams)], device="cuda")
    scores = torch.tensor([[0.0] + [-math.inf] * (beams - 1)] * 2, device="cuda")
    out, ob, ot = torch.empty(2, beams, device="cuda"), torch.empty(2, beams, dtype=torch.int64, device="cuda"), torch.empty(2, beams, dtype=torch.int64, device="cuda")
    for step in range(length):
        slots = torch.arange(slot, slot + 2 * beams, device="cuda")
        slot += 2 * beams
        at = torch.tensor(cached, device="cuda")
        table[torch.arange(2 * beams, device="cuda"), at] = slots.int()
        cached = [c + 1 for c in cached]
        groups = [([b for b in range(r * beams, r * beams + beams)], len(prompts[r]) - 1) for r in range(2)]
        plan = fasttree.fasttree_extend_preparation(cached, [1] * (2 * beams), [i * 64 for i in range(2 * beams)], HQ, HKV, D, torch.float32,
                                                    shared_prefixes=groups + [(list(range(2 * beams)), shared)])
        logits = model.step(cache, tokens, slots, at, table, plan)
        fasttree.fasttree_beam_select(logits.view(2, beams, VOCAB), scores, out, ob, ot)
        ends = torch.tensor([cached[0], cached[beams]], device="cuda")
        fasttree.fasttree_beam_reorder(table, rows, ob, ends=ends)
        fasttree.fasttree_beam_reorder(history, rows, ob, ends=torch.full((2,), step, device="cuda"))
        history[:, step] = ot.flatten()
        tokens, scores = ot.flatten().clone(), out.clone()
    assert lib.read_device_status() == 0
    for r in range(2):
        got = history.view(2, beams, length)[r].tolist()
        assert got == [seq[len(prompts[r]):] for _, seq in expect[r]]
        for s, (want, _) in zip(scores[r].tolist(), expect[r]):
            # fp32 through the model: sums of up to 256 products of numbers of order 1, `length` times
            assert abs(s - want) < length * 256 * 2.0 ** -20
