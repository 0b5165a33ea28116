"""Acceptance of drafted tokens against a walk in Python: types, sizes, ties, trees of every shape, padding, the row table."""
import ctypes
import math

import pytest
import torch

import branch_cases
import fasttree
from ft_b200 import lib

gpu = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def walk(targets, tokens, parents):
    """Path and next token; targets: the model's token behind each token."""
    sees, _ = branch_cases.paths(parents)
    if not parents or parents[0] != -1:
        return [], -1
    path = [0]
    while True:
        want = targets[path[-1]]
        at = next((i for i in range(path[-1] + 1, len(parents)) if parents[i] == path[-1] and tokens[i] == want and sees[i]), None)
        if at is None:
            return path, want
        path.append(at)


class Step:
    def __init__(self, nodes, vocab, dtype, seed=0, agree=0.7, pads=0, vary=1):
        rng = branch_cases.rng_of(seed)
        g = torch.Generator().manual_seed(seed)
        self.trees = [branch_cases.tree(rng, n, min(pads, n - 1), chain=rng.choice((0.3, 0.7, 1.0))) if n else [] for n in nodes]
        total, self.vocab = sum(nodes), vocab
        self.logits = (torch.randn(max(total, 1), vocab, generator=g) * 2).to(dtype)[:total]
        self.tokens = torch.randint(0, vocab, (total,), generator=g)
        at = 0
        for tree in self.trees:
            for i in range(len(tree)):
                kids = [j for j in range(i + 1, len(tree)) if tree[j] == i]
                if kids and rng.random() < agree:                      # the model wants one of the children
                    self.logits[at + i, self.tokens[at + rng.choice(kids)]] = 30.0
            at += len(tree)
        self.cached = [rng.choice((0, 3, rng.randint(0, 200))) for _ in nodes]
        self.width = max((c + n for c, n in zip(self.cached, nodes)), default=0) + 4
        self.slots = torch.randperm(5 * total + 1, generator=g)[:total]
        self.plan = fasttree.fasttree_extend_preparation([c + n for c, n in zip(self.cached, nodes)], nodes,
                                                         [r * self.width for r in range(len(nodes))], 8, 2, 64, torch.float16, draft=True)
        self.nodes = nodes

    def targets(self):
        x = self.logits.double()
        x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x)
        return [int((row == row.max()).nonzero()[0]) for row in x]

    def run(self, index=torch.int32, out=torch.int64, targets=None, extra=2, logits=None):
        n = len(self.nodes)
        accepted = torch.full((n, max(self.nodes, default=0) + extra), -9, dtype=torch.int32, device="cuda")
        counts, following = torch.full((n,), -9, dtype=torch.int32, device="cuda"), torch.full((n,), -9, dtype=out, device="cuda")
        table = torch.full((n, self.width), -5, dtype=torch.int32, device="cuda")
        parents = torch.tensor([p for t in self.trees for p in t], dtype=index, device="cuda")
        logits = None if targets is not None else (self.logits.cuda() if logits is None else logits)
        fasttree.fasttree_draft_accept(logits, self.tokens.to(index).cuda(), parents, self.plan, accepted, counts, following,
                                       slots=self.slots.to(index).cuda(), kv_entries=table, targets=targets)
        torch.cuda.synchronize()
        return accepted.cpu(), counts.cpu(), following.cpu(), table.cpu()

    def check(self, got, targets=None):
        accepted, counts, following, table = got
        targets = self.targets() if targets is None else targets
        at = 0
        for r, tree in enumerate(self.trees):
            n = len(tree)
            path, nxt = walk(targets[at:at + n], self.tokens[at:at + n].tolist(), tree)
            assert accepted[r].tolist() == path + [-1] * (accepted.shape[1] - len(path))
            assert counts[r] == len(path) and following[r] == nxt
            order = path + [i for i in range(n) if i not in path]
            row = [-5] * self.width
            row[self.cached[r]:self.cached[r] + n] = self.slots[at:at + n][order].tolist() if n else []
            assert table[r].tolist() == row
            at += n


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("nodes,vocab,pads", [
    ([1], 1, 0), ([1], 7, 0), ([5], 2, 0), ([16] * 9, 1000, 3), ([1, 40, 0, 3, 17], 8191, 0), ([0, 0], 50, 0), ([33, 64], 32003, 5),
    ([8] * 70, 4096, 0), ([6] * 300, 517, 1), ([4, 5], 200001, 0), ([1024], 300, 9), ([2, 1000, 700], 1025, 0)])
def test_against_a_walk(dtype, nodes, vocab, pads):
    s = Step(nodes, vocab, DTYPES[dtype], seed=vocab + len(nodes), pads=pads)
    s.check(s.run())
    assert lib.read_device_status() == 0
    s.check(s.run(index=torch.int64, out=torch.int32))
    targets = s.targets()
    for kind in (torch.int32, torch.int64):
        s.check(s.run(targets=torch.tensor(targets, dtype=kind, device="cuda")))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_rows_that_start_anywhere(dtype, offset):
    s = Step([12, 9], 1003, DTYPES[dtype], seed=offset)
    for pad in (0, 1, 7):
        store = torch.full((s.logits.shape[0], offset + 1003 + pad), 99.0, dtype=DTYPES[dtype])
        store[:, offset:offset + 1003] = s.logits
        s.check(s.run(logits=store.cuda()[:, offset:offset + 1003]))


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_equal_logits_nan_and_infinities(dtype):
    vocab = 3001
    for seed in range(4):
        s = Step([10] * 6, vocab, DTYPES[dtype], seed=seed, agree=0.0)
        s.logits = (s.logits * 0.3).round()                     # the largest many times over
        s.logits[::3, ::2] = float("nan")
        s.logits[5], s.logits[11] = -math.inf, float("nan")     # nothing to choose from: token 0
        s.logits[17, 2000:] = math.inf
        s.logits[23] = 0.0
        s.logits[23, ::2] = -0.0
        for i, t in enumerate(s.targets()):                     # a child that agrees, and a later one with the same token
            tree, at = s.trees[i // 10], i % 10
            for j in [j for j in range(at + 1, 10) if tree[j] == at][:2]:
                s.tokens[i - at + j] = t
        s.check(s.run())
    assert lib.read_device_status() == 0


@gpu
def test_only_what_hangs_on_the_path_counts():
    s = Step([6, 4, 3], 100, torch.float32, seed=1)
    # a forest: token 0 is the root that counts; children of padding; a first token that is no root; tokens outside the vocabulary
    s.trees = [[-1, -1, 0, 1, 2, -2], [-1, -2, 1, 0], [-2, 0, 0]]
    s.logits[:] = 0
    for i in range(13):
        s.logits[i, 40 + i] = 1
    s.tokens[:] = torch.tensor([0, 40, 40, 41, 42, 44, 0, 46, 47, -3, 0, 50, 50])
    got = s.run()
    assert got[0][:, :4].tolist() == [[0, 2, 4, -1], [0, -1, -1, -1], [-1, -1, -1, -1]]
    assert got[1].tolist() == [3, 1, 0] and got[2].tolist() == [44, 46, -1]
    lib.read_device_status()


@gpu
def test_the_table_may_be_left_out_and_outputs_may_be_views():
    s = Step([7, 9], 300, torch.bfloat16, seed=3)
    wide = torch.full((2, 40), -9, dtype=torch.int32, device="cuda")
    counts, following = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    parents = torch.tensor([p for t in s.trees for p in t], device="cuda")
    fasttree.fasttree_draft_accept(s.logits.cuda(), s.tokens.cuda(), parents, s.plan, wide[:, 5:20], counts, following)
    torch.cuda.synchronize()
    s.check((wide[:, 5:20].cpu(), counts.cpu(), following.cpu(), s.run()[3]))
    assert bool((wide[:, :5] == -9).all()) and bool((wide[:, 20:] == -9).all())


@gpu
def test_requests_that_share_a_prefix_keep_their_rows():
    # the plan puts requests that share together; results go by the caller's numbers
    nodes, cached = [3, 5, 4, 6], [20, 8, 20, 8]
    plan = fasttree.fasttree_extend_preparation([c + n for c, n in zip(cached, nodes)], nodes, [0, 50, 100, 150], 8, 2, 64, torch.float16,
                                                shared_prefixes=[([0, 2], 20), ([1, 3], 8)], draft=True)
    tokens = torch.zeros(18, dtype=torch.int32, device="cuda")
    targets = torch.arange(18, dtype=torch.int32, device="cuda") + 100
    parents = torch.tensor([i - 1 for n in nodes for i in range(n)], dtype=torch.int32, device="cuda")
    table, slots = torch.zeros(200, dtype=torch.int32, device="cuda"), torch.arange(18, dtype=torch.int32, device="cuda") + 1
    accepted = torch.zeros(4, 6, dtype=torch.int32, device="cuda")
    counts, following = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    fasttree.fasttree_draft_accept(None, tokens, parents, plan, accepted, counts, following, slots=slots, kv_entries=table, targets=targets)
    assert counts.tolist() == [1] * 4 and following.tolist() == [100, 103, 108, 112]
    assert table[20:23].tolist() == [1, 2, 3] and table[58:63].tolist() == [4, 5, 6, 7, 8] and table[170 - 12:164].tolist() == [13, 14, 15, 16, 17, 18]


@gpu
def test_captured_and_on_two_streams():
    a, b = Step([20] * 5, 5000, torch.float16, seed=5), Step([20] * 5, 5000, torch.float16, seed=6)
    outs, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for st, s in zip(streams, (a, b)):
        with torch.cuda.stream(st):
            outs.append(s.run())
    for out, s in zip(outs, (a, b)):
        s.check(out)
    logits, tokens = a.logits.cuda(), a.tokens.cuda()
    parents = torch.tensor([p for t in a.trees for p in t], device="cuda")
    accepted = torch.zeros(5, 20, dtype=torch.int32, device="cuda")
    counts, following = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fasttree.fasttree_draft_accept(logits, tokens, parents, a.plan, accepted, counts, following)
    for s in (b, a):
        logits.copy_(s.logits)
        tokens.copy_(s.tokens)
        parents.copy_(torch.tensor([p for t in s.trees for p in t]))
        graph.replay()
        torch.cuda.synchronize()
        s.check((accepted.cpu(), counts.cpu(), following.cpu(), s.run()[3]))


@gpu
def test_refusals():
    s = Step([3, 4], 50, torch.float16)
    lg, tk, pr = s.logits.cuda(), s.tokens.cuda(), torch.zeros(7, dtype=torch.int32, device="cuda") - 1
    acc, cnt, nxt = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    table, targets = torch.zeros(2, 300, dtype=torch.int32, device="cuda"), torch.zeros(7, dtype=torch.int64, device="cuda")
    good = dict(logits=lg, tokens=tk, parents=pr, plan=s.plan, accepted=acc, counts=cnt, next_tokens=nxt)
    fasttree.fasttree_draft_accept(**good)
    for change in ({"logits": None}, {"targets": targets}, {"logits": lg.double()}, {"logits": lg[:6]}, {"logits": lg.t()}, {"logits": lg[:, :0]}, {"tokens": tk.float()},
                   {"tokens": tk[None]}, {"parents": pr[:6]}, {"accepted": acc.long()}, {"accepted": acc[0]}, {"accepted": acc[:1].expand(2, 4)}, {"counts": cnt.long()},
                   {"counts": cnt[:1]}, {"next_tokens": nxt.float()}, {"next_tokens": nxt[:1]}, {"slots": targets}, {"kv_entries": table}, {"logits": s.logits},
                   {"slots": targets[:3], "kv_entries": table}, {"slots": targets, "kv_entries": table.long()}):
        with pytest.raises(ValueError):
            fasttree.fasttree_draft_accept(**{**good, **change})
    for change in ({"accepted": acc[:, :3]}, {"accepted": acc[:1], "counts": cnt[:1], "next_tokens": nxt[:1]},
                   {"slots": targets, "kv_entries": table.view(-1)[:5]}, {"logits": lg[:6], "tokens": tk[:6], "parents": pr[:6]}):
        with pytest.raises(lib.FastTreeError):
            fasttree.fasttree_draft_accept(**{**good, **change})


@gpu
def test_the_rows_may_stand_at_their_entries():
    for seed in range(3):
        s = Step([40], 900, torch.float16, seed=seed)
        expect = s.run()
        table = torch.full((1, s.width), -5, dtype=torch.int32, device="cuda")
        entries = table[0, s.cached[0]:s.cached[0] + 40]
        entries.copy_(s.slots)
        accepted, counts = torch.empty(1, 40, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
        fasttree.fasttree_draft_accept(s.logits.cuda(), s.tokens.cuda(), torch.tensor(s.trees[0], device="cuda"), s.plan, accepted, counts,
                                       torch.empty(1, dtype=torch.int64, device="cuda"), slots=entries, kv_entries=table)
        assert torch.equal(table.cpu(), expect[3])


@gpu
def test_results_that_overlap_what_is_read_are_refused():
    s = Step([3, 4], 50, torch.float16)
    lg, pr = s.logits.cuda(), torch.zeros(7, dtype=torch.int32, device="cuda") - 1
    big = torch.zeros(40, dtype=torch.int32, device="cuda")
    tk, acc, cnt, nxt, table = big[:7], big[8:16].view(2, 4), big[16:18], big[18:20], torch.zeros(2 * s.width, dtype=torch.int32, device="cuda")
    good = dict(logits=lg, tokens=tk, parents=pr, plan=s.plan, accepted=acc, counts=cnt, next_tokens=nxt, slots=big[20:27], kv_entries=table)
    fasttree.fasttree_draft_accept(**good)
    for change in ({"next_tokens": big[5:7]}, {"counts": big[0:2]}, {"accepted": big[4:12].view(2, 4)}, {"counts": big[12:14]}, {"next_tokens": big[17:19]},
                   {"slots": table[3:10]}, {"slots": big[14:21]}, {"parents": big[10:17]}):
        with pytest.raises(lib.FastTreeError, match="overlaps"):
            fasttree.fasttree_draft_accept(**{**good, **change})


def test_refusals_of_the_c_abi():
    handle = lib.load()
    a = lib.DraftAcceptArgs()
    assert handle.ft_draft_accept(ctypes.byref(a)) == -1 and b"drafted" in handle.ft_last_error()
    a.plan.draft, a.plan.num_drafts, a.plan.num_tokens, a.plan.longest_draft, a.plan.tile_tokens, a.plan.table_ints = 1, 1, 3, 3, 128, 64
    assert handle.ft_draft_accept(ctypes.byref(a)) == -1 and b"plan_table" in handle.ft_last_error()
    for field, bad in (("num_drafts", -1), ("num_spans", 9), ("longest_draft", 2000), ("tile_tokens", 96), ("drafts_off", 60), ("drafts_off", -4), ("spans_off", 3),
                       ("extra_off", 68)):
        b = lib.DraftAcceptArgs.from_buffer_copy(a)
        setattr(b.plan, field, bad)
        assert handle.ft_draft_accept(ctypes.byref(b)) == -1
