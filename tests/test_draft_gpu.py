"""Attention of drafted trees against the 64-bit oracle, and the trees' masks and positions in the plan."""
import pytest
import torch

import branch_cases
import extend_cases
import fasttree
from ft_b200 import extend, lib
from test_draft_plan import check_sight

gpu = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


class Step:
    def __init__(self, cached, nodes, shared, hq, hkv, d, dtype, window=0, layout="scattered", seed=0, q_scale=1.0, pad_rows=2, trees=None):
        g, self.rng = torch.Generator().manual_seed(seed), branch_cases.rng_of(seed)
        seq = [c + n for c, n in zip(cached, nodes)]
        self.table, rows = extend_cases.pool(seq, nodes, shared, layout=layout, seed=seed)
        self.k, self.v = torch.randn(rows, hkv, d, generator=g).to(dtype), torch.randn(rows, hkv, d, generator=g).to(dtype)
        self.q = (torch.randn(sum(nodes) + pad_rows, hq, d, generator=g) * q_scale).to(dtype)
        self.plan = fasttree.fasttree_extend_preparation(seq, nodes, [r * self.table.shape[1] for r in range(len(seq))], hq, hkv, d, dtype,
                                                         shared_prefixes=shared, window=window, draft=True)
        self.cached, self.nodes, self.window, self.dtype, self.d, self.scale = cached, nodes, window, dtype, d, d ** -0.5
        self.trees = trees or branch_cases.make_trees(self.rng, nodes)
        self.gq, self.gk, self.gv, self.gt = self.q.cuda(), self.k.cuda(), self.v.cuda(), self.table.cuda()

    def parents(self, dtype=torch.int32):
        return torch.tensor([p for t in self.trees for p in t] + [-1] * (self.q.shape[0] - sum(self.nodes)), dtype=dtype, device="cuda")

    def grow(self, dtype=torch.int32):
        positions = torch.full((self.q.shape[0],), -8, dtype=dtype, device="cuda")
        fasttree.fasttree_draft_tree(self.parents(dtype), self.plan, positions)
        want = [p for c, t in zip(self.cached, self.trees) for p in branch_cases.in_sight(c, t, self.window)[1]]
        assert positions.tolist() == want + [-8] * (self.q.shape[0] - len(want))

    def run(self, path="auto", cap=-1.0):
        o, lse = torch.full_like(self.gq, float("nan")), torch.full(self.q.shape[:2], float("nan"), device="cuda")
        extend.extend(self.gq, self.gk, self.gv, o, self.gt, self.plan, self.scale, logit_cap=cap, o_lse=lse, path=path)
        torch.cuda.synchronize()
        return o, lse

    def check(self, path="auto", cap=-1.0, status=0):
        o, lse = self.run(path, cap)
        assert lib.read_device_status() == status
        out, want_lse, absv, size = branch_cases.oracle(self.q, self.k, self.v, self.table, self.cached, self.trees, self.scale, cap, self.window)
        n = sum(self.nodes)
        assert o[n:].isnan().all() and lse[n:].isnan().all()
        tol, tol_lse = extend_cases.bounds(self.dtype, out, absv, size, cap, self.d)
        err = (o[:n].double().cpu() - out[:n]).abs()
        assert bool((err <= tol[:n]).all()), (err / tol[:n]).max().item()
        empty = want_lse[:n] == -float("inf")
        assert torch.equal(lse[:n].cpu() == -float("inf"), empty) and bool((o[:n].cpu()[empty] == 0).all())
        err = (lse[:n].double().cpu() - want_lse[:n]).abs()[~empty]
        assert bool((err <= tol_lse[:n][~empty]).all())


SHAPES = {
    "one": ([0], [1], []), "one_tree": ([77], [33], []), "no_prefix": ([0, 0, 0], [1, 40, 129], []),
    "borders": ([127, 128, 64, 100], [1, 2, 64, 28], []), "shared": ([199, 220, 199, 333], [10, 64, 1, 30], [([0, 1, 2, 3], 199)]),
    "tree": ([291, 293, 491, 487, 100], [9, 17, 40, 33, 5], [([0, 1], 200), ([2, 3], 470), ([0, 1, 2, 3], 100)]),
    "long": ([700, 5], [70, 257], []),
}
HEADS = [(32, 8, 128), (8, 8, 64), (16, 2, 256), (28, 4, 128), (4, 1, 32), (12, 4, 16)]


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("heads", HEADS, ids=[f"{h[0]}_{h[1]}_{h[2]}" for h in HEADS])
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_against_the_formula(shape, heads, dtype):
    cached, nodes, shared = SHAPES[shape]
    s = Step(cached, nodes, shared, *heads, DTYPES[dtype], seed=len(shape))
    s.grow()
    s.check()
    s.trees = branch_cases.make_trees(s.rng, nodes)          # the next step's trees in the same plan
    s.grow(torch.int64)
    s.check("generic" if shape != "long" else "auto")


@gpu
@pytest.mark.parametrize("heads,dtype", [((32, 8, 128), "bf16"), ((16, 4, 64), "fp16"), ((16, 8, 256), "bf16"), ((8, 2, 128), "fp32")])
@pytest.mark.parametrize("seed", range(8))
def test_windows_caps_and_padding(heads, dtype, seed):
    rng = branch_cases.rng_of(seed)
    cached, nodes, shared, _ = branch_cases.random_step(rng)
    s = Step(cached, nodes, shared, *heads, DTYPES[dtype], window=rng.choice((1, 2, 7, rng.randint(1, 300))), seed=seed, q_scale=3.0)
    s.grow()
    s.check(cap=rng.choice((-1.0, 20.0)))
    sight = s.plan.table.cpu().numpy()
    check_sight(s.plan.info, sight, s.table, cached, s.trees, s.window)


@gpu
def test_chains_are_what_plain_extend_gives():
    cached, nodes, shared = SHAPES["tree"]
    s = Step(cached, nodes, shared, 32, 8, 128, torch.bfloat16, seed=3)
    s.trees = [list(range(-1, n - 1)) for n in nodes]
    s.check()                                               # before any tree is known, too
    s.grow()
    s.check()


@gpu
def test_bad_parents_are_padding():
    s = Step([30, 0], [8, 5], [], 8, 2, 128, torch.float16, trees=[[-1, 5, 0, 1, -7, 2, 1 << 20, 3], [-2, 0, -1, 2, 3]])
    fasttree.fasttree_draft_tree(s.parents(), s.plan)
    torch.cuda.synchronize()
    assert lib.read_device_status() == lib.FT_DEV_BAD_PARENT
    s.check()                                               # (branch_cases.paths takes them the same way)
    far = s.parents(torch.int64)
    far[3] = -(1 << 40)
    fasttree.fasttree_draft_tree(far, s.plan)
    torch.cuda.synchronize()
    assert lib.read_device_status() == lib.FT_DEV_BAD_PARENT


@gpu
@pytest.mark.parametrize("parents", ["chain", "star", "random"])
def test_the_longest_drafts(parents):
    n = lib.FT_MAX_DRAFT
    rng = branch_cases.rng_of(1)
    trees = [{"chain": list(range(-1, n - 1)), "star": [-1] + [0] * (n - 1), "random": branch_cases.tree(rng, n)}[parents]]
    s = Step([100], [n], [], 2, 1, 64, torch.float16, trees=trees)
    s.grow()
    s.check()
    check_sight(s.plan.info, s.plan.table.cpu().numpy(), s.table, [100], trees, 0)


@gpu
def test_nan_and_infinities_out_of_sight():
    # rows of siblings hold infinities and NaN: none of them reaches a token that does not see them
    s = Step([40, 200], [30, 50], [], 16, 4, 128, torch.bfloat16, trees=[[-1] + [0] * 29, [-1] + [0, 0] + [1] * 47], seed=4)
    s.grow()
    clean, _ = s.run()
    for r, row in ((0, 5), (1, 2), (1, 30)):
        slot = s.table[r, s.cached[r] + row]
        s.gk[slot], s.gv[slot] = float("inf"), float("nan")
    dirty, _ = s.run()
    first = [5, 30 + 2, 30 + 30]
    keep = torch.tensor([i not in first for i in range(80)])
    same = dirty[:80].cpu()[keep]
    tol, _ = extend_cases.bounds(s.dtype, *[x for x in branch_cases.oracle(s.q, s.k, s.v, s.table, s.cached, s.trees, s.scale, -1.0, 0) if x.dim() == 3], torch.zeros(82, 16, dtype=torch.float64), -1.0, 128)
    assert bool(same.isfinite().all()) and bool(((same.double() - clean[:80].cpu()[keep].double()).abs() <= 2 * tol[:80][keep]).all())


@gpu
def test_captured_step_with_new_trees():
    s = Step([150, 90, 300], [20, 33, 9], [], 32, 8, 128, torch.float16, seed=5)
    o, parents = torch.empty_like(s.gq), s.parents()
    positions = torch.empty(s.q.shape[0], dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    extend.extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fasttree.fasttree_draft_tree(parents, s.plan, positions)
        fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
    for _ in range(3):
        s.trees = branch_cases.make_trees(s.rng, s.nodes)
        parents.copy_(s.parents())
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone()
        s.grow()
        want, _ = s.run()
        assert torch.equal(got[:62], want[:62]) and positions[:62].tolist() == [p for c, t in zip(s.cached, s.trees) for p in branch_cases.in_sight(c, t, 0)[1]]


@gpu
def test_captured_behind_copies():
    # launches that may start early, with a copy instead of a kernel before them
    s = Step([150, 90], [20, 33], [], 32, 8, 128, torch.float16, seed=6)
    s.grow()
    want, _ = s.run()
    q, o = torch.zeros_like(s.gq), torch.empty_like(s.gq)
    rows = torch.arange(6, device="cuda").view(2, 3)
    beams, source = torch.tensor([[2, 0, 1], [1, 1, 0]], device="cuda"), torch.arange(600, device="cuda").view(6, 100)
    table, graph = torch.zeros_like(source), torch.cuda.CUDAGraph()
    extend.extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        q.copy_(s.gq)
        fasttree.fasttree_extend(q, s.gk, s.gv, o, s.gt, s.plan, s.scale)
        table.copy_(source)
        fasttree.fasttree_beam_reorder(table, rows, beams)
    for _ in range(3):
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o[:53], want[:53]) and torch.equal(table, source[torch.gather(rows, 1, beams).flatten()])


@gpu
def test_refusals():
    s = Step([3], [4], [], 8, 2, 128, torch.float16, pad_rows=0)
    good = s.parents()
    for bad in (good.float(), good.cpu(), good[None], None):
        with pytest.raises(ValueError):
            fasttree.fasttree_draft_tree(bad, s.plan)
    for bad in (good[:2], good.float()):
        with pytest.raises(ValueError):
            fasttree.fasttree_draft_tree(good, s.plan, bad)
    both = torch.zeros(7, dtype=torch.int32, device="cuda") - 1
    for bad in (both[:4], both[3:], both[2:6]):
        with pytest.raises(lib.FastTreeError, match="overlaps"):
            fasttree.fasttree_draft_tree(both[:4], s.plan, bad)
    with pytest.raises(lib.FastTreeError):
        fasttree.fasttree_draft_tree(good[:3], s.plan)
    empty = fasttree.fasttree_extend_preparation([5], [0], [0], 8, 2, 128, torch.float16, draft=True)
    fasttree.fasttree_draft_tree(good[:0], empty)
    none = fasttree.fasttree_extend_preparation([], [], [], 8, 2, 128, torch.float16, draft=True)
    fasttree.fasttree_draft_tree(good[:0], none, good[:0])
