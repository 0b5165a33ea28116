"""Attention that is launched early behind its trees' launch: captured and replayed with new trees, it gives what it gives with a wait
between the two."""
import pytest
import torch

import branch_cases
import fasttree
from ft_b200 import extend, lib
from test_draft_gpu import DTYPES, Step

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("cached,nodes,heads", [
    ([0], [38], (4, 4, 128)), ([0], [5], (8, 2, 64)), ([0, 3], [17, 30], (4, 4, 128)), ([100], [64], (16, 16, 64)), ([0, 0, 0], [9, 1, 40], (8, 8, 128)),
    ([60], [70], (16, 2, 256)), ([130, 10], [20, 11], (32, 8, 128))])
def test_replays_with_new_trees(cached, nodes, heads, dtype):
    s = Step(cached, nodes, [], *heads, DTYPES[dtype], seed=sum(nodes), pad_rows=0)
    steps = []
    for _ in range(8):
        trees = branch_cases.make_trees(s.rng, nodes)
        parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device="cuda")
        fasttree.fasttree_draft_tree(parents, s.plan)
        torch.cuda.synchronize()
        o = torch.empty_like(s.gq)
        extend.extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
        torch.cuda.synchronize()
        steps.append((parents, o))
    parents, o, graph = steps[0][0].clone(), torch.empty_like(s.gq), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(3):                      # trees and attention in turn
            fasttree.fasttree_draft_tree(parents, s.plan)
            fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(40):                         # without a wait on the host between replays
        new, want = steps[i * 3 % len(steps)]
        parents.copy_(new)
        o.fill_(float("nan"))
        graph.replay()
        wrong += (o != want).sum()
    assert wrong.item() == 0 and lib.read_device_status() == 0
    for new, want in steps:                     # and eagerly
        fasttree.fasttree_draft_tree(new, s.plan)
        fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
        assert torch.equal(o, want)
