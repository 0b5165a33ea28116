"""Selection and reordering one behind the other, several steps without a wait between them: the reordering, launched early, goes by
the beams that its selection chose."""
import pytest
import torch

import fasttree
from ft_b200 import lib

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("captured", [False, True])
def test_steps_in_a_row(index, captured):
    batch, beams, vocab, width, steps = 6, 8, 700, 300, 12
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(steps, batch, beams, vocab, generator=g).cuda()
    first = torch.randn(batch, beams, generator=g).cuda()
    scores, ob, ot = first.clone(), torch.zeros(batch, beams, dtype=index, device="cuda"), torch.zeros(batch, beams, dtype=index, device="cuda")
    start = torch.randint(0, 1 << 20, (batch * beams, width), generator=g, dtype=torch.int32).cuda()
    table, rows = start.clone(), torch.arange(batch * beams, device="cuda").to(index).view(batch, beams)

    def run(wait):
        for i in range(steps):
            fasttree.fasttree_beam_select(logits[i], scores, scores, ob, ot)
            if wait:
                torch.cuda.synchronize()
            fasttree.fasttree_beam_reorder(table, rows, ob)

    # what was chosen from is read by torch, step by step
    want = start.clone()
    for i in range(steps):
        fasttree.fasttree_beam_select(logits[i], scores, scores, ob, ot)
        want = want[torch.gather(rows.long(), 1, ob.long()).flatten()]
    want_scores = scores.clone()
    scores.copy_(first)
    run(True)
    assert torch.equal(table, want) and torch.equal(scores, want_scores)
    graph = torch.cuda.CUDAGraph()
    if captured:
        with torch.cuda.graph(graph):
            run(False)
    for _ in range(10):
        scores.copy_(first)
        table.copy_(start)
        graph.replay() if captured else run(False)
        assert torch.equal(table, want) and torch.equal(scores, want_scores)
    assert lib.read_device_status() == 0
