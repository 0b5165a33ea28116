"""Beam selection and reordering against the definition in 64 bits: types, sizes, strides, ties, banned tokens, ended beams."""
import ctypes
import math

import pytest
import torch

import fasttree
from ft_b200 import lib

gpu = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def want(logits, scores, best):
    """Scores in 64 bits, beams and tokens, by sorting everything."""
    x, s = logits.double().cpu(), scores.double().cpu()
    lse = torch.logsumexp(x, -1, keepdim=True)
    dead = ~(torch.isfinite(lse) & torch.isfinite(s[..., None]))
    score = s[..., None] + (x - lse)
    score = torch.where(dead | (x == -math.inf), torch.full_like(score, -math.inf), score)
    batch, beams, vocab = x.shape
    out = torch.full((batch, best), -math.inf, dtype=torch.float64)
    ob, ot = torch.full((batch, best), -1), torch.full((batch, best), -1)
    for r in range(batch):
        flat = score[r].flatten()
        order = torch.sort(flat, descending=True, stable=True).indices[:best]
        order = order[flat[order] > -math.inf]
        n = order.numel()
        out[r, :n], ob[r, :n], ot[r, :n] = flat[order], order // vocab, order % vocab
    return out, ob, ot


def select(logits, scores, best, dtype=torch.int32):
    batch = logits.shape[0]
    out = torch.full((batch, best), float("nan"), device="cuda")
    ob, ot = torch.full((batch, best), -7, dtype=dtype, device="cuda"), torch.full((batch, best), -7, dtype=dtype, device="cuda")
    fasttree.fasttree_beam_select(logits, scores, out, ob, ot)
    torch.cuda.synchronize()
    assert lib.read_device_status() == 0
    return out, ob, ot


def check(logits, scores, best, dtype=torch.int32):
    out, ob, ot = select(logits, scores, best, dtype)
    ws, wb, wt = want(logits, scores, best)
    assert torch.equal(ob.cpu().long(), wb) and torch.equal(ot.cpu().long(), wt)
    # the logarithm: a sum of exponentials, each within 2^-21 (argument up to 2^7 in the power of two, half a step of it, and the
    # function), and of fp32 sums of at most 128 in a chain; then one rounding of the score
    live = ws > -math.inf
    err = (out.cpu().double() - ws)[live].abs()
    assert bool((err <= 2.0 ** -24 * ws[live].abs() + 2.0 ** -17).all()), err.max().item()
    assert bool((out.cpu()[~live] == -math.inf).all())


def inputs(batch, beams, vocab, dtype, seed=0, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(batch, beams, vocab, generator=g) * spread).to(dtype).cuda(), (torch.randn(batch, beams, generator=g) - 5).cuda()


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("batch,beams,vocab,best", [
    (1, 1, 1, 1), (1, 1, 1, 4), (3, 2, 5, 8), (2, 4, 7, 64), (5, 4, 1000, 8), (2, 3, 2047, 3), (2, 3, 2049, 6), (1, 4, 32000, 8),
    (3, 1, 50021, 1), (2, 16, 8193, 32), (1, 64, 1111, 64), (1, 2, 300001, 5), (40, 5, 4096, 10), (7, 8, 65536, 17)])
def test_against_the_definition(dtype, batch, beams, vocab, best):
    check(*inputs(batch, beams, vocab, DTYPES[dtype], seed=vocab), best, torch.int64 if vocab % 2 else torch.int32)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("vocab", [3, 700, 1500, 5000, 40000])
def test_ties_go_to_the_lowest(dtype, vocab):
    logits, scores = inputs(3, 4, vocab, DTYPES[dtype], seed=1)
    logits = (logits * 0.4).round()                    # a handful of values: thousands of equal ones
    logits[1] = 0.25                                   # all of them
    scores[1] = -2.0
    logits[2, 1], scores[2, 1] = logits[2, 0], scores[2, 0]       # two beams alike
    check(logits, scores, 8)
    check(logits, scores, 33)


@gpu
@pytest.mark.parametrize("vocab", [9, 6001, 70000])
def test_banned_tokens_and_ended_beams(vocab):
    logits, scores = inputs(6, 3, vocab, torch.bfloat16, seed=2)
    keep = torch.randperm(vocab, generator=torch.Generator().manual_seed(3))[:5].cuda()
    mask = torch.ones(vocab, dtype=torch.bool, device="cuda")
    mask[keep] = False
    logits[0].masked_fill_(mask, -math.inf)            # five tokens left per beam
    logits[1, 0] = -math.inf                           # nothing from this beam
    logits[2] = -math.inf                              # nothing at all
    scores[3, 1], scores[3, 2] = -math.inf, float("nan")
    scores[4, 0] = math.inf
    logits[5, 0, 1], logits[5, 1, 2] = float("nan"), math.inf
    check(logits, scores, 16)
    half = logits.clone()
    half[:, :, : vocab // 2] = -math.inf               # nothing in the first chunks
    check(half, scores, 4)


@gpu
def test_the_first_step_starts_from_one_beam():
    logits, scores = inputs(2, 4, 3001, torch.float16, seed=4)
    logits[:, 1:], scores[:] = logits[:, :1], -math.inf
    scores[:, 0] = 0
    check(logits, scores, 4)


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("offset,pad", [(0, 3), (1, 0), (3, 8), (8, 8)])
def test_strides(dtype, offset, pad):
    batch, beams, vocab, best = 3, 2, 5000, 6
    g = torch.Generator().manual_seed(5)
    store = torch.randn(beams, batch, vocab + pad + offset, generator=g).to(DTYPES[dtype]).cuda()
    logits = store[..., offset:offset + vocab].transpose(0, 1)
    scores = torch.randn(beams, batch, generator=g).cuda().t()
    wide = torch.full((batch, 2 * best), -7, dtype=torch.int64, device="cuda")
    out = torch.full((batch, best + 3), 9.0, device="cuda")
    fasttree.fasttree_beam_select(logits, scores, out[:, :best], wide[:, :best], wide[:, best:])
    ws, wb, wt = want(logits, scores, best)
    assert torch.equal(wide[:, :best].cpu(), wb) and torch.equal(wide[:, best:].cpu(), wt)
    assert bool((out[:, best:] == 9).all()) and (out[:, :best].cpu().double() - ws).abs().max().item() < 1e-5


@gpu
def test_large_logits_and_far_scores():
    for dtype, big in ((torch.float32, 1e30), (torch.bfloat16, 1e30), (torch.float16, 6e4), (torch.float32, 300.0)):
        logits, scores = inputs(2, 2, 3000, dtype, seed=6)
        logits[0, 0] *= 100
        logits[1, 0, 7] = big
        logits[1, 1] -= 3e4 if dtype == torch.float16 else 1e5
        out, ob, ot = select(logits, scores * 1000, 5)
        _, wb, wt = want(logits, scores * 1000, 5)
        assert torch.equal(ob.cpu().long()[:, 0], wb[:, 0]) and torch.equal(ot.cpu().long()[:, 0], wt[:, 0])
        assert not out.isnan().any()


@gpu
def test_two_calls_at_once_and_in_graphs():
    a, b = inputs(8, 4, 20000, torch.bfloat16, seed=7), inputs(8, 4, 20000, torch.bfloat16, seed=8)
    wants = [want(*x, 8) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        outs = []
        for st, x in zip(streams, (a, b)):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                out = torch.empty(8, 8, device="cuda"), torch.empty(8, 8, dtype=torch.int32, device="cuda"), torch.empty(8, 8, dtype=torch.int32, device="cuda")
                fasttree.fasttree_beam_select(*x, *out)
                outs.append(out)
        torch.cuda.synchronize()
        for out, w in zip(outs, wants):
            assert torch.equal(out[1].cpu().long(), w[1]) and torch.equal(out[2].cpu().long(), w[2])
    logits, scores = (x.clone() for x in a)
    graph, out = torch.cuda.CUDAGraph(), (torch.empty(8, 8, device="cuda"), torch.empty(8, 8, dtype=torch.int32, device="cuda"),
                                          torch.empty(8, 8, dtype=torch.int32, device="cuda"))
    table = torch.arange(64 * 50, dtype=torch.int32, device="cuda").view(64, 50)
    rows = torch.arange(64, device="cuda").view(8, 8)
    fasttree.fasttree_beam_select(logits, scores, *out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fasttree.fasttree_beam_select(logits, scores, *out)
        fasttree.fasttree_beam_reorder(table, rows, out[1])
    for x, w in ((b, wants[1]), (a, wants[0])):
        logits.copy_(x[0])
        scores.copy_(x[1])
        before = table.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[1].cpu().long(), w[1]) and torch.equal(out[2].cpu().long(), w[2])
        assert torch.equal(table, before[torch.gather(rows, 1, out[1].long())].reshape(64, 50))


def moved(table, rows, beams, starts, ends, out_rows):
    new = table.clone()
    for r in range(rows.shape[0]):
        lo, hi = (int(starts[r]) if starts is not None else 0), (int(ends[r]) if ends is not None else table.shape[1])
        for j in range(beams.shape[1]):
            if beams[r, j] >= 0 and lo < hi:
                new[out_rows[r, j], lo:hi] = table[rows[r, beams[r, j]], lo:hi]
    return new


@gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("batch,n,to,width", [(1, 1, 1, 1), (3, 4, 4, 5000), (2, 64, 64, 777), (5, 3, 7, 4097), (4, 16, 2, 1), (2, 5, 5, 20011)])
@pytest.mark.parametrize("in_place", [True, False])
def test_reorder(dtype, index, batch, n, to, width, in_place):
    if in_place and to != n:
        to = n
    g = torch.Generator().manual_seed(batch + width)
    count = batch * (n + to) + 3
    store = torch.randint(0, 1 << 20, (count, width + 5), generator=g).to(dtype).cuda()
    table = store[:, 2:2 + width]
    some = torch.randperm(count, generator=g).to(index)
    rows = some[:batch * n].view(batch, n).cuda()
    out_rows = rows if in_place else some[batch * n:batch * (n + to)].view(batch, to).cuda()
    beams = torch.randint(-1, n, (batch, to), generator=g).to(index).cuda()
    starts = torch.randint(0, width + 1, (batch,), generator=g).to(index).cuda()
    ends = torch.randint(0, width + 1, (batch,), generator=g).to(index).cuda()
    for s, e in ((None, None), (starts, ends), (None, ends)):
        expect, outside = moved(table, rows, beams, s, e, out_rows), store.clone()
        fasttree.fasttree_beam_reorder(table, rows, beams, starts=s, ends=e, out_rows=None if in_place else out_rows)
        torch.cuda.synchronize()
        assert torch.equal(table, expect)
        assert torch.equal(store[:, :2], outside[:, :2]) and torch.equal(store[:, 2 + width:], outside[:, 2 + width:])
    assert lib.read_device_status() == 0


@gpu
def test_rows_and_columns_outside_the_table_are_left_out():
    table = torch.arange(60, dtype=torch.int32, device="cuda").view(6, 10)
    rows = torch.tensor([[0, 1], [2, 9], [4, 5]], device="cuda")
    beams = torch.tensor([[1, 2], [1, 0], [1, -5]], device="cuda")
    out_rows = torch.tensor([[0, 1], [2, -3], [5, 4]], device="cuda")
    before = table.clone()
    for starts, ends in ((None, None), (torch.tensor([-4, 1 << 40, 3], device="cuda"), torch.tensor([99, 5, -(1 << 50)], device="cuda"))):
        table.copy_(before)
        fasttree.fasttree_beam_reorder(table, rows, beams, starts=starts, ends=ends, out_rows=out_rows)
        assert lib.read_device_status() == lib.FT_DEV_BAD_ROW_INDEX
        expect = before.clone()
        expect[0] = before[1]
        assert torch.equal(table, expect)


@gpu
def test_other_rows_of_the_table_take_part_in_nothing():
    table = torch.arange(40, dtype=torch.int64, device="cuda").view(4, 10)
    before = table.clone()
    fasttree.fasttree_beam_reorder(table, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, dtype=torch.int32, device="cuda"))
    fasttree.fasttree_beam_reorder(table[:0], torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda"))
    empty = torch.empty(0, 8, device="cuda"), torch.empty(0, 8, dtype=torch.int32, device="cuda"), torch.empty(0, 8, dtype=torch.int32, device="cuda")
    fasttree.fasttree_beam_select(torch.empty(0, 4, 100, device="cuda"), torch.empty(0, 4, device="cuda"), *empty)
    torch.cuda.synchronize()
    assert lib.read_device_status() == 0 and torch.equal(table, before)


@gpu
def test_refusals():
    x, s = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    out, ob, ot = torch.zeros(2, 4, device="cuda"), torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    wide = torch.zeros(2, 65, device="cuda")
    for args in ((x.double(), s, out, ob, ot), (x[0], s, out, ob, ot), (x, s[:, :2], out, ob, ot), (x, s.half(), out, ob, ot), (x.cpu(), s, out, ob, ot),
                 (x.transpose(1, 2), s, out, ob, ot), (x, s, out, ob[:, :3], ot), (x, s, out, ob.float(), ot), (x, s, out[:1], ob, ot),
                 (x, s, out[:1].expand(2, 4), ob, ot), (None, s, out, ob, ot)):
        with pytest.raises(ValueError):
            fasttree.fasttree_beam_select(*args)
    for args in ((x, s, wide, wide.int(), wide.int()), (torch.zeros(2, 65, 9, device="cuda"), wide, out, ob, ot), (x[..., :0], s, out, ob, ot),
                 (x, s, out[:, :0], ob[:, :0], ot[:, :0])):
        with pytest.raises(lib.FastTreeError):
            fasttree.fasttree_beam_select(*args)
    table, rows = torch.zeros(8, 10, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for args, kw in (((table.half(), rows, rows), {}), ((table.t(), rows, rows), {}), ((table, rows.float(), rows), {}), ((table, rows, rows[:1]), {}),
                     ((table, rows, rows[:, :2]), {}), ((table, rows, rows), {"starts": rows}), ((table, rows, rows), {"ends": torch.zeros(3, dtype=torch.int32, device="cuda")}),
                     ((table, rows[0], rows), {}), ((table[:1].expand(8, 10), rows, rows), {})):
        with pytest.raises(ValueError):
            fasttree.fasttree_beam_reorder(*args, **kw)
    many = torch.zeros(1, 65, dtype=torch.int32, device="cuda")
    with pytest.raises(lib.FastTreeError):
        fasttree.fasttree_beam_reorder(table, many, many)


@gpu
def test_scores_in_place():
    logits, scores = inputs(30, 4, 7000, torch.bfloat16, seed=9)
    out, ob, ot = select(logits, scores, 4)
    again = scores.clone()
    fasttree.fasttree_beam_select(logits, again, again, ob.clone(), ot.clone())
    wide = torch.zeros(30, 9, device="cuda")
    wide[:, :4] = scores
    fasttree.fasttree_beam_select(logits, wide[:, :4], wide[:, :4], ob.clone(), ot.clone())
    assert torch.equal(again, out) and torch.equal(wide[:, :4], out) and bool((wide[:, 4:] == 0).all())
    out, ob, ot = select(logits, scores, 9)
    wide[:, :4] = scores
    fasttree.fasttree_beam_select(logits, wide[:, :4], wide, ob.clone(), ot.clone())
    assert torch.equal(wide, out)


@gpu
def test_results_that_overlap_what_is_read_are_refused():
    logits, scores = inputs(3, 4, 100, torch.float32, seed=9)
    big = torch.zeros(100, device="cuda")
    ints = torch.zeros(100, dtype=torch.int32, device="cuda")
    out, ob, ot = big[50:62].view(3, 4), ints[:12].view(3, 4), ints[12:24].view(3, 4)
    for args in ((logits, scores, logits[:, :, :4][:, 0], ob, ot), (logits, big[:12].view(3, 4), big[4:16].view(3, 4), ob, ot),
                 (logits, big[:24].view(3, 8)[:, ::2], big[:24].view(3, 8)[:, :4], ob, ot),
                 (logits, scores, out, ob, ints[4:16].view(3, 4)), (logits, scores, ints.view(torch.float32)[:12].view(3, 4), ob, ot)):
        with pytest.raises(lib.FastTreeError, match="overlap"):
            fasttree.fasttree_beam_select(*args)
    table = torch.zeros(6, 10, dtype=torch.int32, device="cuda")
    rows = torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2)
    for args, kw in (((table, table[:2, :2], rows), {}), ((table, rows, table[2:4, 3:5]), {}), ((table, rows, rows), {"starts": table[0, :2]}),
                     ((table, rows, rows), {"ends": table[5, 8:]}), ((table, rows, rows), {"out_rows": table[:2, :2]})):
        with pytest.raises(lib.FastTreeError, match="overlap"):
            fasttree.fasttree_beam_reorder(*args, **kw)


def test_refusals_of_the_c_abi():
    handle = lib.load()
    a = lib.BeamSelectArgs()
    a.dtype, a.batch, a.beams, a.vocab, a.best = 1, 2, 4, 1000, 8
    size = handle.ft_beam_select_workspace(ctypes.byref(a))
    assert size > 0 and handle.ft_beam_select(ctypes.byref(a)) == -1 and b"NULL" in handle.ft_last_error()
    a.batch = 0
    assert handle.ft_beam_select(ctypes.byref(a)) == 0
    for field, bad in (("dtype", 9), ("batch", -1), ("beams", 65), ("beams", 0), ("best", 65), ("best", 0), ("vocab", 0)):
        b = lib.BeamSelectArgs.from_buffer_copy(a)
        setattr(b, field, bad)
        assert handle.ft_beam_select(ctypes.byref(b)) == -1 and handle.ft_beam_select_workspace(ctypes.byref(b)) == -1
    r = lib.BeamReorderArgs()
    r.elem_bytes, r.batch, r.from_, r.to, r.table_rows, r.width = 4, 1, 2, 2, 4, 4
    assert handle.ft_beam_reorder(ctypes.byref(r)) == -1 and b"NULL" in handle.ft_last_error()
    for field, bad in (("elem_bytes", 2), ("batch", -1), ("from_", 0), ("to", 65), ("width", -1), ("table_rows", -1)):
        b = lib.BeamReorderArgs.from_buffer_copy(r)
        setattr(b, field, bad)
        assert handle.ft_beam_reorder(ctypes.byref(b)) == -1


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_logits_in_rising_order_and_lists_that_overflow(dtype):
    # every chunk holds larger logits than the ones before it, so each reaches the bound as a whole; then thousands of equal ones
    vocab = 90001
    rising = torch.linspace(-20, 20, vocab).to(DTYPES[dtype])
    plateau = torch.where(torch.arange(vocab) % 3 == 0, torch.tensor(4.0), torch.tensor(-3.0)).to(DTYPES[dtype])
    late = torch.full((vocab,), -math.inf)
    late[60000:] = torch.randn(vocab - 60000, generator=torch.Generator().manual_seed(1))
    rows = torch.stack([rising, plateau, late.to(DTYPES[dtype]), rising.flip(0)])
    logits = rows.repeat(60, 1).view(60, 4, vocab).cuda()
    scores = torch.linspace(-3, 0, 240).view(60, 4).cuda()
    for best in (1, 8, 64):
        out, ob, ot = select(logits, scores, best)
        _, wb, wt = want(logits[:2], scores[:2], best)
        assert torch.equal(ob[:2].cpu().long(), wb) and torch.equal(ot[:2].cpu().long(), wt)
        assert bool((ot == ot[:1]).all())          # the same logits for every request


@gpu
def test_many_short_rows_in_a_cta():
    for batch, beams, vocab in ((900, 3, 300), (2000, 1, 77), (300, 64, 40)):
        logits, scores = inputs(batch, beams, vocab, torch.bfloat16, seed=vocab)
        scores[::7, 0] = -math.inf
        check(logits, scores, 5)
