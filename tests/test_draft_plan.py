"""Plans for drafted trees, checked on the host: what every token is shown, before and after its tree is known."""
import ctypes

import numpy as np
import pytest
import torch

import branch_cases
import extend_cases
import fasttree
from ft_b200 import extend, lib


def plan_of(cached, nodes, shared, hq, hkv, d, dtype=torch.float16, window=0, sms=148):
    seq = [c + n for c, n in zip(cached, nodes)]
    table, _ = extend_cases.pool(seq, nodes, shared)
    info, plan, _, _ = extend.host_plan(seq, nodes, [r * table.shape[1] for r in range(len(seq))], hq, hkv, d, dtype,
                                        shared_prefixes=shared, window=window, num_sms=sms, draft=True)
    return info, plan, table


def grow(info, plan, trees):
    """The trees into the plan's bits, from its own records of what they decide."""
    plan = plan.copy()
    extra, words = plan[info.extra_off:], info.tile_tokens // 32
    first = np.concatenate([[0], np.cumsum([len(t) for t in trees])]).astype(int)
    for i in range(info.num_drafts):
        row, n, cached, _, _, request, span0, spans = plan[info.drafts_off + 8 * i:info.drafts_off + 8 * i + 8]
        parents = trees[request]
        assert n == len(parents) and row == first[request]
        sight, _ = branch_cases.in_sight(int(cached), parents, info.window)
        for s in range(span0, span0 + spans):
            bits, tokens, token0, bit0, bit1, pos0, z0, z1 = plan[info.spans_off + 8 * s:info.spans_off + 8 * s + 8]
            assert 0 <= bit0 < bit1 <= info.tile_tokens and 0 <= token0 and token0 + tokens <= n and z0 == z1 == 0
            for k in range(tokens):
                seen = set(sight[token0 + k])
                for b in range(bit0, bit1):
                    word = bits + k * words + b // 32
                    value = int(extra[word]) & 0xffffffff & ~(1 << (b % 32))
                    if cached + pos0 + b - bit0 in seen:
                        value |= 1 << (b % 32)
                    extra[word] = np.uint32(value).astype(np.int32)
    return plan


def check_sight(info, plan, table, cached, trees, window):
    entries = table.reshape(-1).numpy()
    seen, writers = shown(info, plan, entries)
    row = 0
    for r, (c, parents) in enumerate(zip(cached, trees)):
        sight, _ = branch_cases.in_sight(c, parents, window)
        for i, want in enumerate(sight):
            assert sorted(seen.get(row + i, [])) == sorted(int(table[r, x]) for x in want), (r, i)
            assert writers[row + i] == 1
        row += len(parents)
    assert not [x for x in seen if x >= row]


def shown(info, plan, entries):
    """Per q row the pool rows it is shown and its writers.  (test_extend_plan.shown holds that a token with a partial row sees something
    there: a tree may take that away.)"""
    t = plan.tolist()
    words = info.tile_tokens // 32
    seen, writers = {}, {}
    for n in range(info.num_items):
        it = t[info.items_off + 32 * n:info.items_off + 32 * n + 32]
        for w in range(2):
            tok0, ntok, lo, hi, part, _, first, block_tile = it[8 + 8 * w:16 + 8 * w]
            for tok in range(ntok):
                q_row = t[info.tokens_off + 2 * (tok0 + tok)]
                got = []
                for k in range(lo, hi, it[2]):
                    rec = t[info.tiles_off + 8 * (it[5] + k):info.tiles_off + 8 * (it[5] + k + 1)]
                    place = rec[4 + block_tile]
                    for i in range(rec[2]):
                        if rec[3] < 0:
                            off = ((rec[1] << 32) | (rec[0] & 0xffffffff)) + i
                        else:
                            e = info.extra_off + rec[3] + 2 * i
                            off = (t[e + 1] << 32) | (t[e] & 0xffffffff)
                        if place < 0 or (t[info.extra_off + place + (first + tok) * words + i // 32] >> (i % 32)) & 1:
                            got.append(int(entries[off]))
                seen.setdefault(q_row, []).extend(got)
                if part >= 0:
                    assert not got or t[info.extra_off + part + tok] >= 0     # what a token sees has a place to go
                else:
                    writers[q_row] = writers.get(q_row, 0) + 1
    for i in range(info.num_merged):
        q_row = t[info.merge_off + 4 * i]
        writers[q_row] = writers.get(q_row, 0) + 1
    return seen, writers


HEADS = [(32, 8, 128, torch.float16), (16, 16, 64, torch.bfloat16), (16, 8, 256, torch.float16), (8, 2, 128, torch.float32),
         (28, 4, 32, torch.float16)]


@pytest.mark.parametrize("heads", HEADS, ids=[f"{h[0]}_{h[1]}_{h[2]}" for h in HEADS])
@pytest.mark.parametrize("seed", range(12))
def test_every_token_is_shown_its_path(heads, seed):
    rng = branch_cases.rng_of(1000 * heads[2] + seed)
    cached, nodes, shared, window = branch_cases.random_step(rng)
    trees = branch_cases.make_trees(rng, nodes)
    info, plan, table = plan_of(cached, nodes, shared, *heads, window=window, sms=rng.choice((1, 3, 148)))
    assert info.draft == 1 and info.num_drafts == len(nodes) and info.longest_draft == max(nodes, default=0)
    # before a tree is known the tokens are chains
    check_sight(info, plan, table, cached, [list(range(-1, n - 1)) for n in nodes], window)
    check_sight(info, grow(info, plan, trees), table, cached, trees, window)
    # and a second tree leaves nothing of the first
    again = branch_cases.make_trees(rng, nodes)
    check_sight(info, grow(info, grow(info, plan, trees), again), table, cached, again, window)


def test_plans_of_chains_stay_what_they_were():
    seq, ext, shared = [300, 310, 500], [9, 17, 1], [([0, 1], 200)]
    info, plan, _, _ = extend.host_plan(seq, ext, [0, 600, 1200], 32, 8, 128, torch.float16, shared_prefixes=shared)
    assert (info.draft, info.num_drafts, info.num_spans, info.longest_draft, info.drafts_off, info.spans_off) == (0, 0, 0, 0, 0, 0)
    assert info.table_ints <= len(plan)


def test_the_longest_drafts():
    n = lib.FT_MAX_DRAFT
    for parents in (list(range(-1, n - 1)), [-1] + [0] * (n - 1)):
        info, plan, table = plan_of([130], [n], [], 8, 2, 128)
        check_sight(info, grow(info, plan, [parents]), table, [130], [parents], 0)
    with pytest.raises(ValueError, match="drafted tokens"):
        plan_of([10], [n + 1], [], 8, 2, 128)


def test_refusals():
    handle = lib.load()
    i64 = lambda *x: (ctypes.c_int64 * len(x))(*x)
    out = ctypes.c_void_p()
    args = [i64(20), i64(5), i64(0), i64(0), i64(0)]
    tail = [1, 8, 2, 128, 2, 0, 148, ctypes.byref(out)]
    assert handle.ft_draft_plan_build(*args, None, *tail) == -1                                    # no numbers of the requests
    assert handle.ft_draft_plan_build(*args, (ctypes.c_int32 * 1)(1), *tail) == -1                 # a number that is none
    args[0], args[1] = i64(5000), i64(lib.FT_MAX_DRAFT + 1)
    assert handle.ft_draft_plan_build(*args, (ctypes.c_int32 * 1)(0), *tail) == -5
    for fn in ("ft_draft_tree", "ft_draft_accept", "ft_beam_select", "ft_beam_reorder"):
        assert getattr(handle, fn)(None) == -1
    plain = lib.DraftTreeArgs()
    assert handle.ft_draft_tree(ctypes.byref(plain)) == -1 and b"drafted" in handle.ft_last_error()
    plain.plan.draft, plain.plan.longest_draft = 1, lib.FT_MAX_DRAFT + 1
    assert handle.ft_draft_tree(ctypes.byref(plain)) == -1
    plain.plan.longest_draft, plain.plan.num_drafts, plain.plan.table_ints = 1, 1, 7
    assert handle.ft_draft_tree(ctypes.byref(plain)) == -1 and b"table" in handle.ft_last_error()


def test_plans_of_another_kind_are_refused():
    info, plan, _, _ = extend.host_plan([20], [5], [0], 8, 2, 128, torch.float16)
    ordinary = extend.ExtendPlan(info, torch.from_numpy(plan), [20], [5])
    for wrong in (ordinary, None, object()):
        with pytest.raises(ValueError, match="draft=True"):
            fasttree.fasttree_draft_tree(torch.zeros(5, dtype=torch.int32), wrong)
        with pytest.raises(ValueError, match="draft=True"):
            fasttree.fasttree_draft_accept(None, None, None, wrong, None, None, None)
