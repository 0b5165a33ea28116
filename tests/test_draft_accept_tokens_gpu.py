"""What acceptance makes of tokens, targets and rows that are none."""
import pytest
import torch

import fasttree
from ft_b200 import lib

gpu = pytest.mark.gpu


def accept(tokens, targets, parents, out=torch.int64, slots=None):
    n = len(tokens)
    plan = fasttree.fasttree_extend_preparation([n + 4], [n], [0], 8, 2, 64, torch.float16, draft=True)
    accepted = torch.full((1, n), -9, dtype=torch.int32, device="cuda")
    counts, following = torch.full((1,), -9, dtype=torch.int32, device="cuda"), torch.full((1,), -9, dtype=out, device="cuda")
    table = torch.full((n + 4,), -5, dtype=torch.int32, device="cuda")
    tokens, targets, parents = (torch.tensor(x, dtype=torch.int64, device="cuda") for x in (tokens, targets, parents))
    rows = {} if slots is None else {"slots": torch.tensor(slots, device="cuda"), "kv_entries": table}
    fasttree.fasttree_draft_accept(None, tokens, parents, plan, accepted, counts, following, targets=targets, **rows)
    torch.cuda.synchronize()
    return accepted[0, :int(counts)].tolist(), int(following), table.tolist()


@gpu
@pytest.mark.parametrize("token", [-1, -5, -100, 1 << 31, 1 << 40, -(1 << 40)])
@pytest.mark.parametrize("target", [-1, -5, 1 << 31, 1 << 40])
def test_a_target_that_is_no_token_accepts_nothing(token, target):
    path, following, _ = accept([3, token, 8], [target, 8, 9], [-1, 0, 1])
    assert path == [0] and following == target


@gpu
def test_a_drafted_token_that_is_none_is_passed_over():
    path, following, _ = accept([3, -1, 1 << 33, 7, 9], [7, 5, 5, 9, 4], [-1, 0, 0, 0, 3])
    assert path == [0, 3, 4] and following == 4


@gpu
def test_a_next_token_that_int32_does_not_hold():
    assert accept([3, 4], [4, (1 << 33) + 5], [-1, 0], out=torch.int32)[:2] == ([0, 1], -1)
    assert accept([3, 4], [-(1 << 40), 5], [-1, 0], out=torch.int32)[:2] == ([0], -1)
    assert accept([3, 4], [-7, 5], [-1, 0], out=torch.int32)[:2] == ([0], -7)
    assert accept([3, 4], [(1 << 31) - 1, 5], [-1, 0], out=torch.int32)[:2] == ([0], (1 << 31) - 1)


@gpu
def test_rows_that_int32_does_not_hold():
    lib.read_device_status()
    path, _, table = accept([3, 4, 5], [5, 0, 9], [-1, 0, 0], slots=[11, 12, 13])
    assert path == [0, 2] and table[4:] == [11, 13, 12] and lib.read_device_status() == 0
    path, _, table = accept([3, 4, 5], [5, 0, 9], [-1, 0, 0], slots=[(1 << 32) + 11, -1, 13])
    assert path == [0, 2] and table[4:] == [-1, 13, -1] and lib.read_device_status() == lib.FT_DEV_BAD_KV_INDEX
    path, _, table = accept([3, 4, 5], [5, 0, 9], [-1, 0, 0], slots=[11, 12, -(1 << 40)])
    assert path == [0, 2] and table[4:] == [11, -1, 12] and lib.read_device_status() == lib.FT_DEV_BAD_KV_INDEX
