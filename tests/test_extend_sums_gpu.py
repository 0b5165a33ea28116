"""fp32 scores of few query rows: how far the sum of head_dim products may be off."""
import pytest
import torch

from ft_b200 import extend
from test_extend_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("m", [1, 5, 16, 32, 64, 100, 333])
def test_products_that_round_the_same_way(d, m):
    """One key of equal elements just above 1: a chain of sums loses the same part of each.  In blocks of 32 products no sum has more
    than 32 + d / 32 roundings on its way, each of half a step of at most the score, and the LSE of one key is the score."""
    s = Step([1, 1, 1], [1, 1, 1], [], 4, 1, d, torch.float32)
    assert s.plan.info.rows_per_tile == 16
    s.q.fill_(1.0), s.gq.fill_(1.0)
    s.k.fill_(1 + m * 2.0 ** -23), s.gk.fill_(1 + m * 2.0 ** -23)
    lse = torch.zeros(s.q.shape[:2], device="cuda")
    o = torch.empty_like(s.gq)
    extend.extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, 1.0, o_lse=lse)
    want = d * (1 + m * 2.0 ** -23)
    err = (lse[:3].double().cpu() - want).abs().max().item()
    assert err <= (32 + d / 32) * 2.0 ** -24 * want, err / want * 2 ** 24
    assert torch.equal(o[:3, 0].cpu(), s.v[s.table[:, 0].long(), 0])
