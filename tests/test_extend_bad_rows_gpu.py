"""Row ids outside the pool: flagged, and left out of the attention of every query that would see them, on every path."""
import math

import pytest
import torch

import extend_cases
from ft_b200 import extend, lib
from test_extend_gpu import DTYPES, Step

pytestmark = pytest.mark.gpu


def expected(s, table, cap):
    """The oracle over the row ids that are in the pool; a query without any has output 0 and LSE -inf."""
    g = s.q.shape[1] // s.k.shape[1]
    q, k, v = s.q.double(), s.k.double().repeat_interleave(g, 1), s.v.double().repeat_interleave(g, 1)
    out, absv, size = (torch.zeros(s.q.shape, dtype=torch.float64) for _ in range(3))
    size, lse = torch.zeros(s.q.shape[:2], dtype=torch.float64), torch.full(s.q.shape[:2], -math.inf, dtype=torch.float64)
    at = 0
    for r, (n, e) in enumerate(zip(s.seq, s.ext)):
        rows = table[r, :n].long()
        good = (rows >= 0) & (rows < s.k.shape[0])
        kk, vv = k[rows.clamp(0, s.k.shape[0] - 1)].transpose(0, 1), v[rows.clamp(0, s.k.shape[0] - 1)].transpose(0, 1)
        z = q[at:at + e].transpose(0, 1) @ kk.transpose(1, 2) * s.scale                        # [heads, queries, keys]
        z_abs = q[at:at + e].abs().transpose(0, 1) @ kk.abs().transpose(1, 2) * abs(s.scale)
        age = torch.arange(n - e, n)[:, None] - torch.arange(n)
        seen = (age >= 0) & (age < (s.window or n)) & good
        if cap > 0:
            z = cap * torch.tanh(z / cap)
        z = z.masked_fill(~seen, -math.inf)
        lse[at:at + e] = torch.logsumexp(z, -1).T
        w = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)).masked_fill(~seen, 0.0)
        out[at:at + e], absv[at:at + e] = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
        size[at:at + e] = z_abs.masked_fill(~seen, 0.0).amax(-1).T
        at += e
    return out, lse, absv, size


def check(s, hits, cap=-1.0, path="auto", plan=None):
    """`hits`: (request, position, row id) triples."""
    table = s.table.clone()
    for r, pos, value in hits:
        table[r, pos] = value
    o, lse = torch.full_like(s.gq, float("nan")), torch.full(s.q.shape[:2], float("nan"), device="cuda")
    extend.extend(s.gq, s.gk, s.gv, o, table.cuda(), plan or s.plan, s.scale, logit_cap=cap, o_lse=lse, path=path)
    torch.cuda.synchronize()
    assert lib.read_device_status() == lib.FT_DEV_BAD_KV_INDEX
    n = sum(s.ext)
    out, want, absv, size = expected(s, table, cap)
    tol, tol_lse = extend_cases.bounds(s.dtype, out, absv, size, cap, s.d)
    none = want[:n] == -math.inf
    assert bool(((o[:n].double().cpu() - out[:n]).abs() <= tol[:n]).all())
    assert torch.equal((lse[:n] == -math.inf).cpu(), none) and not o[:n].cpu()[none].any()
    assert bool(((lse[:n].double().cpu() - want[:n]).abs()[~none] <= tol_lse[:n][~none]).all())


FORMS = [("fp16", 64), ("bf16", 128), ("fp16", 256), ("fp32", 128)]


@pytest.mark.parametrize("path", ["auto", "generic"])
@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("cap", [-1.0, 20.0])
def test_rows_outside_the_pool_are_left_out(dtype, d, cap, path):
    s = Step([900, 200, 333], [40, 3, 200], [([0, 2], 130)], 8, 2, d, DTYPES[dtype], q_scale=2.0)
    rows = s.k.shape[0]
    check(s, [(0, 50, rows), (2, 50, rows), (1, 199, -5)], cap, path)             # of a prefix that is shared, and a request's last
    check(s, [(0, 300, -1)], cap, path)                                           # a tile that all see whole
    check(s, [(0, 899, 2 ** 31 - 1), (2, 133, -2 ** 31)], cap, path)
    check(s, [(0, i, rows + i) for i in range(256, 384)] + [(0, 700, -1), (0, 870, -1)], cap, path)    # a whole tile
    check(s, [(0, i, -1) for i in range(130)] + [(2, i, -1) for i in range(330)], cap, path)            # nearly all, from the first on


@pytest.mark.parametrize("dtype,d", FORMS)
def test_queries_that_are_left_with_nothing(dtype, d):
    s = Step([1, 5, 40], [1, 5, 1], [], 8, 2, d, DTYPES[dtype])
    check(s, [(0, 0, -1), (1, 0, -3)])
    check(s, [(2, i, s.k.shape[0]) for i in range(40)])
    s = Step([3000, 2900], [1, 1], [([0, 1], 2500)], 8, 2, d, DTYPES[dtype])      # in partial rows
    check(s, [(r, i, -1) for r in range(2) for i in range(2900)])
    check(s, [(1, i, -1) for i in range(2500, 2900)])


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("window", [0, 150])
def test_over_many_tasks_of_a_block(dtype, d, window):
    """Good and bad tiles in turn in the queue of one CTA: what is noted of a tile is that tile's."""
    seq = [500 + 31 * (i % 5) for i in range(12)]
    s = Step(seq, [60, 1, 200, 33] * 3, [([0, 1, 2], 350), (list(range(4, 9)), 300)], 8, 2, d, DTYPES[dtype], window=window)
    info, table, _, _ = extend.host_plan(seq, s.ext, [r * s.table.shape[1] for r in range(12)], 8, 2, d, s.dtype,
                                         shared_prefixes=s.shared, window=window, num_sms=3)
    plan = extend.ExtendPlan(info, torch.from_numpy(table).cuda(), seq, s.ext)
    hits = [(r, p, -1) for r in (4, 5, 6, 7, 8) for p in (7, 299)] + [(9, 480, s.k.shape[0]), (11, 400, -1), (2, 560, -9), (0, 499, -1)]
    check(s, hits, plan=plan)
    check(s, hits, plan=plan, cap=5.0)


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_scores_far_from_zero(dtype, d, sign):
    """A key of zeros would outweigh all others, or none: every score lies far below or above 0."""
    s = Step([900, 200], [40, 3], [], 8, 2, d, DTYPES[dtype])
    s.q = (s.q.abs() + 0.5).to(s.dtype)
    s.k = (sign * (s.k.abs() + 0.5)).to(s.dtype)
    s.gq, s.gk = s.q.cuda(), s.k.cuda()
    check(s, [(0, 50, -1), (0, 300, -1), (0, 860, -1), (1, 7, s.k.shape[0])])


@pytest.mark.parametrize("dtype,d", FORMS)
def test_rows_that_see_none_keep_their_bits(dtype, d):
    s = Step([700, 300, 260], [200, 40, 1], [([0, 1], 250)], 8, 2, d, DTYPES[dtype])
    want, want_lse = s.run()
    table = s.gt.clone()
    table[0, 600] = -1                                           # seen by request 0's queries from the hundredth on
    o, lse = torch.empty_like(s.gq), torch.empty_like(want_lse)
    extend.extend(s.gq, s.gk, s.gv, o, table, s.plan, s.scale, o_lse=lse)
    assert lib.read_device_status() == lib.FT_DEV_BAD_KV_INDEX
    rows = list(range(100)) + list(range(200, 241))
    assert torch.equal(o[rows], want[rows]) and torch.equal(lse[rows], want_lse[rows])
