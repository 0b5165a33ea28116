"""ft_extend where it can go wrong beside the ordinary shapes: which kernel runs, odd head groups, values that are no numbers,
far rows of a large pool, empty calls, one plan for many layers, trees."""
import math
import subprocess
import sys

import pytest
import torch

import extend_cases
import fasttree
from ft_b200 import extend, lib
from kv_tree_simple import KVTreeNode, assign_requests
from test_extend_gpu import DTYPES, Step

pytestmark = pytest.mark.gpu


def test_kernels_by_type_head_size_and_alignment():
    def name(dtype, d, hq=8, hkv=2, path="auto", q=None, ext=(40, 3)):
        s = Step([300, 200], list(ext), [], hq, hkv, d, dtype)
        return extend.path_name(s.gq if q is None else q(s), s.gk, s.gv, torch.empty_like(s.gq), s.gt, s.plan, 1.0, path=path)

    for d in (64, 128, 256):
        assert name(torch.bfloat16, d, ext=(200, 150)).startswith("extend_tc_kernel")
        assert name(torch.float16, d, path="generic").startswith("extend_generic_kernel")
    for d in (16, 32, 64, 128, 256):
        assert name(torch.float32, d).startswith("extend_f32_kernel")
    assert name(torch.float16, 32).startswith("extend_generic_kernel")
    assert name(torch.float16, 128, hq=130, hkv=1).startswith("extend_generic_kernel")

    def off_by_one(s):
        wide = torch.empty(s.gq.numel() + 1, dtype=s.gq.dtype, device="cuda")
        return wide[1:].view(s.gq.shape)

    assert name(torch.float16, 128, q=off_by_one).startswith("extend_generic_kernel")
    assert name(torch.float32, 128, q=off_by_one).startswith("extend_generic_kernel")
    with pytest.raises(lib.FastTreeError, match="16-byte aligned"):
        name(torch.float16, 128, q=off_by_one, path="tcgen05")
    with pytest.raises(lib.FastTreeError, match="fp32"):
        name(torch.float32, 128, path="tcgen05")
    long = Step([9000], [1], [], 8, 2, 128, torch.float16)
    assert extend.path_name(long.gq, long.gk, long.gv, torch.empty_like(long.gq), long.gt, long.plan, 1.0) == "extend_tc_kernel+extend_merge_kernel"


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 64)])
@pytest.mark.parametrize("hq,hkv", [(3, 1), (10, 2), (12, 2), (24, 1), (27, 3), (97, 1)])
def test_odd_groups(dtype, d, hq, hkv):
    Step([150, 90, 140], [37, 90, 1], [([0, 2], 100)], hq, hkv, d, DTYPES[dtype]).check(cap=20.0)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 128)])
@pytest.mark.parametrize("cap", [-1.0, 25.0])
def test_scores_that_are_no_numbers_spoil_their_rows_alone(dtype, d, cap):
    """A NaN query, a NaN or infinite key in sight: the rows that meet them come out NaN (an infinite score among finite ones
    does so in a plain softmax too; capped it is a number), every other row within its bound."""
    s = Step([200, 170], [60, 30], [([0, 1], 100)], 8, 2, d, DTYPES[dtype])
    out, _, absv, size = extend_cases.oracle(s.q, s.k, s.v, s.table, s.seq, s.ext, s.scale, cap, 0)
    tol, _ = extend_cases.bounds(s.dtype, out, absv, size, cap, d)
    n = sum(s.ext)

    def run(q, k):
        o = torch.empty_like(s.gq)
        extend.extend(q, k, s.gv, o, s.gt, s.plan, s.scale, logit_cap=cap)
        torch.cuda.synchronize()
        return o[:n].cpu()

    q = s.gq.clone()
    q[7, 3, 5] = float("nan")
    o = run(q, s.gk)
    assert o[7, 3].isnan().all()
    good = torch.ones(n, 8, dtype=torch.bool)
    good[7, 3] = False
    assert bool(((o.double() - out[:n]).abs() <= tol[:n])[good].all())
    k = s.gk.clone()
    k[s.table[0, 150].long(), 1, 0] = float("nan")               # request 0's queries from position 150 on, KV head 1
    o = run(s.gq, k)
    good = torch.ones(n, 8, dtype=torch.bool)
    good[10:60, 4:] = False
    assert o[10:60, 4:].isnan().all() and bool(((o.double() - out[:n]).abs() <= tol[:n])[good].all())
    k = s.gk.clone()
    k[s.table[0, 150].long(), 1, 0] = float("inf")
    o = run(s.gq, k)
    assert bool(((o.double() - out[:n]).abs() <= tol[:n])[good].all())
    plus = s.q[10:60, 4:, 0] > 0                                  # score +inf; -inf (weight 0) where the query's element is negative
    if cap < 0:
        assert o[10:60, 4:][plus].isnan().all()
    assert torch.isfinite(o[10:60, 4:][s.q[10:60, 4:, 0] < 0]).all()


def test_large_values_and_ties():
    """Scores that differ by hundreds (one key takes all the weight) and scores that are all alike."""
    for d, dtype in ((64, torch.bfloat16), (128, torch.float16), (256, torch.bfloat16), (128, torch.float32)):
        Step([300, 180], [100, 2], [], 8, 2, d, dtype, q_scale=30.0).check()
        s = Step([300, 180], [100, 2], [], 8, 2, d, dtype)
        s.q.zero_(), s.gq.zero_()
        s.check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_far_rows_of_a_large_pool(dtype):
    rows, hkv, d = 70000 if dtype == torch.float16 else 40000, 128 if dtype == torch.float16 else 256, 256      # offsets beyond 31 bits
    pool = torch.zeros(rows, hkv, d, dtype=dtype, device="cuda")
    g = torch.Generator().manual_seed(1)
    n = 130
    for slots in (torch.arange(rows - n, rows), torch.randperm(rows, generator=g)[:n]):
        pool[slots.cuda()] = torch.randn(n, hkv, d, generator=g).to(dtype).cuda()
        q = torch.randn(3, hkv, d, generator=g).to(dtype)
        plan = fasttree.fasttree_extend_preparation([n], [3], [0], hkv, hkv, d, dtype)
        heads = [0, hkv - 1]
        k = pool[slots.cuda()][:, heads].cpu()
        out, _, absv, size = extend_cases.oracle(q[:, heads], k, k, torch.arange(n)[None], [n], [3], 0.06, -1.0, 0)
        tol, _ = extend_cases.bounds(dtype, out, absv, size, -1.0, d)
        for path in ("auto", "generic"):
            o = torch.empty(3, hkv, d, dtype=dtype, device="cuda")
            extend.extend(q.cuda(), pool, pool, o, slots.int().cuda(), plan, 0.06, path=path)
            assert bool(((o[:, heads].double().cpu() - out).abs() <= tol).all())
    assert lib.read_device_status() == 0


def test_heads_outermost_pools_with_far_heads():
    rows, hkv, d = 70000, 128, 256
    kv = torch.zeros(hkv, rows, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(2)
    slots = torch.randperm(rows, generator=g)[:90]
    kv[:, slots.cuda()] = torch.randn(hkv, 90, d, generator=g).bfloat16().cuda()
    q = torch.randn(2, hkv, d, generator=g).bfloat16()
    plan = fasttree.fasttree_extend_preparation([90], [2], [0], hkv, hkv, d, torch.bfloat16)
    heads = [0, hkv - 1]
    k = kv[heads][:, slots.cuda()].transpose(0, 1).cpu()
    out, _, absv, size = extend_cases.oracle(q[:, heads], k, k, torch.arange(90)[None], [90], [2], 0.06, -1.0, 0)
    tol, _ = extend_cases.bounds(torch.bfloat16, out, absv, size, -1.0, d)
    o = torch.empty(2, hkv, d, dtype=torch.bfloat16, device="cuda")
    fasttree.fasttree_extend(q.cuda(), kv.transpose(0, 1), kv.transpose(0, 1), o, slots.int().cuda(), plan, 0.06)
    assert bool(((o[:, heads].double().cpu() - out).abs() <= tol).all()) and lib.read_device_status() == 0


def test_calls_without_tokens():
    s = Step([30, 20], [0, 0], [], 8, 2, 128, torch.float16, pad_rows=3)
    o = torch.full_like(s.gq, 7.0)
    launches = lib.launch_count()
    fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, 1.0)
    fasttree.fasttree_extend(s.gq[:0], s.gk, s.gv, o[:0], s.gt, s.plan, 1.0)
    assert lib.launch_count() == launches and (o == 7).all()


def test_output_in_the_queries_place_is_refused():
    s = Step([30, 20], [4, 3], [], 8, 2, 64, torch.float16)
    with pytest.raises(ValueError, match="must not be q"):
        fasttree.fasttree_extend(s.gq, s.gk, s.gv, s.gq, s.gt, s.plan, 1.0)


def test_one_plan_for_many_layers_and_inputs():
    s = Step([700, 650, 900], [30, 1, 200], [([0, 1, 2], 600)], 8, 2, 128, torch.bfloat16)
    for seed in range(3):
        g = torch.Generator().manual_seed(100 + seed)
        s.k, s.v = torch.randn(s.k.shape, generator=g).bfloat16(), torch.randn(s.v.shape, generator=g).bfloat16()
        s.q = torch.randn(s.q.shape, generator=g).bfloat16()
        s.gq, s.gk, s.gv = s.q.cuda(), s.k.cuda(), s.v.cuda()
        s.check()


def test_prefixes_of_a_tree():
    """A radix tree of cached prefixes in the tree model of the decode entry points, a question on every leaf."""
    nodes = [KVTreeNode(-1, 0, 300, 2), KVTreeNode(0, 1, 140, 3), KVTreeNode(0, 2, 77, 2)] + [KVTreeNode(1, i, 9 + i, 0) for i in (3, 4, 5)] + [
        KVTreeNode(2, i, 5 * i, 0) for i in (6, 7)]
    batch, ptrs = assign_requests(nodes)
    new = [11, 1, 40, 7, 90]
    path = [[] for _ in range(batch)]
    for nd in nodes:                                             # parents come first
        for r in nd.requests:
            path[r] += list(range(ptrs[nd.id], ptrs[nd.id + 1]))
    at, rows = ptrs[-1], []
    for r in range(batch):
        rows.append(path[r] + list(range(at, at + new[r])))
        at += new[r]
    seq = [len(x) for x in rows]
    table = torch.zeros(batch, max(seq) + 2, dtype=torch.int32)
    for r, x in enumerate(rows):
        table[r, :len(x)] = torch.tensor(x, dtype=torch.int32)
    g = torch.Generator().manual_seed(4)
    hq, hkv, d = 8, 2, 128
    k, v, q = torch.randn(at, hkv, d, generator=g).half(), torch.randn(at, hkv, d, generator=g).half(), torch.randn(sum(new), hq, d, generator=g).half()
    plan = fasttree.fasttree_extend_preparation(seq, new, [r * table.shape[1] for r in range(batch)], hq, hkv, d, torch.float16,
                                                shared_prefixes=extend.tree_prefixes(nodes))
    o = torch.empty_like(q.cuda())
    fasttree.fasttree_extend(q.cuda(), k.cuda(), v.cuda(), o, table.cuda(), plan, d ** -0.5)
    out, _, absv, size = extend_cases.oracle(q, k, v, table, seq, new, d ** -0.5, -1.0, 0)
    tol, _ = extend_cases.bounds(torch.float16, out, absv, size, -1.0, d)
    assert bool(((o.double().cpu() - out).abs() <= tol).all())


def test_beside_decode_steps_on_one_stream():
    """Decode steps and extend calls in turn on one stream: launches that may start early wait for one another."""
    import cases
    import gpu_utils
    c = cases.build_decode_case("rand3_fp16")
    run = gpu_utils.EngineRun(c["nodes"], c["ptrs"], c["batch"], c["q"], c["k"], c["v"], c["hq"], c["hkv"], c["d"], c["tsq"])
    want = run.decode(poison=False, with_lse=False)
    s = Step([3000, 200], [1, 60], [], 8, 2, 128, torch.bfloat16)
    first, _ = s.run()
    n = sum(s.ext)
    outs = [torch.zeros_like(s.gq) for _ in range(6)]
    decoded = []
    for o in outs:
        fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
        run.o = torch.zeros_like(run.q)
        fasttree.fasttree_decode(run.q, run.k, run.v, run.o, *run.aux, run.tiles[0], run.tiles[1], run.scale)
        decoded.append(run.o)
    torch.cuda.synchronize()
    assert all(torch.equal(o[:n], first[:n]) for o in outs)
    assert all(torch.equal(x.float().cpu(), want) for x in decoded) and math.isfinite(want.sum().item())


FIRST_CALLS = """
import sys
sys.path[:0] = {path!r}
import torch
import fasttree
from test_extend_gpu import Step
steps = [Step([5000, 90], [1, 9], [], 8, 2, d, t) for d, t in
         ((64, torch.float16), (128, torch.bfloat16), (256, torch.float16), (32, torch.float16), (128, torch.float32))]
outs, pools = [torch.zeros_like(s.gq) for s in steps], [(torch.zeros_like(s.gk), torch.zeros_like(s.gv)) for s in steps]
slots = torch.arange(4, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    for s, o, (k, v) in zip(steps, outs, pools):
        fasttree.fasttree_append(None, s.gk[:4], s.gv[:4], k, v, slots)
        fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
graph.replay()
torch.cuda.synchronize()
for s, o, (k, v) in zip(steps, outs, pools):
    want, _ = s.run()
    n = sum(s.ext)
    assert torch.equal(o[:n], want[:n]) and not (o[n:] != 0).any()
    assert torch.equal(k[:4], s.gk[:4]) and torch.equal(v[:4], s.gv[:4]) and not (k[4:] != 0).any()
print("first calls captured")
"""


def test_first_calls_of_a_process_in_a_captured_graph():
    """Nothing that a kernel's first call sets up (its code, its shared memory limit, its descriptors) needs the stream."""
    path = [p for p in sys.path if p]
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(path=path)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "first calls captured" in r.stdout, r.stderr[-2000:]
