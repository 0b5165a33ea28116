"""ft_extend against the 64-bit oracle: types, head layouts, lengths from one token on, shared prefixes, windows, caps."""
import ctypes

import pytest
import torch

import extend_cases
import fasttree
from ft_b200 import extend, lib

gpu = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


class Step:
    """One planned step on the GPU with host copies for the oracle."""

    def __init__(self, seq, ext, shared, hq, hkv, d, dtype, window=0, layout="scattered", seed=0, q_scale=1.0, pad_rows=2):
        self.seq, self.ext, self.shared, self.dtype, self.window, self.d = seq, ext, shared, dtype, window, d
        g = torch.Generator().manual_seed(seed)
        self.table, rows = extend_cases.pool(seq, ext, shared, layout=layout, seed=seed)
        self.k, self.v = torch.randn(rows, hkv, d, generator=g).to(dtype), torch.randn(rows, hkv, d, generator=g).to(dtype)
        self.q = (torch.randn(sum(ext) + pad_rows, hq, d, generator=g) * q_scale).to(dtype)
        self.scale = d ** -0.5
        self.plan = fasttree.fasttree_extend_preparation(seq, ext, [r * self.table.shape[1] for r in range(len(seq))], hq, hkv, d,
                                                         dtype, shared_prefixes=shared, window=window)
        self.gq, self.gk, self.gv, self.gt = self.q.cuda(), self.k.cuda(), self.v.cuda(), self.table.cuda()

    def run(self, path="auto", cap=-1.0, scale=None):
        o = torch.full_like(self.gq, float("nan"))
        lse = torch.full(self.q.shape[:2], float("nan"), device="cuda")
        extend.extend(self.gq, self.gk, self.gv, o, self.gt, self.plan, self.scale if scale is None else scale, logit_cap=cap,
                      o_lse=lse, path=path)
        torch.cuda.synchronize()
        assert lib.read_device_status() == 0
        return o, lse

    def check(self, path="auto", cap=-1.0, scale=None):
        o, lse = self.run(path, cap, scale)
        out, want_lse, absv, size = extend_cases.oracle(self.q, self.k, self.v, self.table, self.seq, self.ext,
                                                        self.scale if scale is None else scale, cap, self.window)
        n = sum(self.ext)
        assert o[n:].isnan().all() and lse[n:].isnan().all()     # rows behind the last query stay as they were
        tol, tol_lse = extend_cases.bounds(self.dtype, out, absv, size, cap, self.d)
        err = (o[:n].double().cpu() - out[:n]).abs()
        assert bool((err <= tol[:n]).all()), (err / tol[:n]).max().item()
        err = (lse[:n].double().cpu() - want_lse[:n]).abs()
        assert bool((err <= tol_lse[:n]).all()), (err / tol_lse[:n]).max().item()
        return o, lse


SHAPES = {
    "one_token": ([1], [1], []),
    "tile_borders": ([127, 128, 129, 130], [127, 128, 1, 130], []),
    "ragged": ([5, 301, 77, 260], [5, 40, 1, 33], []),
    "some_without": ([40, 50, 60, 70], [0, 3, 0, 9], []),
    "shared": ([210, 230, 200, 333, 290], [10, 30, 1, 100, 2], [([0, 1, 2, 3, 4], 199)]),
    "tree": ([300, 310, 500, 520, 90], [9, 17, 1, 33, 90], [([0, 1], 200), ([2, 3], 470), ([0, 1, 2, 3], 128)]),
}


@gpu
@pytest.mark.parametrize("dtype,d", [("fp32", 16), ("fp16", 32), ("fp16", 64), ("bf16", 64), ("fp16", 128), ("bf16", 128), ("fp32", 128),
                                     ("fp16", 256), ("bf16", 256), ("fp32", 256)])
@pytest.mark.parametrize("shape", sorted(SHAPES))
def test_against_the_oracle(shape, dtype, d):
    seq, ext, shared = SHAPES[shape]
    for hq, hkv in ((8, 2), (7, 1)):
        Step(seq, ext, shared, hq, hkv, d, DTYPES[dtype], seed=d + len(shape)).check()


@gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 64)])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (16, 1), (40, 2), (128, 1), (130, 1)])
def test_head_layouts(dtype, d, hq, hkv):
    Step([60, 200], [20, 3], [([0, 1], 40)], hq, hkv, d, DTYPES[dtype]).check()


@gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 128)])
@pytest.mark.parametrize("window", [1, 5, 128, 200])
def test_windows(dtype, d, window):
    Step([400, 90, 290], [60, 90, 1], [([0, 2], 250)], 8, 2, d, DTYPES[dtype], window=window).check()


@gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 128)])
@pytest.mark.parametrize("cap", [0.5, 30.0])
def test_capped_scores(dtype, d, cap):
    Step([400, 90, 290], [60, 90, 1], [([0, 2], 250)], 8, 2, d, DTYPES[dtype], q_scale=4.0).check(cap=cap)
    Step([400, 90, 290], [60, 90, 1], [], 8, 2, d, DTYPES[dtype], window=130, q_scale=4.0).check(cap=cap)


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0])
def test_scales(d, scale):
    Step([200, 90], [30, 90], [], 8, 2, d, torch.bfloat16).check(scale=scale)


@gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("layout", ["prefill", "scattered"])
def test_long_contexts_cut_into_items(d, layout):
    s = Step([3000, 2900], [1, 1], [([0, 1], 2500)], 8, 2, d, torch.float16, layout=layout)
    assert s.plan.partial_rows > 0
    s.check()
    Step([2500], [150], [], 4, 1, d, torch.bfloat16, layout=layout).check()
    Step([1500] * 9, [1] * 9, [(list(range(9)), 700)], 8, 2, d, torch.bfloat16, layout=layout, window=1200).check(cap=20.0)


@gpu
def test_many_single_tokens_with_tails_of_their_own():
    seq = [400 + 13 * (i % 7) for i in range(40)]
    Step(seq, [1] * 40, [(list(range(40)), 390)], 8, 2, 128, torch.float16, layout="prefill").check()
    Step(seq, [1] * 40, [(list(range(40)), 390)], 8, 1, 64, torch.bfloat16).check()


@gpu
@pytest.mark.parametrize("dtype,d", [("fp16", 64), ("bf16", 128), ("bf16", 256), ("fp32", 128)])
def test_paths_agree_and_repeat(dtype, d):
    s = Step([300, 310, 500, 520, 90], [9, 17, 1, 33, 90], [([0, 1], 200), ([2, 3], 470)], 8, 2, d, DTYPES[dtype])
    a, _ = s.check("generic")
    b, _ = s.check("auto")
    c, _ = s.run("auto")
    n = sum(s.ext)
    assert torch.equal(b[:n], c[:n])                             # same order of every sum


@gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("bf16", 256), ("fp32", 64)])
def test_infinities_and_nan_out_of_sight(dtype, d):
    """Rows of K and V that a query does not see may hold anything: later positions, other requests' rows, positions behind
    the window, unused pool rows."""
    s = Step([140, 150, 130], [40, 50, 5], [([0, 1, 2], 90)], 8, 2, d, DTYPES[dtype], window=100)
    n = sum(s.ext)
    want, _ = s.run()
    for value in (float("inf"), float("nan"), -float("inf")):
        k, v = s.gk.clone(), s.gv.clone()
        hit = s.table[1, 120].long()                             # seen by request 1's queries from position 120 on
        k[hit], v[hit] = value, value
        first = s.table[0, 3].long()                             # behind the window of every query from position 103 on
        k[first], v[first] = value, value
        unused = torch.ones(k.shape[0], dtype=torch.bool)
        for r, length in enumerate(s.seq):
            unused[s.table[r, :length].long()] = False
        k[unused.cuda()], v[unused.cuda()] = value, value
        o = torch.empty_like(s.gq)
        extend.extend(s.gq, k, v, o, s.gt, s.plan, s.scale)
        torch.cuda.synchronize()
        spoiled = torch.zeros(n, dtype=torch.bool)
        row = 0
        for r, (length, e) in enumerate(zip(s.seq, s.ext)):
            for i in range(e):
                pos = length - e + i
                spoiled[row] = (r == 1 and pos >= 120) or pos < 103
                row += 1
        good = ~spoiled
        assert good.sum() > 20 and torch.isfinite(o[:n][good.cuda()]).all()
        u = 2.0 ** -24 if s.dtype == torch.float32 else torch.finfo(s.dtype).eps / 2
        # the same tokens in another arithmetic: each within the oracle's bound of the true value
        out, _, absv, size = extend_cases.oracle(s.q, s.k, s.v, s.table, s.seq, s.ext, s.scale, -1.0, s.window)
        tol, _ = extend_cases.bounds(s.dtype, out, absv, size, -1.0, s.d)
        assert bool(((o[:n].double().cpu() - out[:n]).abs() <= tol[:n])[good].all()) and u > 0
        assert not torch.isfinite(o[:n][spoiled.cuda()]).all(-1).any()


@gpu
def test_strides_and_odd_alignment():
    s = Step([150, 60], [40, 60], [], 8, 2, 64, torch.float16)
    want, _ = s.run()
    n = sum(s.ext)
    out, _, absv, size = extend_cases.oracle(s.q, s.k, s.v, s.table, s.seq, s.ext, s.scale, -1.0, 0)
    tol, _ = extend_cases.bounds(s.dtype, out, absv, size, -1.0, s.d)

    def near(o):
        return bool(((o[:n].double().cpu() - out[:n]).abs() <= tol[:n]).all())

    wide = torch.zeros(s.q.shape[0], 8 * 64 + 24, dtype=torch.float16, device="cuda")
    for pad in (8, 3):                                           # 16-byte aligned rows, and rows that are not
        q = wide[:, pad:pad + 512].unflatten(1, (8, 64))
        q.copy_(s.gq)
        kv = torch.zeros(s.k.shape[0], 2, 2, 72, dtype=torch.float16, device="cuda")   # K and V interleaved, padded heads
        k, v = kv[:, 0, :, pad - 3 if pad == 3 else 0:][..., :64], kv[:, 1, :, :64]
        k.copy_(s.gk), v.copy_(s.gv)
        o = torch.zeros(s.q.shape[0], 8, 80, dtype=torch.float16, device="cuda")[..., pad:pad + 64]
        extend.extend(q, k, v, o, s.gt.reshape(-1), s.plan, s.scale)
        assert near(o)
    heads_first = s.gk.transpose(0, 1).contiguous().transpose(0, 1), s.gv.transpose(0, 1).contiguous().transpose(0, 1)
    o = torch.empty_like(s.gq)
    extend.extend(s.gq, *heads_first, o, s.gt, s.plan, s.scale)
    assert near(o)
    assert lib.read_device_status() == 0


@gpu
def test_captured_replayed_and_two_streams_at_once():
    s = Step([5000, 4000, 4800], [1, 7, 60], [([0, 1, 2], 3900)], 8, 2, 128, torch.bfloat16)
    n = sum(s.ext)
    want, _ = s.run()
    graphs, outs = [], []
    for _ in range(2):
        o = torch.zeros_like(s.gq)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
        graphs.append(g), outs.append(o)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[:n], want[:n]) and (o[n:] == 0).all()
    outs = [torch.zeros_like(s.gq) for _ in streams]
    for _ in range(5):
        for o, st in zip(outs, streams):
            with torch.cuda.stream(st):
                fasttree.fasttree_extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, s.scale)
    torch.cuda.synchronize()
    assert all(torch.equal(o[:n], want[:n]) for o in outs)


@gpu
def test_bad_pool_rows_are_flagged():
    for d in (64, 256):
        s = Step([300, 200], [40, 3], [], 8, 2, d, torch.float16)
        table = s.gt.clone()
        table[0, 50], table[1, 199] = s.k.shape[0], -5
        o = torch.zeros_like(s.gq)
        extend.extend(s.gq, s.gk, s.gv, o, table, s.plan, s.scale)
        assert lib.read_device_status() == lib.FT_DEV_BAD_KV_INDEX


@gpu
def test_append_then_extend_step_by_step_is_one_prefill():
    """A prompt taken in chunks and then token by token, keys turned on the way into the cache, as a serving loop does it:
    every chunk's outputs are those of the whole prompt at once."""
    hq, hkv, d, dtype, n = 8, 2, 128, torch.bfloat16, 300
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, h, d, generator=g).to(dtype).cuda() for h in (hq, hkv, hkv))
    angle = torch.outer(torch.arange(n, dtype=torch.float64), torch.exp(-torch.arange(d // 2, dtype=torch.float64) / 7))
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
    slots = torch.randperm(n + 20, generator=g)[:n].int().cuda()
    kb, vb = torch.zeros(n + 20, hkv, d, dtype=dtype, device="cuda"), torch.zeros(n + 20, hkv, d, dtype=dtype, device="cuda")
    pos = torch.arange(n, device="cuda")
    whole_q, whole = torch.empty_like(q), torch.empty_like(q)
    fasttree.fasttree_append(q, k, v, kb, vb, slots, q_out=whole_q, positions=pos, cos_sin=cos_sin)
    plan = fasttree.fasttree_extend_preparation([n], [n], [0], hq, hkv, d, dtype)
    fasttree.fasttree_extend(whole_q, kb, vb, whole, slots, plan, d ** -0.5)
    ref, _, absv, size = extend_cases.oracle(whole_q.cpu(), kb.cpu(), vb.cpu(), slots.cpu()[None], [n], [n], d ** -0.5, -1.0, 0)
    tol, _ = extend_cases.bounds(dtype, ref, absv, size, -1.0, d)
    assert bool(((whole.double().cpu() - ref).abs() <= tol).all())
    kb2, vb2 = torch.zeros_like(kb), torch.zeros_like(vb)
    at = 0
    for m in [130, 1, 1, 60, 100, 1, 7]:
        part = slice(at, at + m)
        at += m
        qq, o = q[part].clone(), torch.empty_like(q[part])
        fasttree.fasttree_append(qq, k[part], v[part], kb2, vb2, slots[part], positions=pos[part], cos_sin=cos_sin)
        assert torch.equal(qq, whole_q[part])
        plan = fasttree.fasttree_extend_preparation([at], [m], [0], hq, hkv, d, dtype)
        fasttree.fasttree_extend(qq, kb2, vb2, o, slots, plan, d ** -0.5)
        assert bool(((o.double().cpu() - ref[part]).abs() <= tol[part]).all())
    assert at == n and torch.equal(kb, kb2) and torch.equal(vb, vb2)


def test_refusals_on_the_host():
    handle = lib.load()
    assert handle.ft_extend(None) == -1
    a = lib.ExtendArgs()
    a.dtype, a.num_qo_heads, a.num_kv_heads, a.head_dim = lib.FT_F16, 8, 2, 128
    assert handle.ft_extend(ctypes.byref(a)) == -1 and b"plan was made for" in handle.ft_last_error()
    info, _, _, _ = extend.host_plan([300], [300], [0], 8, 2, 128, torch.float16)
    a.plan = info
    assert handle.ft_extend(ctypes.byref(a)) == -1 and b"NULL" in handle.ft_last_error()
    a.q = a.k_buffer = a.v_buffer = a.o = a.kv_entries = a.plan_table = 4096
    a.kv_rows, a.q_rows, a.kv_entries_len = 10, 299, 300
    assert handle.ft_extend(ctypes.byref(a)) == -1 and b"rows of q" in handle.ft_last_error()
    a.q_rows, a.kv_entries_len = 300, 299
    assert handle.ft_extend(ctypes.byref(a)) == -1 and b"kv_entries" in handle.ft_last_error()
    a.kv_entries_len, a.path = 300, 9
    assert handle.ft_extend(ctypes.byref(a)) == -1
    a.path, a.dtype = 0, lib.FT_F32
    assert handle.ft_extend(ctypes.byref(a)) == -1               # planned for 16-bit elements
    q = torch.zeros(300, 8, 128, dtype=torch.float16)
    with pytest.raises(ValueError):
        fasttree.fasttree_extend(q, q, q, q, q, None, 1.0)
    plan = extend.ExtendPlan(info, torch.zeros(4, dtype=torch.int32), [300], [300])
    with pytest.raises(ValueError, match="no CPU path"):
        fasttree.fasttree_extend(q, q, q, q, torch.zeros(3, dtype=torch.int32), plan, 1.0)


@gpu
def test_refusals_of_tensors():
    s = Step([30, 20], [4, 3], [], 8, 2, 64, torch.float16, pad_rows=0)
    o = torch.empty_like(s.gq)
    ok = dict(q=s.gq, k_buffer=s.gk, v_buffer=s.gv, o=o, kv_entries=s.gt, plan=s.plan, sm_scale=1.0)
    fasttree.fasttree_extend(**ok)
    for bad in (dict(q=s.gq.float()), dict(o=o[:3]), dict(k_buffer=s.gk[..., :32]), dict(v_buffer=s.gv[:9]), dict(kv_entries=s.gt.long()),
                dict(kv_entries=s.gt.cpu()), dict(o_lse=torch.zeros(7, 8, device="cuda").double()), dict(o_lse=torch.zeros(6, 8, device="cuda"))):
        with pytest.raises(ValueError):
            fasttree.fasttree_extend(**{**ok, **bad})
    for bad in (dict(kv_entries=s.gt[:1].contiguous()), dict(q=s.gq[:6], o=o[:6]), dict(k_buffer=s.gk[:, :1], v_buffer=s.gv[:, :1])):
        with pytest.raises(lib.FastTreeError):
            fasttree.fasttree_extend(**{**ok, **bad})
    with pytest.raises(ValueError):
        extend.extend(s.gq, s.gk, s.gv, o, s.gt, s.plan, 1.0, path="fast")
