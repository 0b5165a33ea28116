"""Outputs of ft_append and ft_extend that share memory with what the call reads: refused; columns or heads of one buffer: taken."""
import ctypes

import pytest
import torch

import fasttree
from ft_b200 import extend, lib
from test_extend_gpu import Step

gpu = pytest.mark.gpu
E, Q, D = 2, 8, 64                       # bytes of an element, query heads, head_dim
ROW = Q * D


def extend_answer(o, q=(1 << 20, ROW, D), k=(1 << 28, 2 * D, D), rows=10, tokens=10, hq=Q):
    """Kernel names for (address, strides) triples of o, q and both pools, or the refusal.  Nothing is launched."""
    info, _, _, _ = extend.host_plan([tokens], [tokens], [0], hq, 2 if hq > 1 else 1, D, torch.float16)
    a = lib.ExtendArgs()
    a.dtype, a.num_qo_heads, a.num_kv_heads, a.head_dim, a.plan = lib.FT_F16, hq, 2 if hq > 1 else 1, D, info
    a.sm_scale, a.logit_cap, a.q_rows, a.kv_rows, a.kv_entries_len = 1.0, -1.0, tokens, rows, tokens
    a.kv_entries = a.plan_table = a.mid_o = a.mid_lse = 1 << 34
    a.o, a.o_stride0, a.o_stride1 = o
    a.q, a.q_stride0, a.q_stride1 = q
    a.k_buffer, a.k_stride0, a.k_stride1 = k
    a.v_buffer, a.v_stride0, a.v_stride1 = k
    handle = lib.load()
    name = handle.ft_extend_path_name(ctypes.byref(a))
    return name.decode() if name is not None else handle.ft_last_error().decode()


def test_output_over_the_queries():
    at = 1 << 20
    for shift in (0, E * D, E * ROW, -E * ROW, 9 * E * ROW, E * (9 * ROW + ROW - 8), 16, -16):
        assert extend_answer((at + shift, ROW, D)) == "o overlaps q"
    for shift in (10 * E * ROW, -10 * E * ROW):
        assert extend_answer((at + shift, ROW, D)).startswith("extend_")


def test_columns_and_heads_of_one_buffer():
    at, wide = 1 << 20, 3 * ROW
    assert extend_answer((at + E * ROW, wide, D), (at, wide, D)).startswith("extend_")             # [tokens, 3, heads, d]
    assert extend_answer((at, wide, D), (at + 2 * E * ROW, wide, D)).startswith("extend_")
    assert extend_answer((at + E * (ROW - D), wide, D), (at, wide, D)) == "o overlaps q"
    assert extend_answer((at + E * D, 2 * ROW, 2 * D), (at, 2 * ROW, 2 * D)).startswith("extend_")  # [tokens, heads, 2, d]
    assert extend_answer((at + E * D - 16, 2 * ROW, 2 * D), (at, 2 * ROW, 2 * D)) == "o overlaps q"
    assert extend_answer((at + E * D, D, 20 * D), (at, D, 20 * D)) == "o overlaps q"                # heads outermost, a token apart
    assert extend_answer((at + 10 * E * D, D, 20 * D), (at, D, 20 * D)).startswith("extend_")       # [heads, 2, tokens, d]
    assert extend_answer((at, ROW, D), (at + 8, 3 * ROW, D)) == "o overlaps q"                      # of no common period
    assert extend_answer((at, 7, 5), (at, 7, 5), tokens=1, hq=1) == "o overlaps q"                  # strides along one entry
    assert extend_answer((at + E * D, 7, 5), (at, 7, 5), tokens=1, hq=1).startswith("extend_")


def test_output_over_the_pool():
    at = 1 << 28
    assert extend_answer((at, ROW, D)) == "o overlaps the pool"
    assert extend_answer((at + E * 10 * 2 * D - 16, ROW, D)) == "o overlaps the pool"
    assert extend_answer((at + E * 10 * 2 * D, ROW, D)).startswith("extend_")


@gpu
def test_tensors_of_one_storage():
    s = Step([30, 20], [4, 3], [], Q, 2, D, torch.float16, pad_rows=0)
    both = torch.zeros(15, Q, D, dtype=torch.float16, device="cuda")
    both[:7] = s.gq
    with pytest.raises(lib.FastTreeError, match="o overlaps q"):
        fasttree.fasttree_extend(both[:7], s.gk, s.gv, both[1:8], s.gt, s.plan, s.scale)
    want, _ = s.run()
    o = both[7:14]
    fasttree.fasttree_extend(both[:7], s.gk, s.gv, o, s.gt, s.plan, s.scale)
    assert torch.equal(o, want)
    columns = torch.zeros(7, 2, Q, D, dtype=torch.float16, device="cuda")
    columns[:, 1] = s.gq
    fasttree.fasttree_extend(columns[:, 1], s.gk, s.gv, columns[:, 0], s.gt, s.plan, s.scale)
    assert torch.equal(columns[:, 0], want)
    with pytest.raises(lib.FastTreeError, match="o overlaps the pool"):
        fasttree.fasttree_extend(s.gk[:7].expand(7, 2, D).repeat(1, 4, 1), s.gk, s.gv, s.gv[:28].view(7, Q, D), s.gt, s.plan, s.scale)


@gpu
def test_append_into_memory_that_it_reads():
    t = 6
    buf = torch.randn(t + 1, 2 * Q + 4, D, device="cuda").half()
    q, k, v = buf[:t, :Q], buf[:t, Q:Q + 2], buf[:t, Q + 2:Q + 4]
    kb, vb = torch.zeros(20, 2, D, device="cuda").half(), torch.zeros(20, 2, D, device="cuda").half()
    slots = torch.arange(t, device="cuda")
    keep = buf.clone()
    for out, message in ((buf[1:, :Q], "q_out overlaps q"), (buf[:t, 1:Q + 1], "q_out overlaps q"), (buf[:t, Q:2 * Q], "q_out overlaps k"),
                         (buf[:t, Q + 2:2 * Q + 2], "q_out overlaps v"), (kb.view(5, Q, D)[:5], "q_out overlaps k_buffer"), (vb.view(5, Q, D), "q_out overlaps v_buffer")):
        n = out.shape[0]
        with pytest.raises(lib.FastTreeError, match=message):
            fasttree.fasttree_append(q[:n], k[:n], v[:n], kb, vb, slots[:n], q_out=out)
    assert torch.equal(buf, keep) and not kb.any() and not vb.any()
    out = buf[:t, Q + 4:]                                        # heads of its own in the same rows
    fasttree.fasttree_append(q[:, :Q], k, v, kb, vb, slots, q_out=torch.empty_like(q))
    fasttree.fasttree_append(q, k, v, kb, vb, slots)             # in place
    assert torch.equal(buf, keep) and torch.equal(kb[:t], k) and torch.equal(vb[:t], v)
    fasttree.fasttree_append(buf[:t, 4:Q], k, v, kb, vb, slots, q_out=out[:, :Q - 4])
    assert torch.equal(out[:, :Q - 4], keep[:t, 4:Q])


@gpu
@pytest.mark.parametrize("hkv,dtype", [(2, torch.float16), (40, torch.bfloat16), (3, torch.float32)])
def test_keys_turned_in_the_pool(hkv, dtype):
    """k and v are the pool's own rows: the same as from a copy of them."""
    t, rows = 37, 50
    g = torch.Generator().manual_seed(hkv)
    kb, vb = (torch.randn(rows, hkv, D, generator=g).to(dtype).cuda() for _ in range(2))
    angle = torch.randn(rows, D // 2, generator=g)
    table, pos = torch.cat([angle.cos(), angle.sin()], 1).cuda(), torch.randint(0, rows, (t,), generator=g).cuda()
    slots = torch.arange(5, 5 + t, device="cuda")
    want_k, want_v = kb.clone(), vb.clone()
    fasttree.fasttree_append(None, kb[5:5 + t].clone(), vb[5:5 + t].clone(), want_k, want_v, slots, positions=pos, cos_sin=table)
    fasttree.fasttree_append(None, kb[5:5 + t], vb[5:5 + t], kb, vb, slots, positions=pos, cos_sin=table)
    assert torch.equal(kb, want_k) and torch.equal(vb, want_v)
