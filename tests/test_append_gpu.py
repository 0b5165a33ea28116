"""ft_append: rotation and writes to the paged cache, against the formula in 64 bits."""
import ctypes
import math

import pytest
import torch

import fasttree
from ft_b200 import lib

gpu = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def table_of(length, rot, device="cuda"):
    half = rot // 2
    angle = torch.outer(torch.arange(length, dtype=torch.float64), torch.exp(torch.arange(half, dtype=torch.float64) * (-math.log(1e4) / half)))
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def turned(x, table, positions, sections, interleaved):
    """In 64 bits from the fp32 table: (turned x, sum of the absolute products of every element)."""
    rot = table.shape[1]
    half = rot // 2
    pos = positions.reshape(-1, x.shape[0]).long()
    axis = [a for a, n in enumerate(sections or [half]) for _ in range(n)]
    y = x.double().clone()
    size = x.double().abs()
    for i in range(half):
        c = table[pos[axis[i]], i].double()[:, None]
        s = table[pos[axis[i]], half + i].double()[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        xa, xb = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
        size[..., a], size[..., b] = (xa * c).abs() + (xb * s).abs(), (xb * c).abs() + (xa * s).abs()
    return y, size


def close(got, want, size, dtype):
    # one rounding to the storage type; the two products, their sum and the fp32 intermediate: three half steps of 2^-24 each
    u = 2.0 ** -24 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = torch.finfo(torch.float16).smallest_normal * torch.finfo(torch.float16).eps if dtype == torch.float16 else 0.0
    bound = u * want.abs() + 4 * 2.0 ** -24 * size + tiny
    return bool(((got.double().cpu() - want.cpu()).abs() <= bound.cpu()).all())


def inputs(t, hq, hkv, d, dtype, rows, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(t, (hq + 2 * hkv) * d + pad, generator=g).to(dtype).cuda()
    q, k, v = (x.unflatten(1, (-1, d)) for x in qkv[:, pad:].split([hq * d, hkv * d, hkv * d], 1))
    kb, vb = torch.randn(rows, hkv, d, generator=g).to(dtype).cuda(), torch.randn(rows, hkv, d, generator=g).to(dtype).cuda()
    slots = torch.randperm(rows, generator=g)[:t].cuda()
    return q, k, v, kb, vb, slots


def run_and_check(q, k, v, kb, vb, slots, table, positions, sections, interleaved, dtype, q_out=None):
    want_q, size_q = turned(q, table, positions, sections, interleaved) if table is not None else (q.double(), q.double().abs())
    want_k, size_k = turned(k, table, positions, sections, interleaved) if table is not None else (k.double(), k.double().abs())
    kb0, vb0, k0, v0 = kb.clone(), vb.clone(), k.clone(), v.clone()
    out = q_out if q_out is not None else q
    fasttree.fasttree_append(q, k, v, kb, vb, slots, q_out=q_out, positions=positions, cos_sin=table, sections=sections,
                             interleaved=interleaved)
    torch.cuda.synchronize()
    assert lib.read_device_status() == 0
    assert close(out, want_q, size_q, dtype)
    keep = slots >= 0
    rows = slots[keep].long()
    assert close(kb[rows], want_k[keep], size_k[keep], dtype)
    assert torch.equal(vb[rows], v0[keep]) and torch.equal(k, k0) and torch.equal(v, v0)
    others = torch.ones(kb.shape[0], dtype=torch.bool, device="cuda")
    others[rows] = False
    assert torch.equal(kb[others], kb0[others]) and torch.equal(vb[others], vb0[others])


@gpu
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("t,hq,hkv,d,rot,axes,interleaved,padded", [
    (1, 8, 2, 128, 128, 1, False, 0), (67, 32, 8, 128, 128, 3, False, 5), (33, 28, 4, 64, 32, 1, False, 0),
    (9, 5, 1, 256, 64, 1, True, 2), (130, 16, 16, 64, 64, 3, True, 0), (21, 64, 8, 128, 128, 4, False, 1),
    (5, 4, 2, 16, 16, 1, False, 0), (5, 4, 2, 32, 8, 2, True, 0), (3, 1, 1, 128, 20, 1, False, 0), (3, 7, 1, 256, 256, 1, False, 3),
])
def test_against_the_formula(dtype, t, hq, hkv, d, rot, axes, interleaved, padded):
    dt = DTYPES[dtype]
    q, k, v, kb, vb, slots = inputs(t, hq, hkv, d, dt, t + 9, seed=t + d)
    if padded:
        slots[t - padded:] = -1
    table = table_of(1000, rot)
    half = rot // 2
    sections = None if axes == 1 else [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1)
    pos = torch.randint(0, 1000, (axes, t), generator=torch.Generator().manual_seed(t)).cuda()
    run_and_check(q, k, v, kb, vb, slots, table, pos[0] if axes == 1 else pos, sections, interleaved, dt, q_out=torch.empty_like(q.contiguous()))


@gpu
def test_in_place_int32_tables_strides_and_odd_alignment():
    for pad, dtype in ((0, torch.float16), (3, torch.bfloat16), (1, torch.float32)):
        q, k, v, kb, vb, slots = inputs(40, 8, 2, 128, dtype, 64, pad=pad)
        pos = torch.arange(40, dtype=torch.int32, device="cuda")
        run_and_check(q, k, v, kb, vb, slots.int(), table_of(64, 128), pos, None, False, dtype)
    # heads outermost in the pool, a table with wider rows, positions as one row of a larger tensor
    q, k, v, _, _, slots = inputs(40, 8, 2, 64, torch.float16, 64)
    kb, vb = torch.zeros(2, 64, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 64, 64, dtype=torch.float16, device="cuda")
    wide = torch.zeros(64, 80, device="cuda")
    wide[:, :64] = table_of(64, 64)
    pos = torch.randint(0, 64, (4, 40), device="cuda")
    run_and_check(q, k, v, kb.transpose(0, 1), vb.transpose(0, 1), slots, wide[:, :64], pos[2], None, False, torch.float16)
    run_and_check(q, k, v, kb.transpose(0, 1), vb.transpose(0, 1), slots, wide[:, :64], pos[:, :40][1:4], [8, 12, 12], False, torch.float16)


@gpu
def test_without_rotation_and_without_queries():
    q, k, v, kb, vb, slots = inputs(70, 8, 2, 128, torch.bfloat16, 90)
    run_and_check(q, k, v, kb, vb, slots, None, None, None, False, torch.bfloat16, q_out=torch.empty_like(q.contiguous()))
    kb0 = kb.clone()
    fasttree.fasttree_append(None, v, k, kb, vb, slots)          # the other way round
    assert torch.equal(kb[slots], v) and torch.equal(vb[slots], k) and not torch.equal(kb, kb0)
    pos, table = torch.arange(70, device="cuda"), table_of(70, 128)
    want, size = turned(k, table, pos, None, False)
    fasttree.fasttree_append(None, k, v, kb, vb, slots, positions=pos, cos_sin=table)
    assert close(kb[slots], want, size, torch.bfloat16)
    fasttree.fasttree_append(q[:0], k[:0], v[:0], kb, vb, slots[:0], positions=pos[:0], cos_sin=table)      # no tokens
    assert lib.read_device_status() == 0


@gpu
def test_far_rows_of_a_large_pool():
    rows, hkv, d = 70000, 128, 256                               # 2.3e9 elements: offsets beyond 31 bits
    kb = torch.zeros(rows, hkv, d, dtype=torch.float16, device="cuda")
    k = torch.randn(3, hkv, d, device="cuda").half()
    slots = torch.tensor([rows - 1, 0, 66000], device="cuda")
    fasttree.fasttree_append(None, k, k, kb, kb, slots)
    assert torch.equal(kb[slots], k) and kb[1:66000].abs().max() == 0


@gpu
def test_slots_and_positions_out_of_range_are_flagged():
    q, k, v, kb, vb, slots = inputs(6, 4, 2, 64, torch.float16, 20)
    table = table_of(50, 64)
    pos = torch.arange(6, device="cuda")
    slots[1], slots[2] = 20, -3
    kb0 = kb.clone()
    out = torch.zeros_like(q.contiguous())
    fasttree.fasttree_append(q, k, v, kb, vb, slots, q_out=out, positions=pos, cos_sin=table)
    assert lib.read_device_status() == lib.FT_DEV_BAD_KV_INDEX
    good = slots[[0, 3, 4, 5]]
    rest = [r for r in range(20) if r not in good.tolist()]
    assert torch.equal(kb[rest], kb0[rest]) and (out.abs().amax((1, 2)) > 0).all()
    slots = torch.arange(6, device="cuda")
    pos[4], pos[5] = 50, -1
    out.zero_()
    kb.copy_(kb0)
    fasttree.fasttree_append(q, k, v, kb, vb, slots, q_out=out, positions=pos, cos_sin=table)
    assert lib.read_device_status() == lib.FT_DEV_BAD_POSITION
    assert out[4:].abs().max() == 0 and torch.equal(kb[4:], kb0[4:]) and not torch.equal(kb[:4], kb0[:4])


@gpu
def test_captured_and_on_another_stream():
    q, k, v, kb, vb, slots = inputs(50, 8, 2, 128, torch.float16, 64)
    table, pos = table_of(64, 128), torch.arange(50, device="cuda")
    out = torch.empty_like(q.contiguous())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        fasttree.fasttree_append(q, k, v, kb, vb, slots, q_out=out, positions=pos, cos_sin=table)
    slots.copy_(torch.arange(50, device="cuda").flip(0))
    pos.add_(9)
    graph.replay()
    torch.cuda.synchronize()
    want, size = turned(k, table, pos, None, False)
    assert close(kb[slots], want, size, torch.float16)
    with torch.cuda.stream(side):
        fasttree.fasttree_append(q, k, v, kb, vb, slots, q_out=out, positions=pos, cos_sin=table)
    side.synchronize()
    assert close(out, *turned(q, table, pos, None, False), torch.float16)


def test_refusals_on_the_host():
    f16 = dict(dtype=torch.float16)
    k, kb, slots = torch.zeros(3, 2, 64, **f16), torch.zeros(9, 2, 64, **f16), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        fasttree.fasttree_append(None, k, k, kb, kb, slots)
    with pytest.raises(ValueError, match="torch.Tensor"):
        fasttree.fasttree_append(None, 3, k, kb, kb, slots)
    handle = lib.load()
    a = lib.AppendArgs()
    assert handle.ft_append(None) == -1
    a.dtype, a.num_kv_heads, a.head_dim = 7, 1, 64
    assert handle.ft_append(ctypes.byref(a)) == -1
    a.dtype = lib.FT_F16
    assert handle.ft_append(ctypes.byref(a)) == 0                # no tokens
    a.tokens = 2
    assert handle.ft_append(ctypes.byref(a)) == -1               # no tensors
    for field, value in (("head_dim", 96), ("rot_dim", 7), ("rot_dim", 66), ("tokens", -1), ("num_kv_heads", 0)):
        b = lib.AppendArgs()
        b.dtype, b.num_kv_heads, b.head_dim, b.tokens = lib.FT_F16, 1, 64, 0
        setattr(b, field, value)
        assert handle.ft_append(ctypes.byref(b)) < 0, field
    b = lib.AppendArgs()
    b.dtype, b.num_kv_heads, b.head_dim, b.rot_dim, b.num_axes = lib.FT_F16, 1, 64, 32, 2
    b.sections[0], b.sections[1] = 8, 9
    assert handle.ft_append(ctypes.byref(b)) == -1 and b"pairs" in handle.ft_last_error()
    b.num_axes = 5
    assert handle.ft_append(ctypes.byref(b)) == -1


@gpu
def test_refusals_of_tensors():
    q, k, v, kb, vb, slots = inputs(6, 4, 2, 64, torch.float16, 20)
    pos, table = torch.arange(6, device="cuda"), table_of(50, 64)
    ok = dict(q=q, k=k, v=v, k_buffer=kb, v_buffer=vb, slots=slots, positions=pos, cos_sin=table)
    fasttree.fasttree_append(**ok)
    pair = torch.stack([pos, pos])
    for bad in (dict(k=k.float()), dict(v=v[:5]), dict(q=q[:5]), dict(k_buffer=kb[:, :1]), dict(v_buffer=vb[:10]),
                dict(slots=slots[:5]), dict(slots=slots.float()), dict(positions=None), dict(cos_sin=None),
                dict(cos_sin=table.double()), dict(cos_sin=table[:, :63]), dict(cos_sin=table_of(50, 128)), dict(positions=pos[:4]),
                dict(positions=pair), dict(positions=pair, sections=[16]), dict(positions=pair, sections=[16, 17]),
                dict(positions=pair, sections=[-1, 33]), dict(q_out=q[:, :1]), dict(q=None, q_out=q), dict(positions=None, cos_sin=None, sections=[32]),
                dict(k=k.transpose(1, 2)), dict(slots=slots.repeat(2)[::2]), dict(q=q[0])):
        with pytest.raises(ValueError):
            fasttree.fasttree_append(**{**ok, **bad})
    assert lib.read_device_status() == 0
