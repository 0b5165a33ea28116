"""The schedule of extend attention, checked on the host: what every query token is shown, exactly once, and nothing else."""
import ctypes
import random

import numpy as np
import pytest
import torch

import extend_cases
from ft_b200 import extend, lib

ITEM, TILE = 32, 8


def shown(info, table, entries):
    """Per q row: the pool rows it is shown (with repetitions, were there any), its writers and the partial rows of its merge
    list."""
    t = table.tolist()
    items = [t[info.items_off + ITEM * i:info.items_off + ITEM * (i + 1)] for i in range(info.num_items)]
    words, group = info.tile_tokens // 32, info.num_qo_heads // info.num_kv_heads

    def offsets(rec):
        lo, hi, n, place = rec[:4]
        if place < 0:
            return [((hi << 32) | (lo & 0xffffffff)) + i for i in range(n)]
        e = info.extra_off + place
        return [(t[e + 2 * i + 1] << 32) | (t[e + 2 * i] & 0xffffffff) for i in range(n)]

    seen, writers, parts = {}, {}, {}
    for it in items:
        t0, t1, step, q_tiles, length, tile0 = it[:6]
        recs = {k: t[info.tiles_off + TILE * (tile0 + k):info.tiles_off + TILE * (tile0 + k + 1)] for k in range(t0, t1)}
        offs = {k: offsets(r) for k, r in recs.items()}
        assert it[24:32] == recs[t0] and tile0 + t1 <= info.num_tiles
        assert all(r[2] == min(info.tile_tokens, length - k * info.tile_tokens) > 0 for k, r in recs.items())
        for w in range(2):
            tok0, ntok, lo, hi, part, q_tile, first, block_tile = it[8 + 8 * w:16 + 8 * w]
            assert 0 <= q_tile < q_tiles and block_tile in (0, 1)
            if ntok:
                assert t0 <= lo < hi <= t1 and ntok * group <= max(info.rows_per_tile, group)
            for tok in range(ntok):
                q_row = t[info.tokens_off + 2 * (tok0 + tok)]
                got = []
                for k in range(lo, hi, step):
                    place = recs[k][4 + block_tile]
                    if place < 0:
                        assert recs[k][2] == info.tile_tokens
                        got += offs[k]
                    else:
                        m = info.extra_off + place + (first + tok) * words
                        bits = [(t[m + i // 32] >> (i % 32)) & 1 for i in range(info.tile_tokens)]
                        assert not any(bits[recs[k][2]:])
                        got += [x for x, bit in zip(offs[k], bits) if bit]
                seen.setdefault(q_row, []).extend(int(entries[x]) for x in got)
                if part >= 0:
                    row = t[info.extra_off + part + tok]
                    assert (row == -2) == (not got)
                    if got:
                        parts.setdefault(q_row, []).append(row)
                else:
                    writers[q_row] = writers.get(q_row, 0) + 1
    merged = {}
    for i in range(info.num_merged):
        q_row, off, n, _ = t[info.merge_off + 4 * i:info.merge_off + 4 * i + 4]
        merged[q_row] = t[info.merge_rows_off + off:info.merge_rows_off + off + n]
        writers[q_row] = writers.get(q_row, 0) + 1
    return seen, writers, parts, merged


def check(seq, ext, shared, hq, hkv, d, dtype=torch.float16, window=0, sms=148):
    table, _ = extend_cases.pool(seq, ext, shared)
    width = table.shape[1]
    info, plan, _, _ = extend.host_plan(seq, ext, [r * width for r in range(len(seq))], hq, hkv, d, dtype,
                                        shared_prefixes=shared, window=window, num_sms=sms)
    entries = table.reshape(-1).numpy()
    seen, writers, parts, merged = shown(info, plan, entries)
    row = 0
    for r, (n, e) in enumerate(zip(seq, ext)):
        for i in range(e):
            pos = n - e + i
            want = entries[r * width + (max(0, pos - window + 1) if window else 0):r * width + pos + 1]
            assert sorted(seen[row]) == sorted(want.tolist()), (r, i)
            assert writers[row] == 1
            assert sorted(merged.get(row, [])) == sorted(parts.get(row, []))
            row += 1
    assert row == info.num_tokens == sum(ext) and set(seen) == set(range(row))
    used = sorted(x for p in parts.values() for x in p)
    assert used == list(range(info.partial_rows))                  # no partial row has two writers
    # every task is dealt once
    sms = plan[info.sms_off:info.sms_off + 16 * info.num_sms].reshape(-1, 16)
    tasks = plan[info.sm_tasks_off:info.sm_tasks_off + info.num_items * hkv]
    assert sms[0, 0] == 0 and sms[-1, 1] == info.num_items * hkv
    assert (sms[:, 0] <= sms[:, 1]).all() and (sms[1:, 0] == sms[:-1, 1]).all()
    for a, b, first, _, t0, t1, tile0, _, *rec in sms.tolist():
        assert first == (tasks[a] if a < b else -1)
        if a < b:
            it = plan[info.items_off + ITEM * (first // hkv):info.items_off + ITEM * (first // hkv + 1)].tolist()
            assert [t0, t1, tile0] == [it[0], it[1], it[5]] and rec[:4] == it[24:28]
    assert sorted(tasks.tolist()) == list(range(info.num_items * hkv))
    return info


@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 128), (torch.bfloat16, 256), (torch.float32, 128),
                                     (torch.float16, 16)])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (16, 16), (28, 4), (16, 1), (5, 1)])
def test_every_token_is_shown_its_positions_once(dtype, d, hq, hkv):
    check([1, 130, 257, 40], [1, 130, 7, 40], [], hq, hkv, d, dtype)
    check([700] * 6, [1, 0, 3, 1, 60, 2], [(list(range(6)), 500)], hq, hkv, d, dtype)
    check([300, 310, 500, 520, 90], [9, 17, 1, 33, 90], [([0, 1], 200), ([2, 3], 470), ([0, 1, 2, 3], 128)], hq, hkv, d, dtype)


@pytest.mark.parametrize("window", [1, 2, 100, 128, 1000, 5000])
def test_windows(window):
    check([900, 300, 1500], [40, 300, 1], [], 8, 2, 128, window=window)
    check([700] * 5, [3, 1, 20, 1, 1], [(list(range(5)), 640)], 8, 2, 128, window=window)
    check([700] * 5, [3, 1, 20, 1, 1], [(list(range(5)), 640)], 8, 2, 256, torch.bfloat16, window=window)


def test_no_requests_and_requests_without_new_tokens():
    assert check([], [], [], 8, 2, 128).num_items == 0
    assert check([50, 60], [0, 0], [([0, 1], 50)], 8, 2, 128).num_items == 0
    check([50, 60, 70], [0, 1, 0], [([0, 1, 2], 50)], 8, 2, 128)


def test_long_context_is_cut_into_items():
    info = check([20000], [1], [], 8, 1, 128)
    assert info.num_items > 20 and info.num_merged == 1
    info = check([20000] * 2, [1, 1], [([0, 1], 19990)], 8, 1, 128)
    assert info.num_items > 20


def test_a_shared_prefix_stands_once():
    n = 16
    alone = check([4100] * n, [2] * n, [], 8, 2, 128)
    together = check([4100] * n, [2] * n, [(list(range(n)), 4098)], 8, 2, 128)
    assert together.num_tiles < alone.num_tiles
    def tokens(info, plan):
        return sum(plan[info.tiles_off + TILE * k + 2] for k in range(info.num_tiles))

    table, _ = extend_cases.pool([4100] * n, [2] * n, [(list(range(n)), 4098)])
    starts = [r * table.shape[1] for r in range(n)]
    a = extend.host_plan([4100] * n, [2] * n, starts, 8, 2, 128, torch.float16)
    b = extend.host_plan([4100] * n, [2] * n, starts, 8, 2, 128, torch.float16, shared_prefixes=[(list(range(n)), 4098)])
    assert tokens(b[0], b[1]) == 4098 + 2 * n and tokens(a[0], a[1]) == 4100 * n


def test_random_steps():
    rng = random.Random(5)
    for _ in range(60):
        n = rng.randint(1, 12)
        shared_len = rng.choice((0, rng.randint(1, 600)))
        cached = [shared_len + rng.choice((0, rng.randint(0, 500))) for _ in range(n)]
        ext = [rng.choice((0, 1, rng.randint(1, 90))) for _ in range(n)]
        seq = [c + e for c, e in zip(cached, ext)]
        groups = []
        if shared_len and n > 1:
            groups.append((list(range(n)), shared_len))
            half = list(range(0, n, 2))
            if len(half) > 1:
                groups.append((half, min(cached[m] for m in half)))
        hq, hkv = rng.choice(((8, 2), (4, 4), (7, 1), (16, 2)))
        check(seq, ext, groups, hq, hkv, rng.choice((64, 128, 256)), rng.choice((torch.float16, torch.float32)),
              window=rng.choice((0, 0, rng.randint(1, 700))), sms=rng.choice((4, 148)))


def test_offsets_beyond_32_bits():
    start = [3 << 32, (3 << 32) + 1000]
    info, plan, _, _ = extend.host_plan([300, 200], [5, 6], start, 8, 2, 128, torch.float16)
    places = set()
    for k in range(info.num_tiles):
        lo, hi, n, place = (int(x) for x in plan[info.tiles_off + TILE * k:info.tiles_off + TILE * k + 4])
        if place < 0:
            places |= {((hi << 32) | (lo & 0xffffffff)) + i for i in range(n)}
        else:
            e = plan[info.extra_off + place:info.extra_off + place + 2 * n].reshape(-1, 2).astype(np.int64)
            places |= set(((e[:, 1] << 32) | (e[:, 0] & 0xffffffff)).tolist())
    assert places == set(range(start[0], start[0] + 300)) | set(range(start[1], start[1] + 200))
    assert info.kv_entries_len == (3 << 32) + 1200


def test_refusals():
    ok = dict(seq_lens=[5, 6], extend_lens=[1, 2], kv_starts=[0, 10], num_qo_heads=8, num_kv_heads=2, head_dim=128,
              dtype=torch.float16)
    extend.host_plan(**ok)
    for bad in (dict(extend_lens=[1]), dict(extend_lens=[6, 1]), dict(extend_lens=[-1, 1]), dict(kv_starts=[-1, 0]),
                dict(num_qo_heads=7), dict(num_kv_heads=0), dict(dtype=torch.int8), dict(window=-1), dict(seq_lens=[5.5, 6.5]),
                dict(shared_prefixes=[([0, 1], 5)]), dict(shared_prefixes=[([0, 2], 1)]), dict(shared_prefixes=[([0, 1], -1)])):
        with pytest.raises(ValueError):
            extend.host_plan(**{**ok, **bad})
    with pytest.raises(lib.FastTreeError):
        extend.host_plan(**{**ok, "head_dim": 96})
    with pytest.raises(lib.FastTreeError):
        extend.host_plan(**{**ok, "seq_lens": [2 ** 31, 6]})
    with pytest.raises(ValueError):
        extend.prepare(**ok, device="cpu")


def build(seq, ext, kv, q, shared, batch=None):
    """ft_extend_plan_build as a C program calls it: its status (a plan that it makes is freed)."""
    i64 = ctypes.c_int64 * len(seq)
    handle = ctypes.c_void_p()
    clib = lib.load()
    rc = clib.ft_extend_plan_build(i64(*seq), i64(*ext), i64(*kv), i64(*q), i64(*shared), len(seq), 8, 2, 128, 2, 0, 148,
                                   ctypes.byref(handle))
    assert (rc == 0) == bool(handle.value)
    if handle.value:
        clib.ft_extend_plan_free(handle)
    return rc


def test_refusals_at_the_c_entry():
    top = 2 ** 63 - 1
    assert build([5, 6], [1, 2], [0, 10], [0, 1], [0, 0]) == 0
    assert build([5, 6], [1, 2], [0, 10], [7, 2], [0, 0]) == 0       # rows in any order, with gaps
    assert build([5, 6, 4], [1, 2, 0], [0, 10, 20], [0, 1, 1], [0, 0, 0]) == 0  # a request without queries has no rows
    assert build([5, 6], [1, 2], [0, 10], [1, 0], [0, 0]) != 0       # row 1 twice
    assert build([5, 6], [1, 2], [0, 10], [0, 0], [0, 0]) != 0
    assert build([-2 ** 63, 6], [1, 2], [0, 10], [0, 1], [0, 0]) != 0
    assert build([5, 6], [1, 2], [top, 10], [0, 1], [0, 0]) != 0     # kv_start + seq_len would wrap
    assert build([5, 6], [1, 2], [0, 10], [top, 1], [0, 0]) != 0


def test_descriptions_that_are_no_plan_are_refused():
    """ft_extend reads only the host's description before it launches: one whose parts do not lie in its table, or whose sizes
    no kernel is compiled for, is an error of the call."""
    info = extend.host_plan([9000, 60], [2, 7], [0, 9000], 8, 2, 128, torch.float16)[0]
    clib = lib.load()

    def call(**changes):
        a = lib.ExtendArgs()
        a.dtype, a.num_qo_heads, a.num_kv_heads, a.head_dim = 0, 8, 2, 128  # FT_F16
        ctypes.memmove(ctypes.byref(a.plan), ctypes.byref(info), ctypes.sizeof(info))
        for k, v in changes.items():
            setattr(a.plan, k, v)
        rc = clib.ft_extend(ctypes.byref(a))
        return rc, clib.ft_last_error().decode()

    assert info.num_merged > 0
    assert "is NULL" in call()[1]  # the description itself passes
    for part in ("items_off", "tokens_off", "tiles_off", "extra_off", "sms_off", "sm_tasks_off", "merge_off", "merge_rows_off"):
        for value in (-4, info.table_ints + 4, getattr(info, part) + 1):
            rc, text = call(**{part: value})
            assert rc != 0 and "do not lie in its table" in text, part
    for count in ("num_items", "num_tiles", "num_sms", "num_merged"):
        rc, text = call(**{count: 2 ** 28})
        assert rc != 0 and "do not lie in its table" in text, count
    for sizes in (dict(num_sms=0), dict(tile_tokens=64), dict(tile_tokens=0), dict(rows_per_tile=64), dict(rows_per_tile=0)):
        rc, text = call(**sizes)
        assert rc != 0 and "sizes are not a plan's" in text, sizes
    rc, text = call(num_items=-1)
    assert rc != 0 and "negative" in text
