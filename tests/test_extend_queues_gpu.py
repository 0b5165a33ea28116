"""ft_extend where a CTA works through a queue of tasks: phases, buffers and counters that go on from task to task.  Steps that fit a
test are too small to give one of 148 SMs a second task, so these are planned for a few."""
import random
import threading

import numpy as np
import pytest
import torch

import extend_cases
from ft_b200 import extend, lib
from test_extend_bad_rows_gpu import expected
from test_extend_gpu import DTYPES, Step

pytestmark = pytest.mark.gpu
FORMS = [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 64), ("fp32", 256)]


def replan(s, made_for, num_sms=None, seed=0):
    """The step's plan for `made_for` SMs; its tasks dealt anew, shuffled, to `num_sms` CTAs, if given.  The kinds of its items and
    the length of the longest queue."""
    info, table, _, _ = extend.host_plan(s.seq, s.ext, [r * s.table.shape[1] for r in range(len(s.seq))], s.q.shape[1], s.k.shape[1],
                                         s.d, s.dtype, shared_prefixes=s.shared, window=s.window, num_sms=made_for)
    items = table[info.items_off:info.items_off + 32 * info.num_items].reshape(-1, 32)
    if num_sms is not None:
        tasks = list(range(info.num_items * info.num_kv_heads))
        random.Random(seed).shuffle(tasks)
        queues, at = [tasks[c::num_sms] for c in range(num_sms)], 0
        dealt, sms = [], []
        for queue in queues:
            dealt += queue
            first = items[queue[0] // info.num_kv_heads].tolist() if queue else [0] * 32
            sms += [at, at + len(queue), queue[0] if queue else -1, 0, first[0], first[1], first[5], 0, *first[24:28], 0, 0, 0, 0]
            at += len(queue)
        dealt += [0] * (-len(dealt) % 4)
        info.sm_tasks_off, info.sms_off, info.num_sms = len(table), len(table) + len(dealt), num_sms
        table = np.concatenate([table, np.array(dealt + sms, dtype=np.int32)])
        info.table_ints = len(table)
    s.plan = extend.ExtendPlan(info, torch.from_numpy(table).cuda(), s.seq, s.ext)
    ends = table[info.sms_off:info.sms_off + 16 * info.num_sms].reshape(-1, 16)[:, :2]
    kinds = {"pair" if q_tiles == 2 else "alternate" if step == 2 else "single" for step, q_tiles in items[:, 2:4].tolist()}
    return kinds, int((ends[:, 1] - ends[:, 0]).max())


def against_oracle(s, cap):
    """Runs the step and holds it to the oracle, which is computed once."""
    out, want_lse, absv, size = expected(s, s.table, cap)
    tol, tol_lse = extend_cases.bounds(s.dtype, out, absv, size, cap, s.d)
    n = sum(s.ext)

    def run(rows=slice(None)):
        o, lse = s.run(cap=cap)
        err, err_lse = (o[:n].double().cpu() - out[:n]).abs(), (lse[:n].double().cpu() - want_lse[:n]).abs()
        assert bool((err <= tol[:n])[rows].all()), (err / tol[:n])[rows].max().item()
        assert bool((err_lse <= tol_lse[:n])[rows].all()), (err_lse / tol_lse[:n])[rows].max().item()
        assert o[n:].isnan().all() and lse[n:].isnan().all()

    return run


def mixed(dtype, d, window=0, layout="scattered", seed=0):
    """Prompts of several query tiles, questions, single tokens; alone, on prefixes of two groups, and on one of those nested."""
    seq = [700, 300, 333, 420, 64, 1, 129, 390, 395, 260, 6000, 40, 512, 450, 3500]
    ext = [300, 40, 1, 120, 64, 1, 129, 9, 1, 200, 1, 0, 33, 70, 2]
    shared = [([1, 2, 3, 7, 8], 250), ([3, 7, 8], 290), ([0, 12, 13], 380)]
    return Step(seq, ext, shared, 8, 2, d, DTYPES[dtype], window=window, layout=layout, seed=seed, q_scale=2.0)


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("window", [0, 130, 2500])
@pytest.mark.parametrize("cap", [-1.0, 6.0])
def test_queues_against_the_oracle(dtype, d, window, cap):
    s = mixed(dtype, d, window, layout="prefill" if cap > 0 else "scattered", seed=d + window)
    kinds, check = set(), against_oracle(s, cap)
    for made_for, num_sms in ((1, None), (3, None), (148, 1), (148, 5), (10, 2)):
        some, longest = replan(s, made_for, num_sms, seed=made_for)
        assert longest >= 8
        kinds |= some
        check()
    if d in (64, 128) and dtype != "fp32" and window != 130:
        assert kinds == {"pair", "alternate", "single"}


@pytest.mark.parametrize("dtype,d", FORMS)
def test_queues_repeat_and_do_not_depend_on_the_queue(dtype, d):
    """The same items in other queues give the same bits: nothing of a task reaches the next one."""
    s = mixed(dtype, d)
    n = sum(s.ext)
    _, longest = replan(s, 148, 4096)
    assert longest == 1                                          # every task in a queue of its own
    want, want_lse = s.run(cap=6.0)
    for num_sms in (1, 2, 7):
        for seed in range(3):
            replan(s, 148, num_sms, seed)
            o, lse = s.run(cap=6.0)
            assert torch.equal(o[:n], want[:n]) and torch.equal(lse[:n], want_lse[:n])


@pytest.mark.parametrize("dtype,d", FORMS)
@pytest.mark.parametrize("cap", [-1.0, 6.0])
def test_values_that_are_no_numbers_out_of_sight_in_queues(dtype, d, cap):
    """Every request's newest token holds them: all other queries stay within their bounds."""
    s = mixed(dtype, d)
    check = against_oracle(s, cap)
    last = [sum(s.ext[:r + 1]) - 1 for r in range(len(s.ext)) if s.ext[r]]
    good = [i for i in range(sum(s.ext)) if i not in last]
    newest = torch.stack([s.table[r, s.seq[r] - 1] for r in range(len(s.seq)) if s.ext[r]]).long()
    k, v = s.gk.clone(), s.gv.clone()
    for num_sms in (1, 4):
        replan(s, 148, num_sms)
        for value in (float("nan"), float("inf"), -float("inf")):
            s.gk.copy_(k), s.gv.copy_(v)
            s.gk[newest], s.gv[newest] = value, value
            check(good)


@pytest.mark.parametrize("dtype,d", FORMS)
def test_query_tiles_of_rows_that_are_not_consecutive(dtype, d):
    """Requests of two prefixes in turn: a tile takes every other request's rows of q."""
    seq, ext = [200 + 3 * i for i in range(14)], [1 + i % 4 for i in range(14)]
    s = Step(seq, ext, [(list(range(0, 14, 2)), 190), (list(range(1, 14, 2)), 180)], 8, 2, d, DTYPES[dtype])
    s.check()
    replan(s, 148, 1)
    s.check(cap=5.0)


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 128)])
def test_positions_beyond_16_bits(dtype, d):
    s = Step([70001, 66000], [2, 1], [([0, 1], 65500)], 2, 1, d, DTYPES[dtype])
    check = against_oracle(s, -1.0)
    for made_for, num_sms in ((148, None), (2, None), (148, 3)):
        replan(s, made_for, num_sms)
        check()


def test_threads_at_once():
    """Several host threads, each on a stream of its own, plan and call at the same time."""
    steps = [mixed(dtype, d, seed=i) for i, (dtype, d) in enumerate([("bf16", 64), ("fp16", 128), ("bf16", 256), ("fp32", 64)])]
    want = [s.run(cap=10.0) for s in steps]
    outs, errors = [[] for _ in steps], []

    def work(s, out):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(8):
                    info, table, _, _ = extend.host_plan(s.seq, s.ext, [r * s.table.shape[1] for r in range(len(s.seq))], 8, 2, s.d, s.dtype,
                                                         shared_prefixes=s.shared)
                    plan = extend.ExtendPlan(info, torch.from_numpy(table).cuda(), s.seq, s.ext)
                    o = torch.empty_like(s.gq)
                    extend.extend(s.gq, s.gk, s.gv, o, s.gt, plan, s.scale, logit_cap=10.0)
                    torch.cuda.current_stream().synchronize()
                    out.append(o)
        except Exception as e:                                   # noqa: BLE001 - reported by the test's own thread
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=x) for x in zip(steps, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    torch.cuda.synchronize()
    assert lib.read_device_status() == 0
    for s, (o, _), got in zip(steps, want, outs):
        n = sum(s.ext)
        assert len(got) == 8 and all(torch.equal(x[:n], o[:n]) for x in got)
