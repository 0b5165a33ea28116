"""The bounded waits of ft_extend's tensor-core kernel: short where nothing happens, patient where the CTA goes on."""
import ctypes

import pytest
import torch

from ft_b200 import lib
from test_extend_gpu import Step
from test_extend_queues_gpu import against_oracle, replan


def test_self_test_refuses_bad_arguments():
    handle, res = lib.load(), (ctypes.c_int * 2)()
    assert handle.ft_selftest_extend_wait(2000, None, None) == -1 and b"NULL" in handle.ft_last_error()
    for limit in (-1, 0, 63, (1 << 16) + 1):
        assert handle.ft_selftest_extend_wait(limit, res, None) == -1 and b"probes" in handle.ft_last_error()


@pytest.mark.gpu
def test_waits_run_out_end_on_the_abort_flag_and_follow_steps():
    """No copy, MMA or tensor memory is in flight: what is shown is what the wait routine answers."""
    handle, res = lib.load(), (ctypes.c_int * 2)(7, 7)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for limit in (64, 1000):
        assert handle.ft_selftest_extend_wait(limit, res, stream) == 0
        assert res[0] == 0 and res[1] <= 1 << 16                 # the kernel's own limit is the decode kernels'
        assert lib.read_device_status() == lib.FT_DEV_WAIT_TIMEOUT and lib.read_device_status() == 0
    Step([60, 20], [9, 1], [], 8, 2, 64, torch.float16).check()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_rows_computed_again_for_longer_than_a_wait_lasts(d):
    """NaN in the newest token's value, in a long context on one CTA: the rows that do not see it go one by one, and the other
    roles, and the next task, wait for them for seconds."""
    n, e = 40000, 64
    s = Step([n], [e], [], 4, 2, d, torch.bfloat16)
    replan(s, 1)
    check = against_oracle(s, -1.0)
    s.gv[s.table[0, n - 1].long()] = float("nan")
    check(list(range(e - 1)))
