"""The policy operators' limits at the C-ABI (no GPU): what a launch cannot hold is refused on the host, by name."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from fair_marl_amd import _lib


@pytest.mark.parametrize('B', [(1 << 26) - 3, (1 << 26) - 1])
def test_a_step_of_more_threads_than_a_launch_holds(B):
    """just below 2^26 heads, a wave each: 2^32 threads"""
    lib, rows, p = _lib.load(), _lib.FmarlRows(4096, 16, 16, 16), C.c_void_p(4096)
    m = _lib.FmarlMemory(L=1, B=B, H=1, dk=16, dv=16, dtype=0, scale=1.0, shared_decay=0, q=rows, k=rows, v=rows, log_decay=4096, decay_stride_l=2, decay_stride_b=1, decay_stride_h=1)
    assert lib.fmarl_memory_step(m, rows, p, None) == 1 and b'too many' in lib.fmarl_last_error()


def test_no_rows_need_no_workspace():
    """a batch without rows, few and many actions: a size, not a division by the rows of a chunk (in a process of its own, which such a division would end)"""
    code = """
from fair_marl_amd import _lib
for dtype in (_lib.T_F32, _lib.T_BF16, _lib.T_F16):
    for features, actions in ((1, 1), (64, 5), (64, 90), (300, 5), (16384, 1 << 20)):
        a = _lib.FmarlActions(rows=0, features=features, actions=actions, dtype=dtype, action_type=0, available_type=0, x=None, x_stride=features, weight=4096, weight_stride=features)
        print([_lib.load().fmarl_action_log_probs_workspace(a, backward) for backward in (0, 1)], flush=True)
"""
    done = subprocess.run([sys.executable, '-c', code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and done.stdout.split('\n')[:-1] == ['[256, 256]'] * 15, (done.returncode, done.stdout, done.stderr[-300:])
