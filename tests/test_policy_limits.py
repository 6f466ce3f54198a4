"""The policy operators' limits at the C-ABI (no GPU): what a launch cannot hold is refused on the host, by name."""
import ctypes as C

import pytest

from fair_marl_amd import _lib


@pytest.mark.parametrize('B', [(1 << 26) - 3, (1 << 26) - 1])
def test_a_step_of_more_threads_than_a_launch_holds(B):
    """just below 2^26 heads, a wave each: 2^32 threads"""
    lib, rows, p = _lib.load(), _lib.FmarlRows(4096, 16, 16, 16), C.c_void_p(4096)
    m = _lib.FmarlMemory(L=1, B=B, H=1, dk=16, dv=16, dtype=0, scale=1.0, shared_decay=0, q=rows, k=rows, v=rows, log_decay=4096, decay_stride_l=2, decay_stride_b=1, decay_stride_h=1)
    assert lib.fmarl_memory_step(m, rows, p, None) == 1 and b'too many' in lib.fmarl_last_error()
