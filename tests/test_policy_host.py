"""The policy operators' refusals (no GPU): every bad argument is named before anything is launched -- by the Python entry points and by the C-ABI."""
import ctypes as C

import pytest
import torch

import fair_marl_amd as fm
from fair_marl_amd import _lib


@pytest.fixture(scope='module')
def lib():
    return _lib.load()


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(ValueError, match='GPU'):
        fm.memory_chunk(z(2, 3, 1, 4), z(2, 3, 1, 4), z(2, 3, 1, 4), z(1))
    with pytest.raises(ValueError, match='GPU'):
        fm.memory_step(z(3, 1, 4), z(3, 1, 4), z(3, 1, 4), z(1), None)
    with pytest.raises(ValueError, match='GPU'):
        fm.block_norm(z(3, 4))
    with pytest.raises(ValueError, match='GPU'):
        fm.action_log_probs(z(3, 4), z(5, 4), None, z(3))


def test_shapes_and_types_are_refused_by_name():
    with pytest.raises(ValueError, match='memory_chunk: q, k'):
        fm.memory_chunk(z(3, 1, 4), z(3, 1, 4), z(3, 1, 4), z(1))
    q = z(3, 1, 4).requires_grad_()
    with pytest.raises(ValueError, match='no gradient'):
        fm.memory_step(q, q, q, z(1), None)
    for kw, text in ((dict(groups=3), 'groups'), (dict(gate=z(3, 8)), 'branch'), (dict(pre_norm=False), 'nothing'), (dict(eps=-1.0), 'eps'),
                     (dict(branch=z(3, 8), post_norm=False, post_weight=z(8)), 'post'), (dict(pre_norm=False, branch=z(3, 8), pre_bias=z(8)), 'pre')):
        with pytest.raises(ValueError, match=text):
            fm.block_norm(z(3, 8), **kw)
    with pytest.raises(ValueError, match='last axis'):
        fm.block_norm(z(2, 8193))
    for x, w in ((z(3, 4), z(5, 3)), (z(3, 4), z(4)), (z(3, 0), z(5, 0)), (z(3, 4), z(0, 4))):
        with pytest.raises(ValueError, match='action_log_probs'):
            fm.action_log_probs(x, w, None, z(3))
    with pytest.raises(ValueError, match='bias'):
        fm.action_log_probs(z(3, 4), z(5, 4), z(5, dtype=torch.float64), z(3))


def memory(**kw):
    # (addresses that are never followed: every call here is refused on the host)
    rows = _lib.FmarlRows(4096, 16, 16, 16)
    a = dict(L=4, B=2, H=1, dk=16, dv=16, dtype=0, scale=1.0, shared_decay=0, q=rows, k=rows, v=rows, log_decay=4096, decay_stride_l=2, decay_stride_b=1, decay_stride_h=1)
    a.update(kw)
    return _lib.FmarlMemory(**a)


def test_memory_entry_points_refuse(lib):
    rows, p = _lib.FmarlRows(4096, 16, 16, 16), C.c_void_p(4096)
    err = lambda: lib.fmarl_last_error()  # noqa: E731
    for kw, text in ((dict(dk=0), b'dk'), (dict(dv=129), b'dv'), (dict(L=-1), b'negative'), (dict(H=0), b'H'), (dict(dtype=3), b'dtype'), (dict(shared_decay=2), b'shared_decay'),
                     (dict(shared_decay=1), b'shared_decay'), (dict(B=1 << 31), b'too many'), (dict(log_decay=None), b'null'), (dict(q=_lib.FmarlRows()), b'null')):
        assert lib.fmarl_memory_chunk(memory(**kw), rows, p, p, None) == 1 and text in err(), kw
        assert lib.fmarl_memory_workspace(memory(**kw), 1) == 0 and text in err()
        assert lib.fmarl_memory_chunk_backward(memory(**kw), rows, None, rows, rows, rows, None, None, None, p, None) == 1 and text in err()
    assert lib.fmarl_memory_chunk(None, rows, p, p, None) == 1 and b'null' in err()
    assert lib.fmarl_memory_chunk(memory(L=0), rows, p, p, None) == 1 and b'positive' in err()
    assert lib.fmarl_memory_chunk(memory(), None, p, p, None) == 1 and lib.fmarl_memory_chunk(memory(), rows, None, p, None) == 1 and lib.fmarl_memory_chunk(memory(), rows, p, None, None) == 1
    assert lib.fmarl_memory_step(memory(), rows, p, None) == 1 and b'L must be 1' in err()
    assert lib.fmarl_memory_step(memory(L=1), None, p, None) == 1 and lib.fmarl_memory_step(memory(L=1), rows, None, None) == 1
    for args in ((None, None, rows, rows, rows), (rows, None, None, rows, rows), (rows, None, rows, None, rows), (rows, None, rows, rows, None)):
        assert lib.fmarl_memory_chunk_backward(memory(), *args, None, None, None, p, None) == 1 and b'null' in err()
    assert lib.fmarl_memory_chunk_backward(memory(), rows, None, rows, rows, rows, None, None, None, None, None) == 1
    assert lib.fmarl_memory_chunk(memory(B=0), rows, p, p, None) == 0 and lib.fmarl_memory_step(memory(L=1, B=0), rows, p, None) == 0     # nothing to do
    # the workspace: nothing to cut for many sequences, segment states for few and long ones, more of it backwards
    assert lib.fmarl_memory_workspace(memory(L=10, B=100000), 0) == 256
    few = memory(L=4096, B=2, H=2)
    assert lib.fmarl_memory_workspace(few, 1) > lib.fmarl_memory_workspace(few, 0) > 4 * 16 * 16 * 4 * 4


def block(**kw):
    a = dict(rows=4, dim=8, groups=2, dtype=0, x_dtype=0, kind=0, gate_act=0, post_norm=1, pre_norm=1, eps=1e-5, x=4096, x_stride=8, branch=4096, branch_stride=8)
    a.update(kw)
    return _lib.FmarlBlock(**a)


def test_block_norm_entry_points_refuse(lib):
    p = C.c_void_p(4096)
    w = (C.c_void_p * 5)()
    err = lambda: lib.fmarl_last_error()  # noqa: E731
    for kw, text in ((dict(rows=-1), b'rows'), (dict(dim=0), b'dim'), (dict(dim=8193), b'dim'), (dict(groups=3), b'groups'), (dict(dim=1024, groups=512), b'groups'), (dict(dtype=1, x_dtype=2), b'type'),
                     (dict(dtype=0, x_dtype=1), b'type'), (dict(kind=2), b'kind'), (dict(gate_act=-1), b'gate_act'), (dict(eps=-1.0), b'eps'), (dict(eps=float('nan')), b'eps'), (dict(x=None), b'null'),
                     (dict(branch=None, gate=4096), b'branch'), (dict(post_norm=0, post_bias=4096), b'post')):
        assert lib.fmarl_block_norm(block(**kw), p, p, None) == 1 and text in err(), kw
        assert lib.fmarl_block_norm_workspace(block(**kw)) == 0
        assert lib.fmarl_block_norm_backward(block(**kw), p, 8, p, 8, p, p, p, w, p, None) == 1 and text in err()
    assert lib.fmarl_block_norm(None, p, p, None) == 1 and lib.fmarl_block_norm(block(), None, p, None) == 1 and lib.fmarl_block_norm(block(), p, None, None) == 1
    assert lib.fmarl_block_norm(block(branch=None, pre_norm=0), p, p, None) == 1
    assert lib.fmarl_block_norm(block(rows=0, x=None, branch=None), None, None, None) == 0
    for args in ((None, p, None, w, p), (p, None, None, w, p), (p, p, None, None, p), (p, p, None, w, None)):
        assert lib.fmarl_block_norm_backward(block(), p, 8, p, 8, *args, None) == 1 and b'null' in err()
    assert lib.fmarl_block_norm_backward(block(gate=4096), p, 8, p, 8, p, p, None, w, p, None) == 1
    assert lib.fmarl_block_norm_backward(block(pre_norm=0), p, 8, p, 8, p, p, None, w, p, None) == 1 and b'pre_norm' in err()


def acts(**kw):
    a = dict(rows=4, features=8, actions=5, dtype=0, action_type=0, available_type=0, x=4096, x_stride=8, weight=4096, weight_stride=8, action=4096)
    a.update(kw)
    return _lib.FmarlActions(**a)


def test_action_log_probs_entry_points_refuse(lib):
    p = C.c_void_p(4096)
    err = lambda: lib.fmarl_last_error()  # noqa: E731
    for kw, text in ((dict(rows=-1), b'rows'), (dict(features=0), b'features'), (dict(features=16385), b'features'), (dict(actions=0), b'actions'), (dict(actions=(1 << 20) + 1), b'actions'),
                     (dict(dtype=-1), b'dtype'), (dict(action_type=3), b'action_type'), (dict(available_type=2), b'available_type'), (dict(x=None), b'null'), (dict(weight=None), b'null'),
                     (dict(action=None), b'null')):
        assert lib.fmarl_action_log_probs(acts(**kw), p, p, p, p, None) == 1 and text in err(), kw
        assert lib.fmarl_action_log_probs_workspace(acts(**kw), 0) == 0
        assert lib.fmarl_action_log_probs_backward(acts(**kw), p, p, p, p, p, p, p, p, None) == 1 and text in err()
    for i in range(4):
        args = [p] * 4
        args[i] = None
        assert lib.fmarl_action_log_probs(acts(), *args, None) == 1 and b'null' in err()
    for i in (0, 1, 4, 5, 7):
        args = [p] * 8
        args[i] = None
        assert lib.fmarl_action_log_probs_backward(acts(), *args, None) == 1 and b'null' in err()
    assert lib.fmarl_action_log_probs(acts(rows=0), p, p, p, p, None) == 0
    assert lib.fmarl_action_log_probs_backward(acts(rows=0), p, p, p, p, p, p, p, p, None) == 1 and b'positive' in err()
    # what is kept stays near 256 MB per part however many rows and actions there are
    big = acts(rows=1 << 24, features=256, actions=15625, x_stride=256, weight_stride=256)
    assert lib.fmarl_action_log_probs_workspace(big, 1) < 4 << 30 and lib.fmarl_action_log_probs_workspace(big, 0) < 1 << 30
