"""The policy operators under what would lose their derivatives or their work in silence (no GPU): forward-mode tangents and tracers that record tensor
operations are refused by name, by every entry point, before anything else is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

import fair_marl_amd as fm


def z(*shape):
    return torch.zeros(*shape)


CALLS = {
    'memory_chunk': (lambda a, b: fm.memory_chunk(a, b, a, z(1)), (2, 3, 1, 4)),
    'memory_chunk_backward': (lambda a, b: fm.memory_chunk_backward(a, b, a, z(1), a), (2, 3, 1, 4)),
    'memory_step': (lambda a, b: fm.memory_step(a, b, a, z(1), None), (3, 1, 4)),
    'block_norm': (lambda a, b: fm.block_norm(a, b), (3, 4)),
    'action_log_probs': (lambda a, b: fm.action_log_probs(a, b, None, z(3)), (3, 4)),
}


@pytest.mark.parametrize('name', CALLS)
def test_forward_mode_tangents_are_refused(name):
    call, shape = CALLS[name]
    with fwd.dual_level():
        dual = fwd.make_dual(z(*shape), torch.ones(shape))
        for args in ((dual, z(*shape)), (z(*shape), dual)):
            with pytest.raises(ValueError, match='%s: .*forward' % name):
                call(*args)
        with pytest.raises(ValueError, match='GPU'):     # without a tangent it is an ordinary call
            call(z(*shape), z(*shape))


@pytest.mark.parametrize('name', CALLS)
def test_tracers_are_refused(name):
    call, shape = CALLS[name]
    args = z(*shape), z(*shape)
    with pytest.raises(ValueError, match='%s: .*trac' % name):
        torch.jit.trace(call, args)
    with pytest.raises(ValueError, match='%s: .*trac' % name):
        make_fx(call)(*args)
    with pytest.raises(ValueError, match='GPU'):
        call(*args)
