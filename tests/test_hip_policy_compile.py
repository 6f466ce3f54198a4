"""-m gpu: the policy's operators inside a function that torch.compile takes apart: the results and gradients of the same function as it is."""
import pytest
import torch

import fair_marl_amd as fm

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def rn(*shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(sum(shape))).to(DEV)


def chunk(q, v, g, state):
    out, last = fm.memory_chunk(q * 2, q + 1, v, torch.nn.functional.logsigmoid(g), state)
    return out * 2, last + 1


def block(x, branch, w):
    y, h = fm.block_norm(x * 2, branch, pre_weight=w + 1, groups=2)
    return y + 1, h * 2


def actions(x, w):
    lp, ent = fm.action_log_probs(x * 2, w, None, torch.arange(x.shape[0], device=x.device) % w.shape[0])
    return lp * 2, ent + 1


def step(q, v, g, state):
    out, new = fm.memory_step(q * 2, q + 1, v, g, state)
    return out * 2, new + 1


def chunk_backward(q, v, g, state):
    return [t * 2 for t in fm.memory_chunk_backward(q, q + 1, v, g, v * 3, state=state)]


MEMORY = (rn(9, 3, 2, 8), rn(9, 3, 2, 5), rn(2), rn(3, 2, 8, 5)) if torch.cuda.is_available() else ()
CASES = {'chunk': (chunk, lambda: MEMORY), 'block': (block, lambda: (rn(7, 16), rn(7, 16), rn(16))), 'actions': (actions, lambda: (rn(30, 12), rn(70, 12))),
         'step': (step, lambda: (MEMORY[0][0], MEMORY[1][0]) + MEMORY[2:]), 'chunk_backward': (chunk_backward, lambda: MEMORY)}


@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('name', CASES)
def test_a_compiled_caller(name, grad):
    f, args = CASES[name]
    if grad and name in ('step', 'chunk_backward'):
        pytest.skip('records no gradient')
    leaves = [t.clone().requires_grad_(grad) for t in args()]
    torch._dynamo.reset()
    want, got = f(*leaves), torch.compile(f, backend='eager')(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if grad:
        d = [torch.ones_like(t) for t in want]
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, d), torch.autograd.grad(want, leaves, d)))
