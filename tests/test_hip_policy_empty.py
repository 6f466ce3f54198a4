"""-m gpu: the policy's operators on nothing: every input still has a gradient, of zeros."""
import pytest
import torch

import fair_marl_amd as fm

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def z(*shape, dtype=torch.float32):
    return torch.randn(*shape, device=DEV).to(dtype).requires_grad_()


@pytest.mark.parametrize('decay', ['token', 'head'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize('L,B', [(0, 2), (5, 0), (0, 0)])
def test_no_tokens(L, B, dtype, decay):
    q, k, v, S = z(L, B, 3, 4, dtype=dtype), z(L, B, 3, 4, dtype=dtype), z(L, B, 3, 5, dtype=dtype), z(B, 60)
    g = z(*((L, B, 3) if decay == 'token' else (3,)))
    with torch.no_grad():
        g[..., 0] = -float('inf')
    for state in (S, None):
        out, last = fm.memory_chunk(q, k, v, g, state, torch.ones(L, B, device=DEV))
        assert out.shape == v.shape and out.dtype == dtype and last.shape == (B, 3, 4, 5) and last.dtype == torch.float32
        assert torch.equal(last, torch.zeros_like(last) if state is None else S.view_as(last))
        leaves = [q, k, v, g] + ([] if state is None else [S])
        d = torch.randn_like(last)
        got = torch.autograd.grad((out, last), leaves, (torch.ones_like(out), d))
        assert all(a.shape == t.shape and a.dtype == t.dtype for a, t in zip(got, leaves)) and bool((got[3] == 0).all())
        assert state is None or torch.equal(got[4], d.view_as(S))


def test_no_rows():
    x, branch, gate, w = z(0, 3, 16), z(0, 3, 16), z(0, 3, 16), [z(16) for _ in range(5)]
    y, h = fm.block_norm(x, branch, gate, *w, groups=2, kind='layer')
    assert y.shape == h.shape == x.shape
    got = torch.autograd.grad((y, h), [x, branch, gate] + w, (torch.ones_like(y), torch.ones_like(h)))
    assert all(a.shape == t.shape and bool((a == 0).all()) for a, t in zip(got, [x, branch, gate] + w))
    for V in (5, 90):
        X, W, b = z(0, 7), z(V, 7), z(V)
        out = fm.action_log_probs(X, W, b, torch.zeros(0, dtype=torch.int64, device=DEV))
        got = torch.autograd.grad(out, (X, W, b), [torch.ones_like(t) for t in out])
        assert all(a.shape == t.shape and bool((a == 0).all()) for a, t in zip(got, (X, W, b)))
