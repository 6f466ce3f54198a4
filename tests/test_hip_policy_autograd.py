"""-m gpu: the policy's operators and autograd's bookkeeping -- tensors written in place, tensors kept for the backward pass."""
import pytest
import torch
import torch.utils.checkpoint

import fair_marl_amd as fm
from fair_marl_amd.rollout_buffer import DeviceRolloutBuffer

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def inputs(L, B, H, dk, dv, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV)  # noqa: E731
    return rn(L, B, H, dk), rn(L, B, H, dk), rn(L, B, H, dv), torch.nn.functional.logsigmoid(rn(L, B, H)), rn(B, H, dk, dv)


def test_a_state_stepped_in_place_is_seen():
    """a state that a chunk keeps for its gradient and a step overwrites: an error, as with any operation in place"""
    q, k, v, g, S = inputs(5, 3, 2, 8, 8)
    version = S._version
    out, _ = fm.memory_chunk(q.requires_grad_(), k, v, g, S)
    with torch.no_grad():
        fm.memory_step(q[0], k[0], v[0], g[0], S, out_state=S)
    assert S._version > version
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()
    other = torch.empty_like(S)
    version = S._version, other._version
    with torch.no_grad():
        fm.memory_step(q[0], k[0], v[0], g[0], S, out_state=other)
    assert S._version == version[0] and other._version > version[1]
    with torch.inference_mode():     # tensors without a version
        mine = S.clone()
        fm.memory_step(q[0], k[0], v[0], g[0], mine, out_state=mine)
    assert torch.equal(mine, other)


def test_a_buffer_slot_stepped_in_place_is_seen():
    eng = fm.RolloutEngine(fm.EnvConfig(num_agents=3, num_landmarks=3, num_obstacles=2, episode_length=4), 5, device=DEV)
    buf = DeviceRolloutBuffer(eng).attach_policy(recurrent_N=2, hidden_size=32)
    q, k, v, g, _ = inputs(1, 15, 2, 4, 8)
    out, _ = fm.memory_chunk(q.requires_grad_(), k, v, g, buf.rnn_states[1])
    with torch.no_grad():
        buf.memory_step(0, q.view(5, 3, 2, 4), k.view(5, 3, 2, 4), v.view(5, 3, 2, 8), g.view(5, 3, 2))
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()


@pytest.mark.parametrize('shape', [(2048, 1, 2, 64, 64), (2048, 2, 4, 16, 16)], ids=str)
def test_segment_states_go_with_the_saved_tensors(shape):
    """long sequences: the states at their segments' starts (here as many bytes as the rows, or more) are moved, dropped and freed as every saved tensor is"""
    q, k, v, g, S = inputs(*shape, seed=1)
    leaves = [t.requires_grad_() for t in (q, k, v, g, S)]
    run = lambda: fm.memory_chunk(*leaves)  # noqa: E731
    with torch.no_grad():
        d = [torch.randn_like(t) for t in run()]
    want = torch.autograd.grad(run(), leaves, d)
    own = sum(t.numel() * 4 for t in d)
    asked = lambda: torch.cuda.memory_stats()['requested_bytes.all.current']  # noqa: E731

    def left(f):
        before = asked()
        out = f()
        return out, asked() - before

    with torch.autograd.graph.save_on_cpu():
        offloaded, kept = left(run)
    assert kept <= own, (kept, own)
    again, kept = left(lambda: torch.utils.checkpoint.checkpoint(run, use_reentrant=False))
    assert kept <= own, (kept, own)
    for out in (offloaded, again):
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, d), want))
    out, kept = left(run)
    assert kept > own                                      # an ordinary pass keeps them,
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, d, retain_graph=True), want))
    got, freed = left(lambda: torch.autograd.grad(out, leaves, d))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = sum(t.numel() * 4 for t in leaves)
    assert freed <= grads - (kept - own), (freed, grads, kept, own)   # and gives them back with the graph, while its outputs live
