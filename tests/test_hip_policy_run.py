"""-m gpu: the policy's operators as they are used together -- a rollout whose policy keeps its memory in the buffer's recurrent states and takes its
log-probabilities from its features, then the update's recurrent minibatches over the same buffer -- against the same policy in plain float64 torch."""
import pytest
import torch
import torch.utils.checkpoint

import fair_marl_amd as fm
from fair_marl_amd.rollout_buffer import DeviceRolloutBuffer

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
H, DK, DV, D, V = 2, 8, 8, 16, 5


def parameters(obs_dim, seed):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: (torch.randn(*s, generator=gen) * s[-1] ** -0.5).to(DEV)  # noqa: E731
    return dict(inp=rn(D, obs_dim), proj=rn(H * (2 * DK + DV) + D + H, D), pre1=1 + rn(D), post=1 + rn(D), scale=rn(D) + 0.5, pre2=1 + rn(D), head=rn(V, D), bias=rn(V))


def parts(p, h):
    """q, k, v, gate, log decay of rows h (..., D)"""
    z = h @ p['proj'].t()
    q, k, v, gate, g = z.split([H * DK, H * DK, H * DV, D, H], -1)
    return q.unflatten(-1, (H, DK)), k.unflatten(-1, (H, DK)), v.unflatten(-1, (H, DV)), gate, torch.nn.functional.logsigmoid(g + 2)


def policy(p, obs, memory):
    """features of rows; memory(q, k, v, log_decay) -> (..., H, DV)"""
    x = obs @ p['inp'].t()
    _, h = fm.block_norm(x, pre_weight=p['pre1'])
    q, k, v, gate, g = parts(p, h)
    o = memory(q, k, v, g)
    return fm.block_norm(x, o.flatten(-2), gate, p['scale'], p['post'], None, p['pre2'], groups=H, gate_act='silu')[1]


def rms(a):
    return a / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-5)


def plain(p, obs, state, masks):
    """the same features in plain torch, (L, B, ..)"""
    x = obs @ p['inp'].t()
    q, k, v, gate, g = parts(p, rms(x) * p['pre1'])
    outs, S = [], state.view(-1, H, DK, DV)
    for t in range(obs.shape[0]):
        S = (torch.exp(g[t]) * masks[t])[..., None, None] * S + k[t][..., None] * v[t][..., None, :]
        outs.append((q[t][..., None] * S).sum(-2) * DK ** -0.5)
    u = rms(torch.stack(outs)).flatten(-2) * p['post']
    return rms(x + p['scale'] * u * gate * torch.sigmoid(gate)) * p['pre2']


def reproduced(p, obs, state, masks):
    """How far the log-probabilities of two float32 runs of the policy on the same rows may lie apart, per row (L, B), by arithmetic in units u = 2^-24.
    Magnitudes: X of x's terms, Hm of h's (the norm's gain times X on top), Q, K, W of q, k, v, Gm of the log decays, A of the memory's output: the recurrence run on
    them.  q, k, v and the decays carry at most 4 (D + obs + 80) u of their magnitudes, the recurrence 2 L + dk + dv + 200 more (+ L times the decays'), so out is off by
    gamma A.  A norm's derivative is its gain (1 / rms) times a projection: the error behind it is at most gain * 2-norm of the error before it."""
    u, L = 2.0 ** -24, obs.shape[0]
    X = obs.abs() @ p['inp'].abs().t()
    x = obs @ p['inp'].t()
    gain = lambda a: 1 / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-5)  # noqa: E731
    h = x * gain(x) * p['pre1']
    Hm = h.abs() + gain(x) * X.norm(dim=-1, keepdim=True) * p['pre1'].abs()
    Z = Hm @ p['proj'].abs().t()
    Q, K, W, Gate, Gm = Z.split([H * DK, H * DK, H * DV, D, H], -1)
    Q, K, W = Q.unflatten(-1, (H, DK)), K.unflatten(-1, (H, DK)), W.unflatten(-1, (H, DV))
    q, k, v, gate, g = parts(p, h)
    A, o, S, M = [], [], state.view(-1, H, DK, DV), state.abs().view(-1, H, DK, DV)
    for t in range(L):
        a = (torch.exp(g[t]) * masks[t])[..., None, None]
        S, M = a * S + k[t][..., None] * v[t][..., None, :], a * M + K[t][..., None] * W[t][..., None, :]
        o.append((q[t][..., None] * S).sum(-2) * DK ** -0.5)
        A.append((Q[t][..., None] * M).sum(-2) * DK ** -0.5)
    o, A = torch.stack(o), torch.stack(A)
    base = 4 * (D + obs.shape[-1] + 80)
    gamma = u * (2 * L + DK + DV + 200 + base + L * base * float(Gm.max()))
    un = o * gain(o)
    du = (gain(o) * gamma * A.norm(dim=-1, keepdim=True)).expand_as(o).flatten(-2) * p['post'].abs() + 60 * u * un.flatten(-2).abs() * p['post'].abs()
    act = gate * torch.sigmoid(gate)
    y = x + p['scale'] * un.flatten(-2) * p['post'] * act
    dy = base * u * X + p['scale'].abs() * (du * act.abs() + (un.flatten(-2) * p['post']).abs() * 1.1 * base * u * Gate)
    f = y * gain(y) * p['pre2']
    df = gain(y) * dy.norm(dim=-1, keepdim=True) * p['pre2'].abs() + 60 * u * f.abs()
    return 4 * ((df @ p['head'].abs().t()).amax(-1) + (D + 60) * u * (f.abs() @ p['head'].abs().t() + p['bias'].abs()).amax(-1))   # two runs, 2 max |dz| each


def test_rollout_and_update_with_the_policy_operators():
    n, N, T, L = 24, 3, 20, 5
    eng = fm.RolloutEngine(fm.EnvConfig(num_agents=N, num_landmarks=N, num_obstacles=2, episode_length=8), n, device=DEV, seed=3)
    buf = DeviceRolloutBuffer(eng, episode_length=T).attach_policy(recurrent_N=H, hidden_size=DK * DV, n_actions=V)
    p = parameters(eng.cfg.obs_dim, 1)
    gen = torch.Generator(device=DEV).manual_seed(2)
    buf.available_actions[:, :, 1, 3] = 0
    buf.reset()
    with torch.no_grad():
        for t in range(T):
            feats = policy(p, buf.obs[t], lambda q, k, v, g: buf.memory_step(t, q, k, v, g))
            actions = torch.randint(0, 3, (n, N), device=DEV, generator=gen, dtype=torch.int32)
            logp, ent = buf.insert_actions(t, feats, p['head'], p['bias'], actions)
            assert logp.shape == (n, N, 1) and torch.equal(buf.action_log_probs[t], logp) and torch.equal(buf.actions[t, ..., 0], actions.float())
            buf.insert_step(actions)
    assert float(buf.masks[1:].min()) == 0.0      # episodes ended inside
    buf.value_preds.normal_(generator=gen)
    buf.compute_returns(torch.zeros(n, N, 1, device=DEV))
    adv = buf.advantages()
    leaves = [a.requires_grad_() for a in p.values()]
    wide = {k: a.detach().double().requires_grad_() for k, a in p.items()}
    count = 0
    for sample in buf.recurrent_generator(adv, 2, L):
        s = dict(zip(DeviceRolloutBuffer.GENERATOR_FIELDS, sample))
        B = s['rnn_states'].shape[0]
        feats = policy(p, s['obs'].view(L, B, -1), lambda q, k, v, g: fm.memory_chunk(q, k, v, g, s['rnn_states'], s['masks'])[0])
        logp, ent = fm.action_log_probs(feats, p['head'], p['bias'], s['actions'], s['available_actions'])
        # the policy is the one that acted: the chunks reproduce what the steps stored
        with torch.no_grad():
            apart = (logp.view(-1, 1) - s['old_action_log_probs']).abs().view(L, B).double()
            bound = reproduced({k: a.detach() for k, a in wide.items()}, s['obs'].double().view(L, B, -1), s['rnn_states'].double(), s['masks'].double().view(L, B, 1))
            assert bool((apart <= bound).all()) and float(apart.median()) < 1e-6, float((apart - bound).max())
        ratio = torch.exp(logp.view(-1, 1) - s['old_action_log_probs'])
        loss = (-ratio * s['adv_targ'] * s['active_masks']).mean() - 0.01 * ent.mean()
        got = torch.autograd.grad(loss, leaves)
        d = lambda a: a.double()  # noqa: E731
        wf = plain(wide, d(s['obs']).view(L, B, -1), d(s['rnn_states']), d(s['masks']).view(L, B, 1))
        z = (wf @ wide['head'].t() + wide['bias']).view(-1, V).masked_fill(s['available_actions'] == 0, float('-inf'))
        logs = torch.log_softmax(z, -1)
        wl = logs.gather(1, s['actions'].long())
        went = -(logs.exp() * logs.masked_fill(z == float('-inf'), 0.0)).sum(-1)
        wloss = (-torch.exp(wl - d(s['old_action_log_probs'])) * d(s['adv_targ']) * d(s['active_masks'])).mean() - 0.01 * went.mean()
        want = torch.autograd.grad(wloss, list(wide.values()))
        for name, a, b in zip(p, got, want):
            # float32 against float64 through some ten operators: a few hundred roundings of 2^-24 of the largest entry
            assert float((a.double() - b).abs().max()) <= 1e-4 * float(b.abs().max()) + 1e-7, name
        count += 1
    assert count == 2


def test_buffer_entry_points_refuse():
    eng = fm.RolloutEngine(fm.EnvConfig(num_agents=3, num_landmarks=3, num_obstacles=2, episode_length=4), 5, device=DEV)
    buf = DeviceRolloutBuffer(eng)
    z = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    q, v, g = z(5, 3, 2, 4), z(5, 3, 2, 8), z(2)
    with pytest.raises(RuntimeError, match='attach_policy'):
        buf.memory_step(0, q, q, v, g)
    buf.attach_policy(recurrent_N=2, hidden_size=32)
    assert buf.memory_step(3, q, q, v, g).shape == (5, 3, 2, 8)
    assert buf.memory_step(0, q, q, v, z(5, 3, 2), critic=True).shape == (5, 3, 2, 8)
    for t, a, b in ((4, q, v), (-1, q, v), (0, q, z(5, 3, 2, 4)), (0, z(15, 2, 4), v), (0, z(3, 5, 2, 4), z(3, 5, 2, 8))):
        with pytest.raises(ValueError, match='memory_step'):
            buf.memory_step(t, a, a, b, g)
    with pytest.raises(ValueError, match='insert_actions'):
        buf.insert_actions(4, z(5, 3, 7), z(5, 7), None, z(5, 3))
    lp, en = buf.insert_actions(0, z(5, 3, 7), z(5, 7), None, z(5, 3))
    assert float((en - 5 ** 0 * torch.log(torch.tensor(5.0))).abs().max().cpu()) < 1e-6


def test_saved_tensors_elsewhere_and_second_gradients():
    """what the backward pass needs may be formed again (checkpointing) or come back from the host at another address: the same gradients; a gradient of a gradient is refused"""
    gen = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV).requires_grad_()  # noqa: E731
    big = rn(12, 6, 2, 21)                      # rows with odd strides inside
    x, branch, w, head, bias = rn(72, 20), rn(72, 20), rn(20), rn(V, 20), rn(V)
    q, k, v, g, S = big[..., :8], big[..., 8:16], big[..., 16:], rn(12, 6, 2), rn(6, 2, 8, 5)
    act = torch.randint(0, V, (72,), generator=gen).to(DEV)
    leaves = (big, g, S, x, branch, w, head, bias)

    def loss():
        o, last = fm.memory_chunk(q, k, v, torch.nn.functional.logsigmoid(g), S)
        y, h = fm.block_norm(x, branch, None, w, None, None, w, groups=2, kind='layer')
        lp, ent = fm.action_log_probs(h, head, bias, act)
        return o.square().sum() + last.sum() + y.sum() + (lp * ent).sum()

    want = torch.autograd.grad(loss(), leaves)
    with torch.autograd.graph.save_on_cpu():
        offloaded = loss()
    again = torch.utils.checkpoint.checkpoint(loss, use_reentrant=False)
    for got in (torch.autograd.grad(offloaded, leaves), torch.autograd.grad(again, leaves)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for leaf in (S, x, head):
        first, = torch.autograd.grad(loss(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            first.sum().backward()
