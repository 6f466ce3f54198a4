"""The policy's operators of this framework as they are measured: the memory of a recurrent policy (linear attention with a decay
per head), the norms, gate and residual around a block, and the log-probability / entropy of actions, each in its plain form
(elementary torch operations in 32 bits) and as the framework's own calls.  Sizes: 4 096 x 3 and 65 536 x 10 are the rollouts that
bench.py runs, 25 steps their episodes, 10 the chunk length of the recurrent minibatches, 64 the default hidden size (4 heads of 16),
5 the actions of an agent and 5 ** N the joint actions of N agents."""
import math

import torch

own = False
DEV = 'cuda:0'
DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


# ---- cases ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one env step of a small rollout (128 envs x 3 agents): the recurrent state moves one token on, in the buffer's slots
        dict(name='memory step 128x3', op='memory', what='step', L=1, B=384, H=4, dk=16, dv=16, dtype='f32', decay='token', fused=False),
        # one env step of the 65 536 x 10 rollout: 2.7 GB of state read and written
        dict(name='memory step 65536x10', op='memory', what='step', L=1, B=655360, H=4, dk=16, dv=16, dtype='f32', decay='head', fused=False),
        # the update's recurrent minibatch: all chunks of ten steps of 4 096 x 3 agents over an episode, episode ends inside
        dict(name='memory train chunks of 10', op='memory', what='train', L=10, B=30720, H=4, dk=16, dv=16, dtype='f32', decay='token', fused=False),
        # whole histories in half precision, few of them: q, k, v are views of one projection
        dict(name='memory train 4096 bf16', op='memory', what='train', L=4096, B=8, H=8, dk=64, dv=64, dtype='bf16', decay='token', fused=True),
        # evaluation of ragged histories with head sizes that fill no tile
        dict(name='memory forward 1023 ragged', op='memory', what='forward', L=1023, B=24, H=3, dk=40, dv=72, dtype='f16', decay='head', fused=True),
        # one env step of a small rollout through the block's end
        dict(name='block 384x64 forward', op='block', what='forward', M=384, D=64, groups=4, dtype='f32', kind='rms', act='silu', bias=False),
        # a feed-forward minibatch of 655 360 rows at the default hidden size
        dict(name='block 655360x64 train', op='block', what='train', M=655360, D=64, groups=4, dtype='f32', kind='layer', act='sigmoid', bias=True),
        # wide rows in half precision
        dict(name='block 16383x1000 train', op='block', what='train', M=16383, D=1000, groups=8, dtype='bf16', kind='rms', act='silu', bias=False),
        # the log-probabilities of one env step's actions
        dict(name='actions 384x5 forward', op='actions', what='forward', M=384, K=64, V=5, dtype='f32', avail=True, pad=0.0),
        # the update of 65 536 x 32 agents, one env step a minibatch
        dict(name='actions 2097152x5 train', op='actions', what='train', M=2097152, K=64, V=5, dtype='f32', avail=True, pad=0.05),
        # a centralised policy over the joint actions of four agents, ragged features, unavailable ones
        dict(name='actions 12345x625 train', op='actions', what='train', M=12345, K=100, V=625, dtype='f32', avail=True, pad=0.05),
        # the same over the joint actions of six agents
        dict(name='actions 8192x15625 train', op='actions', what='train', M=8192, K=256, V=15625, dtype='bf16', avail=False, pad=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['memory', 'memory', 'block', 'actions'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'memory':
        what = rng.choice(['step', 'forward', 'train', 'train'])
        L = 1 if what == 'step' else _log(rng, 1, 4096)
        H, dk, dv = rng.randint(1, 8), _log(rng, 4, 128), _log(rng, 4, 128)
        most = min(4e7 / (L * H * (dk + dv)), 1.2e8 / (H * dk * dv), 4e8 / (L * H * dk * dv) if L > 64 else 1e9)
        B = _log(rng, 1, max(2, int(most)))
        return dict(op=op, what=what, L=L, B=B, H=H, dk=dk, dv=dv, dtype=dtype, decay=rng.choice(['head', 'token']), fused=rng.random() < 0.5)
    if op == 'block':
        groups = rng.choice([1, 1, 2, 4, 8])
        D = groups * _log(rng, max(1, 8 // groups), 4096 // groups)
        M = _log(rng, 1, max(2, 40000000 // D))
        return dict(op=op, what=rng.choice(['forward', 'train']), M=M, D=D, groups=groups, dtype=dtype, kind=rng.choice(['rms', 'layer']),
                    act=rng.choice(['sigmoid', 'silu']), bias=rng.random() < 0.5)
    V, K = _log(rng, 2, 15625), _log(rng, 8, 512)
    M = _log(rng, 1, max(2, min(1000000, int(3.2e10 / (V * K)), 10 ** 8 // V, 10 ** 8 // K)))
    return dict(op=op, what=rng.choice(['forward', 'train']), M=M, K=K, V=V, dtype=dtype, avail=rng.random() < 0.5, pad=rng.choice([0.0, 0.05]))


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed * 1000003 + 17)
    dt = DTYPES[case['dtype']]

    def randn(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, device=DEV, generator=gen) * std).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, device=DEV, generator=gen)

    s = dict(case=case)
    train = case['what'] == 'train'
    if case['op'] == 'memory':
        L, B, H, dk, dv = (case[k] for k in ('L', 'B', 'H', 'dk', 'dv'))
        if case['fused']:   # one projection's output; q, k and v are views of it
            qkv = randn(L, B, H * (2 * dk + dv), dtype=dt)
            q, k, v = (t.unflatten(-1, (H, -1)) for t in qkv.split([H * dk, H * dk, H * dv], -1))
        else:
            q, k, v = randn(L, B, H, dk, dtype=dt), randn(L, B, H, dk, dtype=dt), randn(L, B, H, dv, dtype=dt)
        # decays as a gate gives them: most close to one, some forget within a few tokens
        s['log_decay'] = torch.nn.functional.logsigmoid(randn(*((L, B, H) if case['decay'] == 'token' else (H,))) * 2 + 3)
        s['masks'] = (rand(L, B) > 1 / 25).float()   # an episode starts where it is 0
        s['state'] = randn(B, H, dk, dv)
        s['scale'] = dk ** -0.5
        if case['what'] == 'step':
            q, k, v, s['masks'] = q[0], k[0], v[0], s['masks'][0]
            s['log_decay'] = s['log_decay'][0] if case['decay'] == 'token' else s['log_decay']
            s['out_state'] = torch.empty(B, H, dk, dv, device=DEV)   # the buffer's next slot
        if train:
            s['d_out'], s['d_state'] = randn(L, B, H, dv, dtype=dt), randn(B, H, dk, dv)
        s.update(q=q, k=k, v=v)
        leaves = ('q', 'k', 'v', 'log_decay', 'state')
    elif case['op'] == 'block':
        M, D = case['M'], case['D']
        s['x'], s['branch'], s['gate'] = randn(M, D, dtype=dt), randn(M, D, dtype=dt), randn(M, D, dtype=dt)
        s['scale'] = randn(D, std=0.1) + 0.5
        s['post_weight'], s['pre_weight'] = randn(D, std=0.1) + 1, randn(D, std=0.1) + 1
        s['post_bias'], s['pre_bias'] = (randn(D, std=0.1), randn(D, std=0.1)) if case['bias'] else (None, None)
        if train:
            s['d_y'], s['d_h'] = randn(M, D, dtype=dt), randn(M, D, dtype=dt)
        leaves = ('x', 'branch', 'gate', 'scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')
    else:
        M, K, V = case['M'], case['K'], case['V']
        s['features'], s['weight'], s['bias'] = randn(M, K, dtype=dt), randn(V, K, dtype=dt, std=2 * K ** -0.5), randn(V, dtype=dt, std=0.5)
        s['actions'] = torch.randint(0, V, (M,), device=DEV, generator=gen)
        s['available'] = None
        if case['avail']:
            s['available'] = (rand(M, V) > 0.3).float()
            s['available'].scatter_(1, s['actions'][:, None], 1.0)   # the taken action was available
        if case['pad']:
            s['actions'] = torch.where(rand(M) < case['pad'], -1, s['actions'])   # padded rows
        if train:
            s['d_log_prob'], s['d_entropy'] = randn(M, std=1 / M), randn(M, std=0.01 / M)
        leaves = ('features', 'weight', 'bias')
    if train:
        for name in leaves:
            if s[name] is not None:
                s[name] = s[name].requires_grad_() if s[name].is_leaf and s[name]._base is None else s[name].detach().requires_grad_()
    s['leaves'] = [name for name in leaves if s[name] is not None]
    return s


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end ---------------------------------------------
def _plain_memory(q, k, v, g, state, masks, scale):
    L, B, H = q.shape[:3]
    q, k, v, g = q.float(), k.float(), v.float(), g.float().expand(L, B, H)
    outs, S = [], state.float()
    for a in range(0, L, 64):
        qc, kc, vc = (t[a:a + 64].permute(1, 2, 0, 3) for t in (q, k, v))        # (B, H, l, d)
        gc, fresh = g[a:a + 64].permute(1, 2, 0), (masks[a:a + 64] == 0).t()[:, None]
        fresh = fresh | (gc == -math.inf)
        cum, seg = torch.cumsum(gc.masked_fill(fresh, 0.0).double(), -1), torch.cumsum(fresh.long(), -1)
        diff, same = cum[..., :, None] - cum[..., None, :], seg[..., :, None] == seg[..., None, :]
        w = torch.exp(diff.masked_fill(~(same & torch.ones_like(same).tril()), -math.inf)).float()
        carry = torch.exp(cum.masked_fill(seg > 0, -math.inf)).float()
        p = torch.matmul(qc, kc.transpose(-1, -2)) * w
        outs.append((torch.matmul(p, vc) + carry[..., None] * torch.matmul(qc, S)).permute(2, 0, 1, 3) * scale)
        S = carry[..., -1, None, None] * S + torch.matmul((kc * w[..., -1, :, None]).transpose(-1, -2), vc)
    return torch.cat(outs), S


def _plain_norm(a, kind, eps):
    if kind == 'layer':
        a = a - a.mean(-1, keepdim=True)
    return a * torch.rsqrt((a * a).mean(-1, keepdim=True) + eps)


def _plain_block(x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, groups, kind, act, eps=1e-5):
    M, D = x.shape
    u = _plain_norm(branch.float().view(M, groups, -1), kind, eps).view(M, D) * post_weight
    u = u if post_bias is None else u + post_bias
    s = torch.sigmoid(gate.float())
    y = x.float() + scale * (u * (s * gate.float() if act == 'silu' else s))
    h = _plain_norm(y, kind, eps) * pre_weight
    return y, h if pre_bias is None else h + pre_bias


def _plain_actions(features, weight, bias, actions, available):
    z = torch.matmul(features.float(), weight.float().t()) + bias.float()
    if available is not None:
        z = z.masked_fill(available == 0, -math.inf)
    part = (actions >= 0) & (z.amax(-1) > -math.inf)
    z = z.masked_fill(~part[:, None], 0.0)
    top = z.detach().amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1)
    lse = torch.log(total) + top[:, 0]
    log_prob = z.gather(1, actions.clamp(min=0)[:, None])[:, 0] - lse
    entropy = lse - (e / total[:, None] * z.masked_fill(z == -math.inf, 0.0)).sum(-1)
    return log_prob.masked_fill(~part, 0.0), entropy.masked_fill(~part, 0.0)


def _outputs(s):
    case = s['case']
    if case['op'] == 'memory':
        if own:
            import fair_marl_amd as fm
            if case['what'] == 'step':
                return fm.memory_step(s['q'], s['k'], s['v'], s['log_decay'], s['state'], s['masks'], s['scale'], out_state=s['out_state'])
            return fm.memory_chunk(s['q'], s['k'], s['v'], s['log_decay'], s['state'], s['masks'], s['scale'])
        if case['what'] == 'step':
            a = torch.where(s['masks'][:, None] == 0, 0.0, torch.exp(s['log_decay']))[..., None, None]
            q, k, v = (s[n].float() for n in 'qkv')
            S = a * s['state'] + k[..., None] * v[..., None, :]
            return ((q[..., None] * S).sum(-2) * s['scale']).to(s['v'].dtype), S
        out, S = _plain_memory(s['q'], s['k'], s['v'], s['log_decay'], s['state'], s['masks'], s['scale'])
        return out.to(s['v'].dtype), S
    if case['op'] == 'block':
        args = [s[n] for n in ('x', 'branch', 'gate', 'scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')]
        if own:
            import fair_marl_amd as fm
            return fm.block_norm(*args, groups=case['groups'], kind=case['kind'], gate_act=case['act'])
        y, h = _plain_block(*args, case['groups'], case['kind'], case['act'])
        return y.to(s['x'].dtype), h.to(s['x'].dtype)
    if own:
        import fair_marl_amd as fm
        return fm.action_log_probs(s['features'], s['weight'], s['bias'], s['actions'], s['available'])
    return _plain_actions(s['features'], s['weight'], s['bias'], s['actions'], s['available'])


def _upstream(s):
    return {'memory': ('d_out', 'd_state'), 'block': ('d_y', 'd_h'), 'actions': ('d_log_prob', 'd_entropy')}[s['case']['op']]


def run(s):
    if s['case']['what'] != 'train':
        with torch.no_grad():
            return list(_outputs(s))
    out = _outputs(s)
    grads = torch.autograd.grad(out, [s[n] for n in s['leaves']], [s[n] for n in _upstream(s)])
    return [t.detach() for t in out] + list(grads)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    e, train = (4 if case['dtype'] == 'f32' else 2), case['what'] == 'train'
    if case['op'] == 'memory':
        L, B, H, dk, dv = (case[k] for k in ('L', 'B', 'H', 'dk', 'dv'))
        decays = 4 * (L * B * H if case['decay'] == 'token' else H)
        rows, state = L * B * H * e, 4 * B * H * dk * dv
        b = rows * (2 * dk + 2 * dv) + 2 * state + decays + 4 * L * B
        f = 4 * L * B * H * dk * dv
        if train:
            b += rows * (2 * dk + 2 * dv) + 2 * state + decays    # d_out, d_state in; dq, dk, dv, d_decay, d(initial state) out
            f += 10 * L * B * H * dk * dv
        return dict(bytes=b, flops=f)
    if case['op'] == 'block':
        n, w = case['M'] * case['D'], 4 * case['D'] * (5 if case['bias'] else 3)
        return dict(bytes=(10 if train else 5) * n * e + (2 if train else 1) * w, flops=(60 if train else 20) * n)
    M, K, V = case['M'], case['K'], case['V']
    b = e * (M * K + V * K + V) + 8 * M + 8 * M + (4 * M * V if case['avail'] else 0)
    if train:
        b += e * (M * K + V * K + V) + 8 * M
    return dict(bytes=b, flops=(6 if train else 2) * M * V * K)


# ---- the definitions in 64 bits: the recurrence token by token, gradients from their formulas --------------------------------
def _exact_memory(s):
    case, scale = s['case'], s['scale']
    L, B, H, dk, dv = (case[k] for k in ('L', 'B', 'H', 'dk', 'dv'))
    step, train = case['what'] == 'step', case['what'] == 'train'
    if L * B * H * dk * dv * 8 > 6e10 and train:
        return None
    lead = (lambda t: t[None]) if step else (lambda t: t)
    q, k, v, masks = (lead(s[n].detach()) for n in ('q', 'k', 'v', 'masks'))
    g = s['log_decay'].detach().double().expand(L, B, H)
    S, states, outs = s['state'].detach().double(), [], []

    def decay(t):
        return (torch.exp(g[t]) * (masks[t] != 0)[:, None])[..., None, None]

    for t in range(L):
        if train:
            states.append(S)
        S = S * decay(t) + k[t].double().unsqueeze(-1) * v[t].double().unsqueeze(-2)
        outs.append((q[t].double().unsqueeze(-1) * S).sum(-2) * scale)
    res = [outs[0] if step else torch.stack(outs), S]
    if train:
        G = s['d_state'].double()
        dq, dk_, dv_, dg = [None] * L, [None] * L, [None] * L, [None] * L
        for t in range(L - 1, -1, -1):
            do, kt, vt = s['d_out'][t].double(), k[t].double(), v[t].double()
            now = states[t] * decay(t) + kt.unsqueeze(-1) * vt.unsqueeze(-2)
            dq[t] = (now * do.unsqueeze(-2)).sum(-1) * scale
            G = G + scale * q[t].double().unsqueeze(-1) * do.unsqueeze(-2)
            dk_[t], dv_[t] = (G * vt.unsqueeze(-2)).sum(-1), (G * kt.unsqueeze(-1)).sum(-2)
            G = G * decay(t)
            dg[t] = (G * states[t]).sum((-1, -2))
            states[t] = None
        dg = torch.stack(dg)
        res += [torch.stack(dq), torch.stack(dk_), torch.stack(dv_), dg if case['decay'] == 'token' else dg.sum((0, 1)), G]
    return res


def _exact_norm(a, kind, eps=1e-5):
    c = a - a.mean(-1, keepdim=True) if kind == 'layer' else a
    inv = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    n = c * inv

    def back(d):
        d = d - n * (d * n).mean(-1, keepdim=True)
        return inv * (d - d.mean(-1, keepdim=True) if kind == 'layer' else d)
    return n, back


def _exact_block(s):
    case = s['case']
    G, kind = case['groups'], case['kind']
    M, D = case['M'], case['D']
    wide = {n: (s[n].detach().double() if s[n] is not None else None) for n in ('scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')}
    parts, sums = [], {}
    rows = max(1, 2 ** 24 // D)
    for a in range(0, M, rows):
        x, o, gate = (s[n].detach()[a:a + rows].double() for n in ('x', 'branch', 'gate'))
        m = x.shape[0]
        n1, back1 = _exact_norm(o.view(m, G, -1), kind)
        n1 = n1.reshape(m, D)
        u = n1 * wide['post_weight'] + (wide['post_bias'] if case['bias'] else 0.0)
        sg = 1 / (1 + torch.exp(-gate))
        act, slope = (gate * sg, sg + gate * sg * (1 - sg)) if case['act'] == 'silu' else (sg, sg * (1 - sg))
        y = x + wide['scale'] * u * act
        n2, back2 = _exact_norm(y, kind)
        h = n2 * wide['pre_weight'] + (wide['pre_bias'] if case['bias'] else 0.0)
        part = [y, h]
        if case['what'] == 'train':
            dh = s['d_h'][a:a + rows].double()
            dy = s['d_y'][a:a + rows].double() + back2(dh * wide['pre_weight'])
            dr = dy * wide['scale']
            du = dr * act
            part += [dy, back1((du * wide['post_weight']).view(m, G, -1)).reshape(m, D), dr * u * slope]
            for name, t in (('scale', dy * u * act), ('post_weight', du * n1), ('post_bias', du), ('pre_weight', dh * n2), ('pre_bias', dh)):
                sums[name] = sums.get(name, 0) + t.sum(0)
        parts.append(part)
    res = [torch.cat(c) for c in zip(*parts)]
    return res + [sums[n] for n in s['leaves'] if n in sums] if sums else res


def _exact_actions(s):
    case = s['case']
    M, V, train = case['M'], case['V'], case['what'] == 'train'
    W, b = s['weight'].detach().double(), s['bias'].detach().double()
    logp, ent, dX, dW, db = [], [], [], torch.zeros_like(W), torch.zeros_like(b)
    rows = max(1, 2 ** 26 // max(V, case['K']))
    for a in range(0, M, rows):
        X, act = s['features'].detach()[a:a + rows].double(), s['actions'][a:a + rows]
        z = X @ W.t() + b
        if s['available'] is not None:
            z[s['available'][a:a + rows] == 0] = -math.inf
        part = (act >= 0) & (z > -math.inf).any(-1)
        logs = z - torch.logsumexp(z, -1, keepdim=True)
        p = torch.exp(logs)
        plogs = torch.where(p > 0, p * logs, torch.zeros_like(p))
        hot = torch.zeros_like(p).scatter_(1, act.clamp(min=0)[:, None], 1.0)
        H = -plogs.sum(-1)
        logp.append(torch.where(part, logs.gather(1, act.clamp(min=0)[:, None])[:, 0], 0.0))
        ent.append(torch.where(part, H, 0.0))
        if train:
            dl, de = s['d_log_prob'][a:a + rows, None].double(), s['d_entropy'][a:a + rows, None].double()
            dz = torch.where(part[:, None], dl * (hot - p) - de * (plogs + p * H[:, None]), 0.0)
            dX.append(dz @ W)
            dW += dz.t() @ X
            db += dz.sum(0)
    res = [torch.cat(logp), torch.cat(ent)]
    return res + [torch.cat(dX), dW, db] if train else res


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'memory': _exact_memory, 'block': _exact_block, 'actions': _exact_actions}[case['op']](s)
