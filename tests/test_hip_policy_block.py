"""-m gpu: block_norm (norm of the branch, gate, residual scale, residual, norm in one pass) against its formulas in float64, and its gradients.

Tolerances: a norm's statistic is a sum of at most D squares (D + 8 roundings of 2^-24), the element formulas add some twenty roundings and two
approximate functions of a few ulp: every output is within c = (2 D / 8 + 60) 2^-24 of the float64 result, relative to the magnitudes of the terms that
its last sums add up (the sums over a row are formed by at most D / 16 + 20 additions per path); the gradients of the weights add the M rows' terms
in at most M / 16 + 40 float32 additions per path and the rest in float64.  Half a step of the output's type comes on top."""
import itertools

import pytest
import torch

import fair_marl_amd as fm

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ('x', 'branch', 'gate', 'scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')


def formula(t, groups, kind, act, post, pre, eps=1e-5):
    """differentiable in float64: the definition itself"""
    x, branch, gate, scale, pw, pb, rw, rb = t

    def norm(a):
        a = a - a.mean(-1, keepdim=True) if kind == 'layer' else a
        return a / torch.sqrt((a * a).mean(-1, keepdim=True) + eps)
    y = x
    if branch is not None:
        u = norm(branch.unflatten(-1, (groups, -1))).flatten(-2) if post else branch
        u = u if pw is None else u * pw
        u = u if pb is None else u + pb
        if gate is not None:
            u = u * (gate * torch.sigmoid(gate) if act == 'silu' else torch.sigmoid(gate))
        y = x + (u if scale is None else scale * u)
    h = None
    if pre:
        h = norm(y)
        h = h if rw is None else h * rw
        h = h if rb is None else h + rb
    return y, h


def make(M, D, x_dtype, dtype, seed, without=()):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = dict(x=rn(M, D).to(x_dtype), branch=(2 * rn(M, D)).to(dtype), gate=(2 * rn(M, D)).to(dtype), scale=rn(D), post_weight=1 + 0.3 * rn(D), post_bias=rn(D),
             pre_weight=1 + 0.3 * rn(D), pre_bias=rn(D))
    t = [None if n in without else t[n].to(DEV) for n in NAMES]
    return t, rn(M, D).to(x_dtype).to(DEV), rn(M, D).to(dtype).to(DEV)


def check(t, dy, dh, groups=1, kind='rms', act='sigmoid', post=True, pre=True):
    leaves = [a.detach().requires_grad_() for a in t if a is not None]
    it = iter(leaves)
    mine = [None if a is None else next(it) for a in t]
    y, h = fm.block_norm(*mine, groups=groups, kind=kind, gate_act=act, post_norm=post, pre_norm=pre)
    outs = [(o, d) for o, d in ((y, dy), (h, dh)) if o is not None and o.requires_grad and not (o is mine[0])]
    got = torch.autograd.grad([o for o, _ in outs], leaves, [d for _, d in outs])
    wide = [a.detach().double().requires_grad_() for a in leaves]
    it = iter(wide)
    wy, wh = formula([None if a is None else next(it) for a in t], groups, kind, act, post, pre)
    wouts = [(o, d) for o, d, m in ((wy, dy, y), (wh, dh, h)) if o is not None and not (m is mine[0])]
    want = torch.autograd.grad([o for o, _ in wouts], wide, [d.double() for _, d in wouts])
    M, D = t[0].shape
    c = (D / 4 + 60) * 2.0 ** -24
    pairs = [('y', y, wy), ('h', h, wh)] + [(n, g, w) for n, g, w in zip([n for n, a in zip(NAMES, t) if a is not None], got, want)]
    for name, g, w in pairs:
        if g is None:
            continue
        w = w.detach()
        # the terms of a row (of a column, for a weight) are of the row's (column's) largest magnitude or below
        big = w.abs().amax(0 if name in NAMES[3:] else -1, keepdim=True) + 1
        extra = (M / 16 + 40) * 2.0 ** -24 * M ** 0.5 * (w.abs().amax() + 1) if name in NAMES[3:] else 0.0
        if name in NAMES[3:]:
            big = w.abs().amax() + M ** 0.5
        bound = 8 * c * big + extra + w.abs() * (torch.finfo(g.dtype).eps / 2) + (2.0 ** -25 if g.dtype == F16 else 0)
        err = (g.detach().double() - w).abs() - bound
        assert g.shape == w.shape and bool((err <= 0).all()), '%s: %.3g over its bound' % (name, float(err.max()))


TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]


@pytest.mark.parametrize('types', TYPES, ids=str)
@pytest.mark.parametrize('shape', [(1, 1, 1), (3, 7, 7), (385, 64, 4), (70, 65, 5), (33, 128, 2), (19, 200, 8), (40, 256, 1), (37, 300, 1), (21, 512, 4), (9, 999, 3), (50, 1000, 8),
                                   (11, 1024, 8), (7, 1500, 12), (5, 2048, 16), (6, 4096, 64), (4, 4100, 1), (3, 8192, 256), (5, 8190, 2)], ids=str)
def test_block_and_gradients(shape, types):
    M, D, groups = shape
    t, dy, dh = make(M, D, *types, seed=M + D)
    check(t, dy, dh, groups, 'layer', 'silu')
    check(t, dy, dh, groups, 'rms', 'sigmoid')


@pytest.mark.parametrize('without', [('branch', 'gate', 'scale', 'post_weight', 'post_bias'), ('gate',), ('scale', 'post_bias', 'pre_bias'),
                                     ('scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias'), ('branch', 'gate', 'scale', 'post_weight', 'post_bias', 'pre_bias')], ids=str)
def test_parts_left_out(without):
    for D, kind in ((64, 'rms'), (130, 'layer'), (1200, 'layer')):
        t, dy, dh = make(67, D, F32, F32, 4, without)
        check(t, dy, dh, 2 if t[1] is not None else 1, kind, 'silu')
        if t[1] is not None:
            check(t, dy, dh, 2, kind, 'silu', pre=True, post=True)
            t2 = [a if n not in ('post_weight', 'post_bias') else None for n, a in zip(NAMES, t)]
            check(t2, dy, dh, 1, kind, 'sigmoid', post=False)
            t2 = [a if n not in ('pre_weight', 'pre_bias') else None for n, a in zip(NAMES, t)]
            check(t2, dy, dh, 2, kind, 'sigmoid', pre=False)


def test_strides_and_alignment():
    """rows out of wider ones, odd offsets, an order other than the tested one: the same bits as the contiguous form"""
    gen = torch.Generator().manual_seed(1)
    for D, groups in ((64, 4), (61, 1), (1000, 8)):
        wide = torch.randn(3, 50, 3 * D + 5, generator=gen).to(DEV)
        x, b, g = wide[:, :, 1:D + 1], wide[:, :, D + 2:2 * D + 2], wide[:, :, 2 * D + 5:3 * D + 5]
        flip = lambda a: a.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # noqa: E731
        w = torch.randn(5, 2 * D, generator=gen).to(DEV)[:, ::2]
        want = fm.block_norm(x.contiguous(), b.contiguous(), g.contiguous(), *[a.contiguous() for a in w], groups=groups, kind='layer')
        for args in ((x, b, g), (flip(x), flip(b), g), (x.transpose(0, 1).contiguous().transpose(0, 1), b, flip(g))):
            got = fm.block_norm(*args, *w, groups=groups, kind='layer')
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_gradient_against_differences():
    """central differences in float64 of the definition along one direction against the framework's gradients"""
    for kind, act in itertools.product(('rms', 'layer'), ('sigmoid', 'silu')):
        t, dy, dh = make(13, 48, F32, F32, 9)
        leaves = [a.requires_grad_() for a in t]
        grads = torch.autograd.grad(fm.block_norm(*leaves, groups=3, kind=kind, gate_act=act), leaves, (dy, dh))
        gen = torch.Generator().manual_seed(3)
        dirs = [torch.randn(a.shape, generator=gen).double().to(DEV) for a in t]

        def f(e):
            y, h = formula([a.detach().double() + e * d for a, d in zip(t, dirs)], 3, kind, act, True, True)
            return float((y * dy.double()).sum() + (h * dh.double()).sum())
        want = (f(1e-5) - f(-1e-5)) / 2e-5
        size = sum(float((g.double() * d).abs().sum()) for g, d in zip(grads, dirs))
        assert abs(sum(float((g.double() * d).sum()) for g, d in zip(grads, dirs)) - want) < 1e-5 * size


def test_rows_do_not_reach_each_other_and_edges():
    t, _, _ = make(10, 64, F32, F32, 2)
    clean = fm.block_norm(*t, groups=4)
    x, b, g = (a.clone() for a in t[:3])
    x[3], b[5, 7], g[8] = float('nan'), float('inf'), float('nan')
    got = fm.block_norm(x, b, g, *t[3:], groups=4)
    rest = [0, 1, 2, 4, 6, 7, 9]
    assert all(torch.equal(p[rest], q[rest]) for p, q in zip(got, clean))
    b[5] = 0
    zero = fm.block_norm(x[:1], torch.zeros_like(b[:1]), None, groups=4)[0]
    assert torch.equal(zero, x[:1])                                        # a branch of zeros norms to zeros
    g[0], g[1] = 200.0, -200.0
    y = fm.block_norm(x[:2], b[:2], g[:2], groups=4, pre_norm=False)[0]
    u = fm.block_norm(x[:2], b[:2], groups=4, pre_norm=False)[0]
    assert torch.equal(y[0], u[0]) and torch.equal(y[1], x[1])             # a gate far open and far shut
    e = [torch.empty(0, 64, device=DEV).requires_grad_() for _ in range(3)]
    w = torch.ones(64, device=DEV).requires_grad_()
    y, h = fm.block_norm(*e, w)
    assert y.shape == h.shape == (0, 64)
    assert bool((torch.autograd.grad((y, h), w, (y.detach(), h.detach()))[0] == 0).all())
    one = fm.block_norm(torch.ones(64, device=DEV))                         # a single row without a batch axis
    assert one[1].shape == (64,) and float((one[1] - (1 + 1e-5) ** -0.5).abs().max()) < 1e-6


def test_streams_and_graphs():
    t, dy, dh = make(1000, 64, F32, F32, 7)
    run = lambda: fm.block_norm(*t, groups=4, kind='layer')  # noqa: E731
    leaves = [a.detach().requires_grad_() for a in t]
    grads = lambda: torch.autograd.grad(fm.block_norm(*leaves, groups=4, kind='layer'), leaves, (dy, dh))  # noqa: E731
    want, wgrad = [a.clone() for a in run()], [a.clone() for a in grads()]
    assert all(torch.equal(a, b) for a, b in zip(grads(), wgrad))          # the same bits again
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, ggrad = run(), grads()
    for seed in (30, 31, 32):
        new, _, _ = make(1000, 64, F32, F32, seed)
        for a, b, c in zip(t, leaves, new):
            a.copy_(c)
            with torch.no_grad():
                b.copy_(c)
        want, wgrad = [a.clone() for a in run()], [a.clone() for a in grads()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(ggrad, wgrad))
