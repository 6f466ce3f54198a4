"""-m gpu: log-probability and entropy of discrete actions from the features, and their gradients, against the definition in float64.

Tolerances, in units u = 2^-24 of float32: a logit is a sum of K products, off by at most ez = (K + 4) u sum |x w| (largest over a row's logits); the softmax's
sum of V terms adds (V + 40) u relative, so log_prob is off by 2 ez + (V + 40) u + 2 u (|z_a| + |lse|) and the entropy by (2 H + 2) ez + 2 (V + 64) u (H + 2).
dz = dl (1 - p) - de p (log p + H) follows by the product rule from p's relative error ep = 2 ez + (V + 40) u + 4 u |log p|; the products dx = dz W and dW = dz^T x
add (n + 8) u over their n terms, half a step of the operands' type for dz where it is stored, and half a step of the output's."""
import math

import pytest
import torch

import fair_marl_amd as fm

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def definition(X, W, b, act, avail, dl=None, de=None):
    z = X @ W.t() + (0 if b is None else b)
    if avail is not None:
        z = z.masked_fill(~avail, -math.inf)
    part = (act >= 0) & (z > -math.inf).any(-1)
    zz = z.masked_fill(~part[:, None], 0.0)
    lse = torch.logsumexp(zz, -1)
    logs = zz - lse[:, None]
    p = torch.exp(logs)
    plogs = torch.where(p > 0, p * logs, torch.zeros_like(p))
    H = -plogs.sum(-1)
    lp = logs.gather(1, act.clamp(min=0)[:, None])[:, 0]
    out = [torch.where(part, lp, 0.0), torch.where(part, H, 0.0)]
    if dl is None:
        return out, z, p, logs, part
    hot = torch.zeros_like(p).scatter_(1, act.clamp(min=0)[:, None], 1.0).masked_fill(z == -math.inf, 0.0)
    dz = torch.where(part[:, None], dl[:, None] * (hot - p) - de[:, None] * (plogs + p * H[:, None]), 0.0)
    X = X.masked_fill(~part[:, None], 0.0)
    return out + [dz @ W, dz.t() @ X, dz.sum(0)], z, p, logs, part, dz


def make(M, K, V, dtype, seed, avail=True, pad=0.1, small=1.0):
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    X, W, b = rn(M, K).to(dtype), (2 * K ** -0.5 * rn(V, K)).to(dtype), (0.5 * rn(V)).to(dtype)
    act = torch.randint(0, V, (M,), generator=gen)
    av = None
    if avail:
        av = torch.rand(M, V, generator=gen) > 0.3
        av[torch.arange(M), act] = True
        av[torch.rand(M, generator=gen) < 0.05] = False           # rows with nothing available
    act = torch.where(torch.rand(M, generator=gen) < pad, -1 - torch.randint(0, 5, (M,), generator=gen), act)
    dl, de = small * rn(M), 0.1 * small * rn(M)
    return [None if t is None else t.to(DEV) for t in (X, W, b, act, av, dl, de)]


def check(X, W, b, act, av, dl, de, got):
    K, V, M = X.shape[1], W.shape[0], X.shape[0]
    Xd, Wd, bd = X.double(), W.double(), None if b is None else b.double()
    want, z, p, logs, part, dz = definition(Xd, Wd, bd, act, av, dl.double(), de.double())
    ez = ((K + 4) * U * (Xd.abs() @ Wd.abs().t() + (0 if b is None else bd.abs()))).amax(-1)
    H, lse = want[1], (z.masked_fill(~part[:, None], 0.0)).logsumexp(-1)
    lp = torch.where(torch.isfinite(want[0]), want[0], 0.0)
    e_lp = 2 * ez + (V + 40) * U + 4 * U * (lp.abs() + 2 * lse.abs())
    e_H = (2 * H + 2) * ez + 2 * (V + 64) * U * (H + 2)
    l0 = torch.where(p > 0, logs, 0.0)
    ep = (2 * ez + (V + 40) * U)[:, None] + 4 * U * (l0.abs() + lse.abs()[:, None])
    e_dz = dl.double().abs()[:, None] * (p * ep + U) + de.double().abs()[:, None] * p * (ep * ((l0 + H[:, None]).abs() + 2) + e_H[:, None] + 4 * U * (l0.abs() + H[:, None]))
    half = torch.finfo(X.dtype).eps / 2 if X.dtype != F32 else 0.0
    # float16: dz is stored times a power of two that brings the largest upstream value to about 2^12: its smallest step is then 2^-24 / 2^11 of that
    floor = 2.0 ** -35 * float((dl.abs() + de.abs() * (1 + math.log(V))).max()) if X.dtype == F16 else 0.0
    e_dz = torch.where(part[:, None], e_dz + half * dz.abs() + floor, 0.0)
    Xz = Xd.masked_fill(~part[:, None], 0.0).abs()
    bounds = [torch.where(part, e_lp, 0.0), torch.where(part, e_H, 0.0), e_dz @ Wd.abs() + (V + 8) * U * (dz.abs() @ Wd.abs()),
              e_dz.t() @ Xz + (M + 8) * U * (dz.abs().t() @ Xz), e_dz.sum(0) + (M + 8) * U * dz.abs().sum(0)]
    for name, g, w, bound in zip(('log_prob', 'entropy', 'dx', 'dW', 'db'), got, want, bounds):
        if g is None:
            continue
        g = g.double()
        fin = torch.isfinite(w)
        assert torch.equal(torch.isfinite(g), fin) and torch.equal(g[~fin], w[~fin]), name
        t = {2: 'dx', 3: 'dW'}
        out = torch.finfo(X.dtype).eps / 2 * w.abs() + (2.0 ** -25 if X.dtype == F16 else 0.0) if name in t.values() or name == 'db' else U * w.abs()
        err = ((g - w).abs() - bound - out)[fin]
        assert err.numel() == 0 or float(err.max()) <= 0, '%s: %.3g over its bound' % (name, float(err.max()))


def run(X, W, b, act, av, dl, de):
    leaves = [t.detach().requires_grad_() for t in (X, W, b) if t is not None]
    out = fm.action_log_probs(leaves[0], leaves[1], leaves[2] if b is not None else None, act, av)
    grads = torch.autograd.grad(out, leaves, (dl, de))
    return [t.detach() for t in out] + list(grads) + ([None] if b is None else [])


SHAPES = [(1, 1, 1), (3, 5, 2), (384, 64, 5), (1000, 64, 5), (50, 100, 7), (77, 256, 16), (200, 30, 25), (65, 128, 32), (33, 64, 64), (129, 33, 50), (70000, 24, 5),
          (5, 300, 5), (130, 128, 33), (300, 65, 65), (257, 100, 625), (1, 64, 1000), (129, 129, 129), (64, 513, 300)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_log_probs_entropy_and_gradients(shape, dtype):
    t = make(*shape, dtype, seed=sum(shape))
    check(*t, run(*t))


@pytest.mark.parametrize('shape', [(40, 64, 5), (140, 64, 200)], ids=str)
def test_forms_of_the_arguments(shape):
    """no bias, a float32 bias, no mask; actions as the buffer holds them (float32, a trailing 1) and int32; masks as bool, bytes and float32; strided and unaligned rows"""
    X, W, b, act, av, dl, de = make(*shape, BF16, seed=2)
    check(X, W, None, act, av, dl, de, run(X, W, None, act, av, dl, de))
    check(X, W, b, act.clamp(min=0), None, dl, de, run(X, W, b, act.clamp(min=0), None, dl, de))
    check(X, W, b.float(), act, av, dl, de, run(X, W, b.float(), act, av, dl, de))
    want = fm.action_log_probs(X, W, b, act, av)
    wide = torch.randn(shape[0], shape[1] + 3, device=DEV).to(BF16)
    wide[:, 1:-2] = X
    ww = torch.randn(shape[2], shape[1] + 5, device=DEV).to(BF16)
    ww[:, 3:-2] = W
    am = torch.zeros(shape[0], shape[2] + 1, device=DEV)
    am[:, 1:] = av
    for got in (fm.action_log_probs(X, W, b, act.float().unsqueeze(-1), av.float()), fm.action_log_probs(X, W, b, act.int(), av.to(torch.uint8)),
                fm.action_log_probs(wide[:, 1:-2], ww[:, 3:-2], b.float(), act, am[:, 1:]),
                fm.action_log_probs(X.t().contiguous().t(), W.t().contiguous().t(), b, act, av.t().contiguous().t())):
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    lead = fm.action_log_probs(X.view(4, -1, shape[1]), W, b, act.view(4, -1, 1), av.view(4, -1, shape[2]))
    assert lead[0].shape == (4, shape[0] // 4) and torch.equal(lead[0].reshape(-1), want[0])


@pytest.mark.parametrize('V', [5, 40, 300])
def test_rows_that_take_no_part(V):
    """padding and rows without an available action, whatever they hold; an unavailable action, one that does not exist, a NaN and an infinity in a row of their own"""
    X, W, b, act, av, dl, de = make(200, 32, V, F32, seed=V, pad=0.0)
    av = torch.ones_like(av)
    base = run(X, W, b, act, av, dl, de)
    drop = torch.tensor([3, 17, 60, 130], device=DEV)
    rest = torch.ones(200, dtype=torch.bool, device=DEV)
    rest[drop] = False
    X2, act2, av2, dl2, de2 = X.clone(), act.clone(), av.clone(), dl.clone(), de.clone()
    X2[drop[:2]], act2[drop[:2]], av2[drop[2:]] = math.nan, -1, False
    X2[drop[2]], dl2[drop], de2[drop] = math.inf, math.nan, math.inf
    got = run(X2, W, b, act2, av2, dl2, de2)
    clean = run(X[rest], W, b, act[rest], av[rest], dl[rest], de[rest])
    assert bool((got[0][drop] == 0).all()) and bool((got[1][drop] == 0).all()) and bool((got[2][drop] == 0).all())
    assert all(torch.equal(g[rest], c) for g, c in zip(got[:3], clean[:3]))
    for g, c in zip(got[3:], clean[3:]):
        assert float((g - c).abs().max()) <= 300 * U * float(dl.abs().sum()) * 4
    # unavailable: -inf with the others' gradient; not there: NaN without one; neither reaches another row
    act3, av3 = act.clone(), av.clone()
    act3[5], act3[9] = V, V + 1000
    av3[7, act3[7]] = False
    got = run(X, W, b, act3, av3, dl, de)
    keep = [i for i in range(200) if i not in (5, 7, 9)]
    assert bool(torch.isnan(got[0][[5, 9]]).all()) and bool((got[2][[5, 9]] == 0).all()) and float(got[0][7]) == -math.inf and bool(torch.isfinite(got[2]).all())
    assert torch.equal(got[0][keep], base[0][keep]) and torch.equal(got[2][keep], base[2][keep]) and bool(torch.isfinite(got[3]).all())
    X4 = X.clone()
    X4[11, 3] = math.nan
    lp, en = fm.action_log_probs(X4, W, b, act, av)
    assert bool(torch.isnan(lp[11])) and bool(torch.isnan(en[11])) and int(torch.isnan(lp).sum()) == 1
    # a single available action: log_prob and entropy exactly 0, no gradient
    one = torch.zeros_like(av)
    one[torch.arange(200, device=DEV), act] = True
    got = run(X, W, b, act, one, dl, de)
    assert bool((got[0] == 0).all()) and bool((got[1] == 0).all()) and float(got[2].abs().max()) <= 4 * U * float(dl.abs().max()) * float(W.abs().max()) * 4


def test_large_logits_and_small_upstream_gradients():
    """logits of a thousand neither overflow nor lose the row; upstream gradients of a mean over a million rows survive half precision"""
    for V in (5, 200):
        t = make(100, 64, V, F32, seed=1)
        t[0] = t[0] * 200
        check(*t, run(*t))
        for dtype in (F16, BF16):
            t = make(300, 64, V, dtype, seed=2, small=1e-7)
            lp, en, dx, dw, db = run(*t)
            s = 2.0 ** 24
            X, W, b, act, av, dl, de = t
            big = run(X, W, b, act, av, dl * s, de * s)
            tiny = torch.finfo(dtype).tiny if dtype == F16 else 0.0
            step = 2 * torch.finfo(dtype).eps
            for g, w in zip((dx, dw, db), big[2:]):     # the same numbers times 2^24, where the type can hold them
                assert bool(((g.double() * s - w.double()).abs() <= step * w.double().abs() + s * tiny * 2.0 ** -10 + 1e-30 + step * float(w.abs().max())).all())


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('V', [5, 90])
def test_bias_of_the_lowest_value(V, dtype):
    """float32's lowest value in the bias where an action is not wanted: it is there all the same, with probability 0 and the gradient of a taken action; -inf takes it away"""
    X, W, b, act, _, dl, _ = make(60, 32, V, dtype, seed=5, avail=False, pad=0.0)
    b = b.float()
    b[1], b[3] = torch.finfo(F32).min, -math.inf
    act[:20], act[20:30] = 1, 3
    act[30:] = torch.where((act[30:] == 1) | (act[30:] == 3), 0, act[30:])
    leaves = [t.requires_grad_() for t in (X, W, b)]
    lp, ent = fm.action_log_probs(X, W, b, act)
    dX, dW, db = torch.autograd.grad((lp, ent), leaves, (dl, torch.ones_like(ent)))
    assert bool((lp[:20] < -1e38).all()) and bool(torch.isfinite(lp[:20]).all()) and bool((lp[20:30] == -math.inf).all()) and bool(torch.isfinite(lp[30:]).all())
    assert all(bool(torch.isfinite(t).all()) for t in (ent, dX, dW, db)) and float(db[3]) == 0
    assert abs(float(db[1] - dl[:20].double().sum())) < 1e-5     # the taken action's 1 - p, p = 0: 20 additions of numbers up to 4, 20 x 4 x 2^-24 off at most
    rest = [i for i in range(V) if i not in (1, 3)]
    with torch.no_grad():   # the same rows without the two actions, in float64; the bounds as above
        Xd, Wd = X[30:].double(), W[rest].double()
        want, z, *_ = definition(Xd, Wd, b[rest].double(), torch.tensor([rest.index(int(a)) for a in act[30:]], device=DEV), None)
        ez = ((32 + 4) * U * (Xd.abs() @ Wd.abs().t() + b[rest].double().abs())).amax(-1)
        e_lp = 2 * ez + (V + 40) * U + 4 * U * (want[0].abs() + 2 * z.logsumexp(-1).abs())
        e_H = (2 * want[1] + 2) * ez + 2 * (V + 64) * U * (want[1] + 2)
        assert bool(((lp[30:] - want[0]).abs() <= e_lp).all()) and bool(((ent[30:] - want[1]).abs() <= e_H).all())


@pytest.mark.parametrize('shape', [(30, 24, 5), (30, 24, 80)], ids=str)
def test_gradient_against_differences(shape):
    X, W, b, act, av, dl, de = make(*shape, F32, seed=4)
    got = run(X, W, b, act, av, dl, de)
    gen = torch.Generator().manual_seed(5)
    dirs = [torch.randn(t.shape, generator=gen).double().to(DEV) for t in (X, W, b)]

    def f(e):
        out = definition(*[t.double() + e * d for t, d in zip((X, W, b), dirs)], act, av)[0]
        return float((out[0] * dl.double()).sum() + (out[1] * de.double()).sum())
    want = (f(1e-5) - f(-1e-5)) / 2e-5
    size = sum(float((g.double() * d).abs().sum()) for g, d in zip(got[2:], dirs))
    assert abs(sum(float((g.double() * d).sum()) for g, d in zip(got[2:], dirs)) - want) < 1e-5 * size


def test_pieces_of_the_rows_and_of_the_actions():
    """more rows than a chunk holds and more actions than a piece: sums run over both (70 000 rows: two chunks; 2 200 actions there: three pieces)"""
    t = make(70000, 16, 2200, F32, seed=6, avail=False)
    check(*t, run(*t))
    t = make(66000, 40, 70, BF16, seed=7)
    check(*t, run(*t))


def test_one_output_no_rows_and_single_features():
    X, W, b, act, av, dl, de = make(100, 64, 5, F32, seed=8)
    z = torch.zeros_like(dl)
    for use, d in ((0, (dl, z)), (1, (z, de))):
        leaves = [t.detach().requires_grad_() for t in (X, W, b)]
        got = torch.autograd.grad(fm.action_log_probs(*leaves, act, av)[use], leaves, d[use])
        assert all(torch.equal(a, c) for a, c in zip(got, run(X, W, b, act, av, *d)[2:]))
    leaves = [X[:0].detach().requires_grad_(), W.detach().requires_grad_()]
    out = fm.action_log_probs(*leaves, None, act[:0], av[:0])
    assert out[0].shape == (0,)
    g = torch.autograd.grad(out, leaves, (z[:0], z[:0]))
    assert g[0].shape == (0, 64) and bool((g[1] == 0).all())
    lp, en = fm.action_log_probs(X[0], W, b, act[:1].clamp(min=0))
    assert lp.shape == () and en.shape == ()


@pytest.mark.parametrize('shape', [(300, 64, 5), (300, 64, 500)], ids=str)
def test_streams_and_graphs(shape):
    t = make(*shape, F16, seed=9)
    X, W, b, act, av, dl, de = t
    b = b.float()
    leaves = [a.detach().requires_grad_() for a in (X, W, b)]

    def go():
        out = fm.action_log_probs(*leaves, act, av)
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, (dl, de)))
    want = [a.clone() for a in go()]
    assert all(torch.equal(p, q) for p, q in zip(go(), want))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = go()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = go()
    for seed in (40, 41, 42):
        new = make(*shape, F16, seed=seed)
        with torch.no_grad():
            for dst, src in zip(leaves + [act, av, dl, de], new):
                dst.copy_(src)
        want = [a.clone() for a in go()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, want))
