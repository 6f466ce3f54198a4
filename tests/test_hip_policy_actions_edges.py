"""-m gpu: action_log_probs where its tiles, pieces and chunks end and begin, and at the ends of its types.  Definition and bounds are those of test_hip_policy_actions.py."""
import math

import pytest
import torch

import fair_marl_amd as fm
from fair_marl_amd import _lib
from test_hip_policy_actions import BF16, DEV, F16, F32, U, check, make, run

pytestmark = pytest.mark.gpu


def up(n, m):
    return (n + m - 1) // m * m


def half_plan(M, K, V, backward):
    """The sizes of the half precision way for many actions: (tiles in a workgroup's run, pieces of the actions, chunks of the rows), after a look that the library still works by
    them: its workspace is the sum of what they ask for."""
    Mp, Kp, Vp = up(M, 256), up(K, 256), up(V, 256)
    Mc = min(Mp, max(1024, min(65536, (256 << 20) // (2 * Kp) // 256 * 256)))
    P = min(Vp, max(256, (256 << 20) // (2 * Mc) // 256 * 256))
    tm, tk, tv = Mc // 256, Kp // 256, P // 256
    parts = lambda tiles, steps: max(1, min(256 // tiles, steps // 4, 16))  # noqa: E731
    sx, sw = parts(tm * tk, P // 64), parts(tv * tk, Mc // 64)
    turns, rest = (tm, tv) if backward else (Vp // 256, tm)
    sz = max(1, min(256 // rest, turns))
    sizes = [2 * Mc * Kp, 2 * Vp * Kp, 4 * Vp, 4 * Mc, 16 * Mc if backward else 0]
    if backward:
        sizes += [2 * Mc * P, 4 * max(sx * Mc * Kp, sw * P * Kp), 4 * Mc * Kp if P < Vp else 0, 4 * Vp * Kp if Mc < Mp else 0, 4 * (Mc // 64) * P, 4 * 257]
    else:
        sizes += [12 * 2 * sz * Mc, 4 * Mc]
    a = _lib.FmarlActions(M, K, V, _lib.T_BF16, 0, 0, 0, 4096, K, 4096, K, None, 4096, None, 0)
    assert _lib.load().fmarl_action_log_probs_workspace(a, int(backward)) == sum(up(n, 256) for n in sizes), 'the plan is another one: choose sizes that have several tiles and pieces'
    return -(-turns // sz), -(-Vp // P), -(-Mp // Mc)


@pytest.mark.parametrize('dtype', [BF16, F16], ids=str)
@pytest.mark.parametrize('shape,kind', [((16384, 24, 4096), 'maxima that rise'), ((16384, 96, 4096), 'maxima that fall'), ((16300, 40, 4000), 'tiles without an action'),
                                        ((16300, 300, 4000), 'without a mask')], ids=str)
def test_runs_of_several_tiles(shape, kind, dtype):
    """a workgroup walks four tiles one after the other, forwards and backwards: the running maximum and sums, the loads over a tile's end (one step a tile: three tiles on their way)"""
    assert half_plan(*shape, False)[0] >= 3 and half_plan(*shape, True)[0] >= 3
    t = make(*shape, dtype, seed=sum(shape), avail=kind == 'tiles without an action')
    V, b, act, av = shape[2], t[2], t[3], t[4]
    tile = torch.arange(V, device=DEV) // 256
    if kind == 'maxima that rise':
        b.add_(2.0 * tile.to(dtype))
    if kind == 'maxima that fall':
        b.sub_(2.0 * tile.to(dtype))
    if av is not None:      # first, middle and last tiles of a run without an available action, and all but one of them
        rows = torch.arange(shape[0], device=DEV)[:, None] % 5
        av &= ~(((rows == 0) & (tile % 4 == 0)) | ((rows == 1) & (tile % 4 == 2)) | ((rows == 2) & (tile % 4 == 3)) | ((rows == 3) & (tile != 6)))
        av[torch.arange(shape[0], device=DEV), act.clamp(min=0)] |= act >= 0
    check(*t, run(*t))


@pytest.mark.parametrize('dtype', [BF16, F16], ids=str)
def test_pieces_of_the_actions_in_half_precision(dtype):
    """two pieces of the actions, the last one narrower, for each of two chunks of the rows"""
    shape = (66000, 16, 2200)
    assert half_plan(*shape, True)[1:] == (2, 2)
    t = make(*shape, dtype, seed=70, avail=False)
    check(*t, run(*t))


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('V', [5, 90])
def test_a_single_action_whose_bias_is_the_lowest_value(V, dtype):
    """rows whose one available action has float32's lowest value for a bias: it is taken with certainty, and no gradient comes of it"""
    X, W, b, act, _, dl, de = make(60, 32, V, dtype, seed=71, avail=False, pad=0.0)
    b = b.float()
    b[1] = torch.finfo(F32).min
    act[:30] = 1
    act[30:] = torch.where(act[30:] == 1, 0, act[30:])
    av = torch.ones(60, V, dtype=torch.bool, device=DEV)
    av[:30] = False
    av[:30, 1] = True
    lp, ent, dX, dW, db = run(X, W, b, act, av, dl, de)
    assert bool((lp[:30] == 0).all()) and bool((ent[:30] == 0).all()) and bool((dX[:30] == 0).all())
    assert float(db[1]) == 0 and bool((dW[1] == 0).all())        # the rows that have others: probability 0
    rest = run(X[30:], W, b, act[30:], None, dl[30:], de[30:])
    assert torch.equal(lp[30:], rest[0]) and torch.equal(ent[30:], rest[1])


def test_more_weights_than_threads_of_a_launch():
    """2^32 weights (524 288 actions of 8 192 features): every row of their gradient is formed"""
    M, K, V = 3, 8192, 1 << 19
    gen = torch.Generator(device=DEV).manual_seed(72)
    X = torch.randn(M, K, device=DEV, generator=gen).to(BF16)
    W = torch.empty(V, K, dtype=BF16, device=DEV)
    for a in range(0, V, 1 << 16):      # (rows of a table: 4 billion normal numbers take longer than the rest)
        W[a:a + (1 << 16)] = torch.randn(1 << 10, K, device=DEV, generator=gen).to(BF16).repeat(64, 1) * K ** -0.5
    act = torch.tensor([0, V // 2 + 1, V - 1], device=DEV)
    dl = torch.tensor([1.0, -2.0, 0.5], device=DEV)
    leaves = X.requires_grad_(), W.requires_grad_()
    lp, ent = fm.action_log_probs(*leaves, None, act)
    dX, dW = torch.autograd.grad(lp, leaves, dl)
    with torch.no_grad():
        z = torch.cat([(X.float() @ W[a:a + (1 << 16)].float().t()).double() for a in range(0, V, 1 << 16)], 1)
        p = torch.softmax(z, -1)
        want = torch.log_softmax(z, -1)[torch.arange(M, device=DEV), act]
        # a logit is off by K u sum |x w| (here: K 0.64 K^-0.5 = 58 on average, within 12 of it), the sums over V terms by V u at most
        ez = (K + 4) * U * 70.0
        assert float((lp.double() - want).abs().max()) <= 2 * ez + (V + 40) * U + 4 * U * 40
        for rows in (slice(0, 600), slice(V // 2 - 300, V // 2 + 300), slice(V - 600, V)):
            hot = (torch.arange(V, device=DEV)[rows][None] == act[:, None]).double()
            dz = dl.double()[:, None] * (hot - p[:, rows])
            exact, size = dz.t() @ X.double(), dz.abs().t() @ X.double().abs()
            # dz: p's relative error, half a step of its type; the product's three terms, half a step of its own type
            bound = (2 * ez + (V + 40) * U + 8 * U * 40 + 2.0 ** -8) * size + 8 * U * size + 2.0 ** -8 * exact.abs()
            assert bool(((dW[rows].double() - exact).abs() <= bound).all())
        assert not bool((dW.view(-1, 1 << 16).abs().amax(1) == 0).any())     # no stretch is left out
