"""-m gpu: block_norm at the borders of its arguments, against its formulas in float64 (the bounds of test_hip_policy_block.py)."""
import pytest
import torch

import fair_marl_amd as fm
from test_hip_policy_block import DEV, F32, NAMES, formula, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('without', [(), ('branch', 'gate', 'scale', 'post_weight', 'post_bias')], ids=['branch', 'no branch'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('shape', [(17, 64, 4), (1, 60, 3), (9, 128, 4), (5, 256, 8), (3, 250, 5), (5, 1000, 8)], ids=str)
@pytest.mark.parametrize('eps', [0.0, 1e-60])
def test_no_eps(eps, shape, kind, without):
    """rows that are not zero need no eps: the formulas, whatever number of rows a workgroup holds"""
    M, D, groups = shape
    t, dy, dh = make(M, D, F32, F32, seed=M + D, without=without)
    leaves = [a.requires_grad_() for a in t if a is not None]
    y, h = fm.block_norm(*t, groups=groups, kind=kind, eps=eps)
    outs, ds = ([h], [dh]) if 'branch' in without else ([y, h], [dy, dh])
    got = torch.autograd.grad(outs, leaves, ds)
    wide = [None if a is None else a.detach().double().requires_grad_() for a in t]
    wy, wh = formula(wide, groups, kind, 'sigmoid', True, True, eps)
    want = torch.autograd.grad([wh] if 'branch' in without else [wy, wh], [a for a in wide if a is not None], [d.double() for d in ds])
    c = (D / 4 + 60) * 2.0 ** -24
    for name, a, b in [('h', h, wh)] + list(zip([n for n, a in zip(NAMES, t) if a is not None], got, want)):
        b = b.detach()
        if name in NAMES[3:]:
            big, extra = b.abs().amax() + M ** 0.5, (M / 16 + 40) * 2.0 ** -24 * M ** 0.5 * (b.abs().amax() + 1)
        else:
            big, extra = b.abs().amax(-1, keepdim=True) + 1, 0.0
        err = (a.detach().double() - b).abs() - (8 * c * big + extra + b.abs() * 2.0 ** -24)
        assert bool((err <= 0).all()), '%s: %.3g over its bound' % (name, float(err.max()))
