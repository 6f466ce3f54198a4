"""-m gpu: the policy's memory where one form of its kernels ends and the next begins, with values that cancel, overflow or are no numbers.  The recurrence in float64 and the
bounds are those of test_hip_policy_memory.py."""
import math

import pytest
import torch

import fair_marl_amd as fm
from test_hip_policy_memory import BF16, DEV, F16, F32, close, compare, make, recurrence, step_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('decay', ['token', 'head'])
@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('shape', [(1, 3, 2, 64, 64), (10, 37, 2, 64, 64), (10, 5, 3, 33, 100), (7, 3, 1, 128, 128), (32, 3, 2, 48, 16), (9, 5, 1, 65, 39), (10, 3, 3, 97, 5)], ids=str)
def test_few_tokens_of_wide_heads(shape, dtype, decay):
    """rows of lanes that share a head: two up to 64 wide, four beyond, the last with a part of its share or none; heads that do not fill the last wave"""
    q, k, v, g, S, masks, do, dS = make(*shape, dtype, decay, seed=sum(shape) + 1)
    leaves = [t.requires_grad_() for t in (q, k, v, g, S)]
    out, last = fm.memory_chunk(q, k, v, g, S, masks)
    grads = torch.autograd.grad((out, last), leaves, (do, dS))
    with torch.no_grad():
        compare((out, last) + grads, q, k, v, g, S, masks, shape[3] ** -0.5, do, dS)


SHAPES = [(12, 2, 2, 16, 16), (16, 5, 1, 5, 7), (40, 2, 1, 5, 7), (30, 2, 2, 100, 12), (90, 2, 2, 40, 24), (700, 1, 1, 16, 16), (700, 1, 2, 64, 64), (300, 1, 1, 128, 100)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('bad', [math.nan, math.inf])
@pytest.mark.parametrize('shape', SHAPES, ids=str)
def test_the_decays_gradient_next_to_what_is_no_number(shape, bad, dtype):
    """dg_t = r_t e^{g_t} <S_{t-1}, G_t>: what is not finite in k or v reaches the tokens behind it, in q or d_out those before it, and none of another episode; between the two,
    and beside a start, the gradient is finite"""
    L, B, H, dk, dv = shape
    for at, what in enumerate(('d_out', 'k', 'd_out, then v', 'q at a start', 'k, then d_out', 'states')):
        q, k, v, g, S, masks, do, dS = make(*shape, dtype, 'token', seed=50 + at)
        clean = [t.clone() for t in (q, k, v, g, S, masks, do, dS)]
        e0, s1, s2, e1 = L // 6, L // 3, L // 3 + max(2, L // 4), L - L // 6    # an episode and two of its tokens
        masks.fill_(1)
        masks[e0, 0] = masks[e1, 0] = 0
        if what.startswith('d_out'):
            do[s1, 0, :, dv // 2] = bad
        if what == 'k':
            k[s2, 0, 0] = bad
        if what == 'd_out, then v':
            v[s2, 0, :, 0] = bad
        if what == 'q at a start':
            q[e0, 0, :, dk - 1] = bad
        if what == 'k, then d_out':
            k[s1, 0, :, 0], do[s2, 0, :, 0] = bad, bad
        if what == 'states':
            S[0, 0], dS[0, H - 1, 0, 0] = bad, bad
        got = fm.memory_chunk_backward(q, k, v, g, do, dS, S, masks)
        shared = fm.memory_chunk_backward(q, k, v, g[0, 0].contiguous(), do, dS, S, masks)[3]
        wide = [t.double() for t in (q, k, v)]
        want = recurrence(*wide, g.double(), S.double(), masks == 0, dk ** -0.5, do.double(), dS.double())[5]
        cq, ck, cv, _, cS, _, cdo, cdS = [t.double().abs() for t in clean]
        mag = recurrence(cq, ck, cv, g.double(), cS, masks == 0, dk ** -0.5, cdo, cdS)
        gamma = (2 * L + dk + dv + 200) * 2.0 ** -24
        add = (cq * mag[2]).sum(-1) + (ck * mag[3]).sum(-1)
        bound = gamma * ((cS * mag[6]).sum((-1, -2)) + torch.cumsum(add, 0))
        fine = torch.isfinite(want)
        assert bool((~fine).any()) or what == 'q at a start'
        assert torch.equal(torch.isfinite(got[3]), fine), what
        close(torch.where(fine, got[3], 0.0), torch.where(fine, want, 0.0), torch.where(fine, bound + want.abs() * 2.0 ** -24, 0.0), what)
        head = recurrence(*wide, g[0, 0].double().expand(L, B, H), S.double(), masks == 0, dk ** -0.5, do.double(), dS.double())[5].sum((0, 1))
        assert torch.equal(torch.isfinite(shared), torch.isfinite(head)), what
        if what == 'q at a start':
            mag = recurrence(cq, ck, cv, g[0, 0].double().expand(L, B, H), cS, masks == 0, dk ** -0.5, cdo, cdS)
            run = (cS * mag[6]).sum((-1, -2)) + torch.cumsum((cq * mag[2]).sum(-1) + (ck * mag[3]).sum(-1), 0)
            close(shared, head, gamma * run.sum((0, 1)) + head.abs() * 2.0 ** -24, what)


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
@pytest.mark.parametrize('shape', [(40, 2, 1, 64, 64), (300, 1, 2, 100, 40)], ids=str)
def test_states_that_cancel(shape, dtype):
    """q (k, backwards) takes the difference of two rows of a state of about a thousand; nothing decays and nothing is added.  The products are exact, so out is within two float32
    additions of the terms, and its own rounding, of the difference: the state is float32 in whatever form the matrix units take it."""
    L, B, H, dk, dv = shape
    gen = torch.Generator().manual_seed(60)
    S = (1000 + torch.randn(B, H, dk, dv, generator=gen)).to(DEV)
    pick = torch.zeros(L, B, H, dk, dtype=dtype, device=DEV)
    for t in range(L):
        pick[t, :, :, t % dk], pick[t, :, :, (7 * t + 1) % dk] = 1, -1
    zero, none = torch.zeros_like(pick), torch.zeros(L, B, H, dv, dtype=dtype, device=DEV)
    g = torch.zeros(H, device=DEV)
    want = (pick.double().unsqueeze(-1) * S.double()).sum(-2)
    bound = 2 * 2.0 ** -24 * (pick.double().abs().unsqueeze(-1) * S.double()).sum(-2)
    out, last = fm.memory_chunk(pick, zero, none, g, S, scale=1.0)
    close(out, want, bound + step_of(out, want), 'out')
    assert torch.equal(last, S)
    dv_ = fm.memory_chunk_backward(zero, pick, none, g, none, S, None, scale=1.0)[2]
    close(dv_, want, bound + step_of(dv_, want), 'dv')


@pytest.mark.parametrize('dtype', [F32, BF16, F16], ids=str)
def test_products_that_cancel(dtype):
    """two keys whose products with q are near 1025.6 and -1025.6, their values equal: out is the small difference, to the float32 additions of the two terms and its own rounding"""
    L, dk, dv = 48, 64, 64
    gen = torch.Generator().manual_seed(61)
    q = torch.zeros(L, 1, 1, dk, dtype=dtype)
    k, v = torch.zeros_like(q), torch.zeros(L, 1, 1, dv, dtype=dtype)
    q[8:, 0, 0, 0], q[8:, 0, 0, 1], q[8:, 0, 0, 2] = 16, 2.0 ** -4, 1
    k[2, 0, 0, 0], k[5, 0, 0, 0], k[2, 0, 0, 2], k[5, 0, 0, 2] = 64, -64, 1.5, -1.5
    k[2, 0, 0, 1], k[5, 0, 0, 1] = torch.rand(2, generator=gen).to(dtype) + 1
    v[2], v[5] = 1, 1
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    out, _ = fm.memory_chunk(q, k, v, torch.zeros(1, device=DEV), None, scale=1.0)
    want = recurrence(q.double(), k.double(), v.double(), torch.zeros(L, 1, 1, device=DEV).double(), torch.zeros(1, 1, dk, dv, device=DEV).double(), torch.zeros(L, 1, device=DEV) != 0, 1.0)[0]
    mag = recurrence(q.double().abs(), k.double().abs(), v.double(), torch.zeros(L, 1, 1, device=DEV).double(), torch.zeros(1, 1, dk, dv, device=DEV).double(),
                     torch.zeros(L, 1, device=DEV) != 0, 1.0)[0]
    close(out, want, 2 * 2.0 ** -24 * mag + step_of(out, want), 'out')     # near 1024 a rounding is off by 2^-14 at most: one in each product q k, two where the terms are added


@pytest.mark.parametrize('value', [torch.finfo(F32).min, torch.finfo(F32).max])
@pytest.mark.parametrize('shape', [(10, 3, 2, 16, 16), (40, 2, 1, 64, 64), (40, 2, 1, 16, 100), (300, 1, 2, 100, 40)], ids=str)
def test_the_types_lowest_value_in_another_episode(shape, value):
    """padding of float32's lowest or largest value before an episode's start, in q, k, v and d_out: nothing of it behind the start, nor before it backwards"""
    L, B, H, dk, dv = shape
    q, k, v, g, S, masks, do, dS = make(*shape, F32, 'token', seed=62)
    masks.fill_(1)
    then = L // 2
    masks[then] = 0
    clean = [t.clone() for t in (q, k, v, do)]
    for t in (q, k, v, do):
        t[then - 2] = value
    out, last = fm.memory_chunk(q, k, v, g, S, masks)
    grads = fm.memory_chunk_backward(q, k, v, g, do, dS, S, masks)
    cq, ck, cv, cdo = [t.double() for t in clean]
    args = g.double(), S.double(), masks == 0, dk ** -0.5
    want = recurrence(cq, ck, cv, *args, cdo, dS.double())
    mag = recurrence(cq.abs(), ck.abs(), cv.abs(), g.double(), S.double().abs(), masks == 0, dk ** -0.5, cdo.abs(), dS.double().abs())
    gamma = (2 * L + dk + dv + 200) * 2.0 ** -24
    for name, a, i in (('out', out, 0), ('dq', grads[0], 2), ('dk', grads[1], 3), ('dv', grads[2], 4)):
        close(a[then:], want[i][then:], gamma * mag[i][then:] + step_of(a, want[i][then:]), name)
    close(last, want[1], gamma * mag[1] + step_of(last, want[1]), 'state')
    # the other way round: in the later episode, nothing of it before the start
    q, k, v, do = (t.float() for t in clean)
    for t in (q, k, v, do):
        t[then + 1] = value
    out, _ = fm.memory_chunk(q, k, v, g, S, masks)
    grads = fm.memory_chunk_backward(q, k, v, g, do, dS, S, masks)
    for name, a, i in (('out', out, 0), ('dq', grads[0], 2), ('dk', grads[1], 3), ('dv', grads[2], 4)):
        close(a[:then], want[i][:then], gamma * mag[i][:then] + step_of(a, want[i][:then]), name)
    close(grads[4], want[6], gamma * mag[6] + step_of(grads[4], want[6]), 'dS0')


@pytest.mark.parametrize('L', [6, 16])
def test_the_running_difference_of_few_tokens_keeps_small_terms(L):
    """one row, one column, nothing decays: dg_t = S G_t with G_t the sum of q_j d_out_j behind, 2^24, 2^24 + 1 and 1.  Every term is exact in float32, their sum is not on its way"""
    z = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    q, k, do = z(L, 1, 1, 1), z(L, 1, 1, 1), z(L, 1, 1, 1)
    q[-1], do[-1], q[-2], do[-2], q[-4], do[-4] = 4096, 4096, 1, 1, -4096, 4096
    want = torch.ones(L, dtype=torch.float64)
    want[-1], want[-2], want[-3] = 2.0 ** 24, 2.0 ** 24 + 1, 2.0 ** 24 + 1
    for g in (z(L, 1, 1), z(1)):
        dg = fm.memory_chunk_backward(q, k, k.clone(), g, do, None, torch.ones(1, 1, 1, 1, device=DEV), None, scale=1.0)[3]
        exact = want.view(L, 1, 1) if g.dim() == 3 else want.sum().view(1)
        assert torch.equal(dg.cpu(), exact.float())
