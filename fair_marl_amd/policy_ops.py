"""The policy's operators on the device: what a recurrent policy computes on the fields of the rollout buffer.

* ``memory_chunk`` / ``memory_step``: linear attention with a decay per head -- the policy's memory.  Where the reference runs a GRU over
  ``rnn_states`` and ``masks`` (onpolicy/algorithms/utils/rnn.py:26-84: one step in the rollout, chunks of ``data_chunk_length`` with the
  episodes' ends inside in the update), these carry a matrix per head through the same slots.
* ``block_norm``: the end of a residual block and the start of the next in one pass -- norm of the branch, gate, residual scale, residual, norm.
* ``action_log_probs``: log-probability and entropy of the taken actions straight from the features (the reference's ``ACTLayer.evaluate_actions``,
  onpolicy/algorithms/utils/act.py:120-177), for the env's five actions as for the joint actions of several agents; no logits are kept.

All run on the current stream of their tensors' device, take any strides as long as the last axis is contiguous (a tensor whose last axis is
not is copied), read nothing back and are capturable in a graph.  Gradients come through torch.autograd; ``memory_chunk_backward`` is the
same gradient as a plain call, for a step that is captured without an autograd graph.  There is no CPU form: tensors off the GPU are refused.  So are
forward-mode tangents, and calls under a tracer (torch.jit.trace, make_fx), which would keep nothing of them; torch.compile runs them between its graphs.
"""
import ctypes as C
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.T_F32, torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16}
_F32 = torch.float32
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)   # (2 us less per call than torch.cuda.current_stream(..).cuda_stream)


# A call's host time is most of a small call's: arguments are checked by plain conditions, messages are formed only when one fails.
def _refuse(text, *args):
    raise ValueError(text % args if args else text)


_tracing, _dispatch_mode, _PROXY, _compiling = torch._C._get_tracing_state, torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY, torch.compiler.is_compiling


def _seen_by_torch(op, *tensors):
    """Refuses a call whose kernels torch would have to know of: one that it records, one that it forms a tangent of (it sees new, unwritten tensors only)."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _refuse('%s: no forward-mode derivative', op)
    if _tracing() is not None or _dispatch_mode(_PROXY) is not None:
        _refuse('%s: cannot be traced', op)


def _uncompiled(op):
    """op as torch.compile has to call it: as it is, between two graphs (what it does with the C-ABI's structures is not what a compiler takes it for)."""
    @functools.wraps(op)
    def call(*args, **kwargs):
        return (torch.compiler.disable(op) if _compiling() else op)(*args, **kwargs)
    return call


def _same_device(op, first, *rest):
    if not first.is_cuda:
        _refuse('%s: tensors must be on a GPU, got one on %s', op, first.device)
    dev = first.get_device()
    for t in rest:
        if t is not None and t.get_device() != dev:
            _refuse('%s: all tensors must be on %s, got one on %s', op, first.device, t.device)


def _once(backward):
    """once_differentiable, without its context manager where no second gradient is asked for."""
    guarded = once_differentiable(backward)
    return staticmethod(lambda ctx, *grads: guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads))


def _last(t):
    """t with a contiguous last axis."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _flat(t, n):
    """t as rows of n, the last axis contiguous."""
    return t if t.dim() == 2 and t.stride(1) == 1 else _last(t.reshape(-1, n))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _run(entry, dev, *args):
    """One call of the C-ABI on the current stream of the device with that number."""
    call = getattr(_lib.load(), entry)
    if torch.cuda.current_device() == dev:
        rc = call(*args, _raw_stream(dev) if _raw_stream else torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = call(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        _lib.check(rc, entry)


def _workspace(like, nbytes):
    return like.new_empty(nbytes, dtype=torch.uint8)


def _rows(t):
    """FmarlRows of a (L, B, H, d) or (B, H, d) tensor."""
    s = t.stride()
    return _lib.FmarlRows(t.data_ptr(), s[0] if len(s) == 4 else 0, s[-3], s[-2])


# ---- memory ---------------------------------------------------------------------------------------------------------------------
def _memory_args(op, q, k, v, log_decay, state, masks, scale, lead):
    """The checked, laid out arguments: (FmarlMemory, tensors to keep)."""
    _same_device(op, q, k, v, log_decay, state, masks)
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        _refuse('%s: q, k and v must be of one type out of float32, bfloat16, float16, got %s, %s, %s', op, q.dtype, k.dtype, v.dtype)
    shape, vshape = q.shape, v.shape
    if len(shape) != lead + 2 or k.shape != shape or len(vshape) != lead + 2 or vshape[:-1] != shape[:-1]:
        _refuse('%s: q and k (%sB, H, dk), v (%sB, H, dv), got %s, %s, %s', op, 'L, ' * (lead - 1), 'L, ' * (lead - 1), tuple(shape), tuple(k.shape), tuple(vshape))
    B, H, dk = shape[-3:]
    L, dv = shape[0] if lead == 2 else 1, vshape[-1]
    if log_decay.dtype != _F32 or log_decay.shape != (shape[:-1] if log_decay.dim() != 1 else (H,)):
        _refuse('%s: log_decay must be float32 (H,) or %s, got %s %s', op, tuple(shape[:-1]), log_decay.dtype, tuple(log_decay.shape))
    if masks is not None:
        if masks.numel() != L * B:
            _refuse('%s: masks must hold %d entries, got %s', op, L * B, tuple(masks.shape))
        if masks.dtype != _F32:
            masks = masks.to(_F32)
        masks = masks.reshape(B) if lead == 1 else masks.reshape(L, B)
    if state is not None:
        if state.dtype != _F32 or state.numel() != B * H * dk * dv:
            _refuse('%s: state must be float32 with B H dk dv = %d entries, got %s %s', op, B * H * dk * dv, state.dtype, tuple(state.shape))
        state = state.contiguous()
    keep = (_last(q), _last(k), _last(v), log_decay, state, masks)
    return _memory_struct(*keep, dk ** -0.5 if scale is None else float(scale)), keep


def _memory_struct(q, k, v, g, state, masks, scale):
    """FmarlMemory of checked, laid out tensors: masks (L, B) or (B)."""
    shape, gs = q.shape, g.stride()
    token, ms = len(gs) != 1, (0, 0) if masks is None else masks.stride()
    return _lib.FmarlMemory(shape[0] if len(shape) == 4 else 1, shape[-3], shape[-2], shape[-1], v.shape[-1], _DTYPES[q.dtype], scale, 0 if token else 1, _rows(q), _rows(k), _rows(v),
                            g.data_ptr(), gs[0] if len(gs) == 3 else 0, gs[-2] if token else 0, gs[-1], _ptr(masks), ms[0] if len(ms) == 2 else 0, ms[-1], _ptr(state))


def _launch_chunk(m, keep):
    v = keep[2]
    out, state = v.new_empty(v.shape), v.new_empty((m.B, m.H, m.dk, m.dv), dtype=_F32)
    ws = _workspace(v, _lib.load().fmarl_memory_workspace(m, 0))
    _run('fmarl_memory_chunk', v.get_device(), m, _rows(out), state.data_ptr(), ws.data_ptr())
    return out, state, ws


def _launch_chunk_backward(m, keep, d_out, d_state, want_decay=True, forward_ws=None):
    q, k, v, g, state = keep[:5]
    d_out = _last(d_out)
    if d_state is not None:
        d_state = d_state.contiguous()
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    dg = g.new_empty(g.shape) if want_decay else None
    ds = g.new_empty((m.B, m.H, m.dk, m.dv))
    ws = _workspace(v, _lib.load().fmarl_memory_workspace(m, 1))
    _run('fmarl_memory_chunk_backward', v.get_device(), m, _rows(d_out), _ptr(d_state), _rows(dq), _rows(dk), _rows(dv), _ptr(dg), ds.data_ptr(), _ptr(forward_ws),
         ws.data_ptr())
    return dq, dk, dv, dg, ds


def _no_tokens(v, state, shape):
    return v.new_empty(v.shape), v.new_zeros(shape, dtype=_F32) if state is None else state.reshape(shape).clone()


class _MemoryChunk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, masks, scale):
        m, keep = _memory_args('memory_chunk', q, k, v, log_decay, state, masks, scale, 2)
        if m.L == 0 or m.B == 0:
            out, last, ws = _no_tokens(v, state, (m.B, m.H, m.dk, m.dv)) + (v.new_empty(0),)
        else:
            out, last, ws = _launch_chunk(m, keep)
        ctx.save_for_backward(*keep, ws if ws.numel() > 256 else None)   # long sequences: the states at their segments' starts
        ctx.scale, ctx.state_shape = m.scale, None if state is None else state.shape
        ctx.set_materialize_grads(False)
        return out, last

    @_once
    def backward(ctx, d_out, d_state):
        *keep, ws = ctx.saved_tensors
        v, state = keep[2], keep[4]
        m = _memory_struct(*keep, ctx.scale)
        if m.L == 0 or m.B == 0:
            ds = None if state is None else torch.zeros_like(state) if d_state is None else d_state.clone()
            return (*(torch.zeros_like(t) for t in keep[:4]), None if ds is None else ds.reshape(ctx.state_shape), None, None)
        if d_out is None:
            d_out = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        dq, dk, dv, dg, ds = _launch_chunk_backward(m, keep, d_out, d_state, ctx.needs_input_grad[3], ws)
        return dq, dk, dv, dg, None if state is None else ds.view(ctx.state_shape), None, None


@_uncompiled
def memory_chunk(q, k, v, log_decay, state=None, masks=None, scale=None):
    """Linear attention with a decay per head over L tokens of B sequences: ``(out, last_state)``.

        S_t = r_t exp(log_decay_t) S_{t-1} + k_t^T v_t,    out_t = scale q_t S_t,    r_t = 0 where masks_t == 0, else 1

    q, k (L, B, H, dk), v (L, B, H, dv) of one type (float32, bfloat16, float16), 1 <= dk, dv <= 128; out has v's type.  log_decay float32: (H,)
    or one per token, (L, B, H); below -128 (-inf, a type's lowest value) it forgets everything.  state: what the sequences bring, float32 with B H dk dv entries in any shape
    (the generator's ``rnn_states`` rows), None for zeros; the last state comes back as (B, H, dk, dv).  masks: L B entries as the
    generator's ``masks`` (0: an episode starts at the token).  scale: dk ** -0.5 if None.  Rows ordered (L, chunk) as ``recurrent_generator``
    yields them are this layout: ``q.view(L, chunks, H, dk)``.  States, decays and all sums are float32 (the decays' prefix sums float64).
    Differentiable in q, k, v, log_decay and state, once."""
    _seen_by_torch('memory_chunk', q, k, v, log_decay, state)
    if q.dim() != 4 or v.dim() != 4:
        _refuse('memory_chunk: q, k (L, B, H, dk) and v (L, B, H, dv), got %s, %s', tuple(q.shape), tuple(v.shape))
    if not _wants_grad(q, k, v, log_decay, state):
        m, keep = _memory_args('memory_chunk', q, k, v, log_decay, state, masks, scale, 2)
        if m.L == 0 or m.B == 0:
            return _no_tokens(v, state, (m.B, m.H, m.dk, m.dv))
        return _launch_chunk(m, keep)[:2]
    return _MemoryChunk.apply(q, k, v, log_decay, state, masks, scale)


@_uncompiled
def memory_chunk_backward(q, k, v, log_decay, d_out, d_state=None, state=None, masks=None, scale=None):
    """The gradients of ``memory_chunk`` as a plain call: (dq, dk, dv, d_log_decay, d_state0) from d_out (L, B, H, dv) and the gradient of the last
    state (None: zeros)."""
    _seen_by_torch('memory_chunk_backward', q, k, v, log_decay, d_out, d_state, state)
    m, keep = _memory_args('memory_chunk_backward', q, k, v, log_decay, state, masks, scale, 2)
    if m.L == 0 or m.B == 0:
        _refuse('memory_chunk_backward: no tokens')
    _same_device('memory_chunk_backward', q, d_out, d_state)
    if d_out.shape != v.shape or d_out.dtype != v.dtype:
        _refuse('memory_chunk_backward: d_out must be %s %s, got %s %s', tuple(v.shape), v.dtype, tuple(d_out.shape), d_out.dtype)
    if d_state is not None and (d_state.dtype != _F32 or d_state.numel() != m.B * m.H * m.dk * m.dv):
        _refuse('memory_chunk_backward: d_state must be float32 (B, H, dk, dv), got %s %s', d_state.dtype, tuple(d_state.shape))
    return _launch_chunk_backward(m, keep, d_out, d_state)


@_uncompiled
def memory_step(q, k, v, log_decay, state, masks=None, scale=None, out_state=None):
    """``memory_chunk`` for one token per sequence, as an env step of the rollout takes it: ``(out, out_state)``.  q, k (B, H, dk), v (B, H, dv), log_decay
    (H,) or (B, H), masks B entries, state None or float32 with B H dk dv entries.  out_state: where the new state goes (float32, contiguous; the buffer's next slot, or ``state``
    itself), a new (B, H, dk, dv) tensor if None; to autograd it is written in place.  No gradient: refused where one would be recorded."""
    _seen_by_torch('memory_step', q, k, v, log_decay, state)
    if _wants_grad(q, k, v, log_decay, state):
        _refuse('memory_step records no gradient: call it under torch.no_grad(), or use memory_chunk')
    m, keep = _memory_args('memory_step', q, k, v, log_decay, state, masks, scale, 1)
    n = m.B * m.H * m.dk * m.dv
    given = out_state is not None
    if not given:
        out_state = v.new_empty((m.B, m.H, m.dk, m.dv), dtype=_F32)
    else:
        if out_state.device != q.device or out_state.dtype != _F32 or out_state.numel() != n or not out_state.is_contiguous():
            _refuse('memory_step: out_state must be contiguous float32 with %d entries on %s', n, q.device)
        if keep[4] is not None:
            gap = abs(out_state.data_ptr() - m.state) if n else 0
            if gap and gap < 4 * n:
                _refuse('memory_step: out_state overlaps state without being it')
    out = v.new_empty(v.shape)
    _run('fmarl_memory_step', q.get_device(), m, _rows(out), out_state.data_ptr())
    if given:
        torch.autograd.graph.increment_version(out_state)   # written behind autograd's back: a graph that keeps what it held has to see that
    return out, out_state


# ---- block_norm -----------------------------------------------------------------------------------------------------------------
_WEIGHTS = ('scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')


def _block_args(x, branch, gate, weights, groups, layer, silu, post_norm, pre_norm, eps):
    """(FmarlBlock, the tensors it points into, which have to live until the launch)."""
    _same_device('block_norm', x, branch, gate, *weights)
    shape, D = x.shape, x.shape[-1]
    dtype = x.dtype if branch is None else branch.dtype
    if dtype not in _DTYPES or (x.dtype != dtype and x.dtype != _F32):
        _refuse('block_norm: float32, bfloat16 or float16; x of the branch\'s type or float32, got %s, %s', x.dtype, dtype)
    if branch is not None and branch.shape != shape:
        _refuse('block_norm: branch must be %s, got %s', tuple(shape), tuple(branch.shape))
    if gate is not None and (gate.shape != shape or gate.dtype != dtype):
        _refuse('block_norm: gate must be %s %s, got %s %s', tuple(shape), dtype, tuple(gate.shape), gate.dtype)
    for name, w in zip(_WEIGHTS, weights):
        if w is not None and (w.dtype != _F32 or w.shape != (D,)):
            _refuse('block_norm: %s must be float32 (%d,), got %s %s', name, D, w.dtype, tuple(w.shape))
    return _block_struct(x, branch, gate, weights, groups, layer, silu, post_norm, pre_norm, eps)


def _block_struct(x, branch, gate, weights, groups, layer, silu, post_norm, pre_norm, eps):
    """The same of checked tensors."""
    D, dtype = x.shape[-1], x.dtype if branch is None else branch.dtype
    x2, b2, g2 = _flat(x, D), None if branch is None else _flat(branch, D), None if gate is None else _flat(gate, D)
    ws = [None if w is None else w.contiguous() for w in weights]
    b = _lib.FmarlBlock(x2.shape[0], D, groups, _DTYPES[dtype], _DTYPES[x.dtype], layer, silu, post_norm, pre_norm, eps, 0, x2.data_ptr(), x2.stride(0), _ptr(b2),
                        0 if b2 is None else b2.stride(0), _ptr(g2), 0 if g2 is None else g2.stride(0), *[None if w is None else w.data_ptr() for w in ws])
    return b, (x2, b2, g2, ws)


def _launch_block(x, branch, gate, weights, options):
    b, keep = _block_args(x, branch, gate, weights, *options)
    y = None if branch is None else x.new_empty(x.shape)
    h = (x if branch is None else branch).new_empty(x.shape) if options[4] else None
    _run('fmarl_block_norm', x.get_device(), b, _ptr(y), _ptr(h))
    return y, h


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, options):
        weights = (scale, post_weight, post_bias, pre_weight, pre_bias)
        out = _launch_block(x, branch, gate, weights, options)
        ctx.save_for_backward(x, branch, gate, *weights)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return out

    @_once
    def backward(ctx, dy, dh):
        x, branch, gate, *weights = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 9
        need = ctx.needs_input_grad
        b, keep = _block_struct(x, branch, gate, weights, *ctx.options)
        D = b.dim
        dy, dh = None if dy is None else _flat(dy, D), None if dh is None else _flat(dh, D)
        dx = x.new_empty(x.shape)
        dbranch = None if branch is None else branch.new_empty(x.shape)
        dgate = None if gate is None else gate.new_empty(x.shape)
        dw = [w.new_empty(D) if w is not None and n else None for w, n in zip(weights, need[3:8])]
        ws = _workspace(x, _lib.load().fmarl_block_norm_workspace(b))
        _run('fmarl_block_norm_backward', x.get_device(), b, _ptr(dy), 0 if dy is None else dy.stride(0), _ptr(dh), 0 if dh is None else dh.stride(0), dx.data_ptr(),
             _ptr(dbranch), _ptr(dgate), (C.c_void_p * 5)(*[_ptr(t) for t in dw]), ws.data_ptr())
        return (dx, dbranch, dgate, *dw, None)


@_uncompiled
def block_norm(x, branch=None, gate=None, scale=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, groups=1, kind='rms',
               gate_act='sigmoid', post_norm=True, pre_norm=True, eps=1e-5):
    """The end of a residual block and the start of the next one in one pass: ``(y, h)``.

        u = n_groups(branch) post_weight + post_bias,   y = x + scale u act(gate),   h = n(y) pre_weight + pre_bias

    over the last axis of x (..., D), D <= 8192; n is ``'rms'`` (a / sqrt(mean a^2 + eps)) or ``'layer'`` (LayerNorm, what the reference's MLPs use:
    onpolicy/algorithms/utils/mlp.py:25-40); ``groups`` equal runs of the branch's columns (its heads) are normed by themselves.  branch and gate: x's
    shape, of one type; x has that type or is float32 (a residual stream kept wide); y has x's type, h the branch's.  scale, weights and
    biases: float32 (D,).  Whatever is None is left out (factor 1, bias 0).  Without a branch y is x and h = n(x) pre_weight + pre_bias: the first
    block's start; ``post_norm=False`` takes the branch as it is, ``pre_norm=False`` returns h = None: the last block's end.  h is formed from y before its
    rounding.  Differentiable in all tensors, once; nothing but the inputs is kept for the backward pass."""
    weights = (scale, post_weight, post_bias, pre_weight, pre_bias)
    _seen_by_torch('block_norm', x, branch, gate, *weights)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        _refuse('block_norm: the last axis must hold 1..8192 elements, got %s', tuple(x.shape))
    if not isinstance(groups, int) or not 1 <= groups <= 256 or x.shape[-1] % groups:
        _refuse('block_norm: groups must lie in 1..256 and divide %d, got %r', x.shape[-1], groups)
    if kind not in ('rms', 'layer'):
        _refuse('block_norm: kind must be rms or layer, got %r', kind)
    if gate_act not in ('sigmoid', 'silu'):
        _refuse('block_norm: gate_act must be sigmoid or silu, got %r', gate_act)
    if branch is None and not (gate is None and scale is None and post_weight is None and post_bias is None):
        _refuse('block_norm: gate, scale and post weights need a branch')
    if not post_norm and not (post_weight is None and post_bias is None):
        _refuse('block_norm: post weights need post_norm')
    if not pre_norm and not (pre_weight is None and pre_bias is None):
        _refuse('block_norm: pre weights need pre_norm')
    if branch is None and not pre_norm:
        _refuse('block_norm: without a branch and without pre_norm there is nothing to do')
    if not eps >= 0:
        _refuse('block_norm: eps must not be negative, got %r', eps)
    options = (groups, int(kind == 'layer'), int(gate_act == 'silu'), int(bool(post_norm)), int(bool(pre_norm)), eps)
    if _wants_grad(x, branch, gate, *weights):
        y, h = _BlockNorm.apply(x, branch, gate, *weights, options)
    else:
        y, h = _launch_block(x, branch, gate, weights, options)
    return (x if branch is None else y), h


# ---- action_log_probs -----------------------------------------------------------------------------------------------------------
_ACTION_TYPES = {torch.int64: 0, torch.int32: 1, torch.float32: 2}


def _action_args(features, weight, bias, actions, available):
    """(FmarlActions, the laid out tensors, which have to live until the launch)."""
    _same_device('action_log_probs', features, weight, bias, actions, available)
    V, K = weight.shape
    if features.dtype not in _DTYPES or weight.dtype != features.dtype:
        _refuse('action_log_probs: features and weight must be of one type out of float32, bfloat16, float16, got %s, %s', features.dtype, weight.dtype)
    if bias is not None and bias.shape != (V,):
        _refuse('action_log_probs: bias must be (%d,), got %s', V, tuple(bias.shape))
    M = features.numel() // K
    if actions.dtype not in _ACTION_TYPES or actions.numel() != M:
        _refuse('action_log_probs: actions must be int64, int32 or float32 with %d entries, got %s %s', M, actions.dtype, tuple(actions.shape))
    if available is not None and (available.dtype not in (_F32, torch.bool, torch.uint8) or available.numel() != M * V or available.shape[-1] != V):
        _refuse('action_log_probs: available_actions must be float32, bool or uint8 (..., %d) with %d entries, got %s %s', V, M * V, available.dtype, tuple(available.shape))
    return _action_struct(features, weight, bias, actions, available)


def _action_struct(features, weight, bias, actions, available):
    """The same of checked tensors."""
    V, K = weight.shape
    x, w, actions = _flat(features, K), _last(weight), actions.contiguous()
    M = x.shape[0]
    if bias is not None:
        bias = bias.contiguous()
    kind = stride = 0
    if available is not None:
        available = _last(available.reshape(M, V))
        kind, stride = int(available.dtype != _F32), available.stride(0)
    a = _lib.FmarlActions(M, K, V, _DTYPES[x.dtype], _ACTION_TYPES[actions.dtype], kind, 0, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), _ptr(bias),
                          actions.data_ptr(), _ptr(available), stride)
    return a, (x, w, bias, actions, available)


def _launch_actions(features, weight, bias, actions, available):
    a, keep = _action_args(features, weight, bias, actions, available)
    shape = features.shape[:-1]
    log_probs, entropy, lse = (features.new_empty(shape, dtype=_F32) for _ in range(3))
    ws = _workspace(features, _lib.load().fmarl_action_log_probs_workspace(a, 0))
    _run('fmarl_action_log_probs', features.get_device(), a, log_probs.data_ptr(), entropy.data_ptr(), lse.data_ptr(), ws.data_ptr())
    return log_probs, entropy, lse


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, weight, bias, actions, available):
        log_probs, entropy, lse = _launch_actions(features, weight, bias, actions, available)
        ctx.save_for_backward(features, weight, bias, actions, available, entropy, lse)
        ctx.set_materialize_grads(False)
        return log_probs, entropy

    @_once
    def backward(ctx, d_log_probs, d_entropy):
        features, weight, bias, actions, available, entropy, lse = ctx.saved_tensors
        if d_log_probs is None and d_entropy is None:
            return (None,) * 5
        a, keep = _action_struct(features, weight, bias, actions, available)
        dx, dw = features.new_empty(features.shape), weight.new_empty(weight.shape)
        db = bias.new_empty(bias.shape) if bias is not None and ctx.needs_input_grad[2] else None
        if a.rows == 0:
            return dx, dw.zero_(), None if db is None else db.zero_(), None, None
        dl, de = (None if t is None else t.contiguous() for t in (d_log_probs, d_entropy))
        ws = _workspace(features, _lib.load().fmarl_action_log_probs_workspace(a, 1))
        _run('fmarl_action_log_probs_backward', features.get_device(), a, entropy.data_ptr(), lse.data_ptr(), _ptr(dl), _ptr(de), dx.data_ptr(), dw.data_ptr(), _ptr(db),
             ws.data_ptr())
        return dx, dw, db, None, None


@_uncompiled
def action_log_probs(features, weight, bias, actions, available_actions=None):
    """Log-probability and entropy of discrete actions: ``(log_probs, entropy)``, float32, of the features' leading shape.

        z = features weight^T + bias, -inf where available_actions == 0;   log_probs = z_action - lse(z),   entropy = -sum_v p_v log p_v

    features (..., K), weight (V, K) of one type (float32, bfloat16, float16), K <= 16 384, V <= 1 048 576; bias (V,) float32 or the weight's type, or None; actions:
    one per row, int64, int32 or float32 (the buffer's ``actions``; a trailing 1 is fine); available_actions: (..., V) float32, bool or uint8, or None.  A row with a
    negative action (padding) or nothing available takes no part: 0, 0 and no gradient.  An unavailable action has log-probability
    -inf, one that does not exist (>= V) NaN (and no gradient).  The logits are never stored: for many actions the softmax runs over pieces of them, and they
    are formed again for the gradient, with the row's log-sum in float32: logits in the thousands cost the gradient's probabilities their last digits (2^-24 of the logit).
    Differentiable in features, weight and bias, once.  Half precision operands: products are exact, sums float32; with many actions the gradient's dz is rounded to the operands'
    type before its two products (the gradients' error is 1.4 times that of their own rounding)."""
    _seen_by_torch('action_log_probs', features, weight, bias)
    if weight.dim() != 2 or features.dim() < 1 or features.shape[-1] != weight.shape[1] or not 1 <= weight.shape[1] <= 16384 or not 1 <= weight.shape[0] <= 1 << 20:
        _refuse('action_log_probs: features (..., K) and weight (V, K) with K in 1..16384, V in 1..1048576, got %s, %s', tuple(features.shape), tuple(weight.shape))
    if bias is not None and bias.dtype != _F32:
        if bias.dtype != weight.dtype:
            _refuse('action_log_probs: bias must be float32 or of the weight\'s type, got %s', bias.dtype)
        bias = bias.float()
    if not _wants_grad(features, weight, bias):
        return _launch_actions(features, weight, bias, actions, available_actions)[:2]
    return _ActionLogProbs.apply(features, weight, bias, actions, available_actions)
