"""The policy's operators on the device: what a recurrent policy computes on the fields of the rollout buffer.

* ``memory_chunk`` / ``memory_step``: linear attention with a decay per head -- the policy's memory.  Where the reference runs a GRU over
  ``rnn_states`` and ``masks`` (onpolicy/algorithms/utils/rnn.py:26-84: one step in the rollout, chunks of ``data_chunk_length`` with the
  episodes' ends inside in the update), these carry a matrix per head through the same slots.
* ``block_norm``: the end of a residual block and the start of the next in one pass -- norm of the branch, gate, residual scale, residual, norm.
* ``action_log_probs``: log-probability and entropy of the taken actions straight from the features (the reference's ``ACTLayer.evaluate_actions``,
  onpolicy/algorithms/utils/act.py:120-177), for the env's five actions as for the joint actions of several agents; no logits are kept.

All run on the current stream of their tensors' device, take any strides as long as the last axis is contiguous (a tensor whose last axis is
not is copied), read nothing back and are capturable in a graph.  Gradients come through torch.autograd; ``memory_chunk_backward`` is the
same gradient as a plain call, for a step that is captured without an autograd graph.  There is no CPU form: tensors off the GPU are refused.
"""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.T_F32, torch.bfloat16: _lib.T_BF16, torch.float16: _lib.T_F16}


def _need(ok, text, *args):
    if not ok:
        raise ValueError(text % args if args else text)


def _same_device(op, first, *rest):
    _need(first.is_cuda, '%s: tensors must be on a GPU, got one on %s', op, first.device)
    for t in rest:
        _need(t is None or t.device == first.device, '%s: all tensors must be on %s', op, first.device)


def _last(t):
    """t with a contiguous last axis."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _rows(t):
    """FmarlRows of a (L, B, H, d) or (B, H, d) tensor."""
    s = t.stride()
    return _lib.FmarlRows(t.data_ptr(), s[0] if len(s) == 4 else 0, s[-3], s[-2])


# ---- memory ---------------------------------------------------------------------------------------------------------------------
def _memory_args(op, q, k, v, log_decay, state, masks, scale, lead):
    """The checked, laid out arguments: (FmarlMemory, tensors to keep)."""
    _same_device(op, q, k, v, log_decay, state, masks)
    _need(q.dtype in _DTYPES and k.dtype == q.dtype and v.dtype == q.dtype, '%s: q, k and v must be of one type out of float32, bfloat16, float16', op)
    _need(q.dim() == lead + 2 and k.shape == q.shape and v.shape[:-1] == q.shape[:-1] and v.dim() == q.dim(),
          '%s: q and k (%sB, H, dk), v (%sB, H, dv), got %s, %s, %s', op, 'L, ' * (lead - 1), 'L, ' * (lead - 1), tuple(q.shape), tuple(k.shape), tuple(v.shape))
    L = q.shape[0] if lead == 2 else 1
    B, H, dk, dv = q.shape[-3], q.shape[-2], q.shape[-1], v.shape[-1]
    _need(log_decay.dtype == torch.float32, '%s: log_decay must be float32', op)
    token = log_decay.dim() != 1
    _need(tuple(log_decay.shape) == (tuple(q.shape[:-1]) if token else (H,)), '%s: log_decay must be (H,) or %s, got %s', op, tuple(q.shape[:-1]),
          tuple(log_decay.shape))
    if masks is not None:
        _need(masks.numel() == L * B, '%s: masks must hold %d entries, got %s', op, L * B, tuple(masks.shape))
        masks = masks.to(torch.float32).reshape(L, B)
    if state is not None:
        _need(state.dtype == torch.float32 and state.numel() == B * H * dk * dv, '%s: state must be float32 with B H dk dv = %d entries, got %s %s', op,
              B * H * dk * dv, state.dtype, tuple(state.shape))
        state = state.contiguous()
    q, k, v = _last(q), _last(k), _last(v)
    gs = log_decay.stride()
    m = _lib.FmarlMemory(L, B, H, dk, dv, _DTYPES[q.dtype], dk ** -0.5 if scale is None else float(scale), 0 if token else 1, _rows(q), _rows(k), _rows(v),
                         log_decay.data_ptr(), gs[0] if len(gs) == 3 else 0, gs[-2] if token else 0, gs[-1], _ptr(masks),
                         masks.stride(0) if masks is not None else 0, masks.stride(1) if masks is not None else 0, _ptr(state))
    return m, (q, k, v, log_decay, state, masks)


def _launch_chunk(m, keep):
    q, v = keep[0], keep[2]
    dev = q.device
    out = torch.empty(v.shape, dtype=v.dtype, device=dev)
    state = torch.empty(m.B, m.H, m.dk, m.dv, dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws = torch.empty(lib.fmarl_memory_workspace(m, 0), dtype=torch.uint8, device=dev)
        _lib.check(lib.fmarl_memory_chunk(m, _rows(out), state.data_ptr(), ws.data_ptr(), _stream(dev)), 'fmarl_memory_chunk')
    return out, state, ws


def _launch_chunk_backward(m, keep, d_out, d_state, want_decay=True, forward_ws=None):
    q, k, v, g, state = keep[:5]
    dev = q.device
    d_out = _last(d_out)
    if d_state is not None:
        d_state = d_state.contiguous()
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
    dg = torch.empty(g.shape, dtype=torch.float32, device=dev) if want_decay else None
    ds = torch.empty(m.B, m.H, m.dk, m.dv, dtype=torch.float32, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        ws = torch.empty(lib.fmarl_memory_workspace(m, 1), dtype=torch.uint8, device=dev)
        _lib.check(lib.fmarl_memory_chunk_backward(m, _rows(d_out), _ptr(d_state), _rows(dq), _rows(dk), _rows(dv), _ptr(dg), ds.data_ptr(), _ptr(forward_ws),
                                                   ws.data_ptr(),
                                                   _stream(dev)), 'fmarl_memory_chunk_backward')
    return dq, dk, dv, dg, ds


class _MemoryChunk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, masks, scale):
        m, keep = _memory_args('memory_chunk', q, k, v, log_decay, state, masks, scale, 2)
        out, last, ws = _launch_chunk(m, keep)
        ctx.save_for_backward(*keep)
        ctx.forward_ws = ws if any(ctx.needs_input_grad) else None   # long sequences: the states at their segments' starts
        ctx.scale, ctx.state_shape = m.scale, None if state is None else state.shape
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_state):
        q, k, v, g, state, masks = ctx.saved_tensors
        m, keep = _memory_args('memory_chunk', q, k, v, g, state, masks, ctx.scale, 2)
        if d_out is None:
            d_out = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        dq, dk, dv, dg, ds = _launch_chunk_backward(m, keep, d_out, d_state, ctx.needs_input_grad[3], ctx.forward_ws)
        return dq, dk, dv, dg, None if state is None else ds.view(ctx.state_shape), None, None


def memory_chunk(q, k, v, log_decay, state=None, masks=None, scale=None):
    """Linear attention with a decay per head over L tokens of B sequences: ``(out, last_state)``.

        S_t = r_t exp(log_decay_t) S_{t-1} + k_t^T v_t,    out_t = scale q_t S_t,    r_t = 0 where masks_t == 0, else 1

    q, k (L, B, H, dk), v (L, B, H, dv) of one type (float32, bfloat16, float16), 1 <= dk, dv <= 128; out has v's type.  log_decay float32: (H,)
    or one per token, (L, B, H); -inf forgets everything.  state: what the sequences bring, float32 with B H dk dv entries in any shape
    (the generator's ``rnn_states`` rows), None for zeros; the last state comes back as (B, H, dk, dv).  masks: L B entries as the
    generator's ``masks`` (0: an episode starts at the token).  scale: dk ** -0.5 if None.  Rows ordered (L, chunk) as ``recurrent_generator``
    yields them are this layout: ``q.view(L, chunks, H, dk)``.  States, decays and all sums are float32 (the decays' prefix sums float64).
    Differentiable in q, k, v, log_decay and state, once."""
    _need(q.dim() == 4 and v.dim() == 4, 'memory_chunk: q, k (L, B, H, dk) and v (L, B, H, dv), got %s, %s', tuple(q.shape), tuple(v.shape))
    if q.shape[0] == 0 or q.shape[1] == 0:
        _memory_args('memory_chunk', q, k, v, log_decay, state, masks, scale, 2)
        shape = (q.shape[1], q.shape[2], q.shape[3], v.shape[3])
        return v.clone(), torch.zeros(shape, dtype=torch.float32, device=q.device) if state is None else state.reshape(shape).clone()
    return _MemoryChunk.apply(q, k, v, log_decay, state, masks, scale)


def memory_chunk_backward(q, k, v, log_decay, d_out, d_state=None, state=None, masks=None, scale=None):
    """The gradients of ``memory_chunk`` as a plain call: (dq, dk, dv, d_log_decay, d_state0) from d_out (L, B, H, dv) and the gradient of the last
    state (None: zeros)."""
    m, keep = _memory_args('memory_chunk_backward', q, k, v, log_decay, state, masks, scale, 2)
    _need(m.L > 0 and m.B > 0, 'memory_chunk_backward: no tokens')
    _same_device('memory_chunk_backward', q, d_out, d_state)
    _need(d_out.shape == v.shape and d_out.dtype == v.dtype, 'memory_chunk_backward: d_out must be %s %s', tuple(v.shape), v.dtype)
    if d_state is not None:
        _need(d_state.dtype == torch.float32 and d_state.numel() == m.B * m.H * m.dk * m.dv, 'memory_chunk_backward: d_state must be float32 (B, H, dk, dv)')
    return _launch_chunk_backward(m, keep, d_out, d_state)


def memory_step(q, k, v, log_decay, state, masks=None, scale=None, out_state=None):
    """``memory_chunk`` for one token per sequence, as an env step of the rollout takes it: ``(out, out_state)``.  q, k (B, H, dk), v (B, H, dv), log_decay
    (H,) or (B, H), masks B entries, state None or float32 with B H dk dv entries.  out_state: where the new state goes (float32, contiguous; the buffer's next slot, or ``state``
    itself), a new (B, H, dk, dv) tensor if None.  No gradient: refused where one would be recorded."""
    _need(not (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, state))),
          'memory_step records no gradient: call it under torch.no_grad(), or use memory_chunk')
    m, keep = _memory_args('memory_step', q, k, v, log_decay, state, masks, scale, 1)
    dev, n = q.device, m.B * m.H * m.dk * m.dv
    if out_state is None:
        out_state = torch.empty(m.B, m.H, m.dk, m.dv, dtype=torch.float32, device=dev)
    else:
        _need(out_state.device == dev and out_state.dtype == torch.float32 and out_state.numel() == n and out_state.is_contiguous(),
              'memory_step: out_state must be contiguous float32 with %d entries on %s', n, dev)
        if keep[4] is not None:
            gap = abs(out_state.data_ptr() - keep[4].data_ptr())
            _need(gap == 0 or gap >= 4 * n, 'memory_step: out_state overlaps state without being it')
    out = torch.empty(v.shape, dtype=v.dtype, device=dev)
    lib = _lib.load()
    with torch.cuda.device(dev):
        _lib.check(lib.fmarl_memory_step(m, _rows(out), out_state.data_ptr(), _stream(dev)), 'fmarl_memory_step')
    return out, out_state


# ---- block_norm -----------------------------------------------------------------------------------------------------------------
_WEIGHTS = ('scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')


def _block_args(x, branch, gate, weights, groups, kind, gate_act, post_norm, pre_norm, eps):
    """(FmarlBlock, 2-d views of x, branch and gate, the float32 weights); what has to live until the launch is in there."""
    _same_device('block_norm', x, branch, gate, *weights)
    D = x.shape[-1] if x.dim() else 0
    dtype = x.dtype if branch is None else branch.dtype
    _need(dtype in _DTYPES and x.dtype in (dtype, torch.float32), 'block_norm: float32, bfloat16 or float16; x of the branch\'s type or float32, got %s, %s',
          x.dtype, dtype)
    for name, t in (('branch', branch), ('gate', gate)):
        _need(t is None or (t.shape == x.shape and t.dtype == dtype), 'block_norm: %s must be %s %s', name, tuple(x.shape), dtype)
    for name, w in zip(_WEIGHTS, weights):
        _need(w is None or (tuple(w.shape) == (D,) and w.dtype == torch.float32), 'block_norm: %s must be float32 (%d,)', name, D)
    _need(kind in ('rms', 'layer'), 'block_norm: kind must be rms or layer, got %r', kind)
    _need(gate_act in ('sigmoid', 'silu'), 'block_norm: gate_act must be sigmoid or silu, got %r', gate_act)
    rows = [None if t is None else _last(t.reshape(-1, D)) for t in (x, branch, gate)]
    weights = [None if w is None else w.contiguous() for w in weights]
    st = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    b = _lib.FmarlBlock(rows[0].shape[0], D, int(groups), _DTYPES[dtype], _DTYPES[x.dtype], int(kind == 'layer'), int(gate_act == 'silu'), int(bool(post_norm)),
                        int(bool(pre_norm)), float(eps), 0, _ptr(rows[0]), st(rows[0]), _ptr(rows[1]), st(rows[1]), _ptr(rows[2]), st(rows[2]),
                        *[_ptr(w) for w in weights])
    return b, rows, weights


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, options):
        weights = (scale, post_weight, post_bias, pre_weight, pre_bias)
        b, rows, weights = _block_args(x, branch, gate, weights, *options)
        dev = x.device
        y = None if branch is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
        h = torch.empty(x.shape, dtype=x.dtype if branch is None else branch.dtype, device=dev) if options[4] else None
        lib = _lib.load()
        with torch.cuda.device(dev):
            _lib.check(lib.fmarl_block_norm(b, _ptr(y), _ptr(h), _stream(dev)), 'fmarl_block_norm')
        ctx.save_for_backward(x, branch, gate, *weights)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh):
        x, branch, gate, *weights = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 9
        need = ctx.needs_input_grad
        b, rows, weights = _block_args(x, branch, gate, weights, *ctx.options)
        dev, D = x.device, x.shape[-1]
        dy, dh = (None if t is None else _last(t.reshape(-1, D)) for t in (dy, dh))
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        dbranch, dgate = (None if t is None else torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (branch, gate))
        dw = [torch.empty(D, dtype=torch.float32, device=dev) if w is not None and n else None for w, n in zip(weights, need[3:8])]
        lib = _lib.load()
        with torch.cuda.device(dev):
            ws = torch.empty(lib.fmarl_block_norm_workspace(b), dtype=torch.uint8, device=dev)
            _lib.check(lib.fmarl_block_norm_backward(b, _ptr(dy), 0 if dy is None else dy.stride(0), _ptr(dh), 0 if dh is None else dh.stride(0), dx.data_ptr(),
                                                     _ptr(dbranch), _ptr(dgate), (C.c_void_p * 5)(*[_ptr(t) for t in dw]), ws.data_ptr(), _stream(dev)),
                       'fmarl_block_norm_backward')
        return (dx, dbranch, dgate, *dw, None)


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
    _need(x.dim() >= 1 and 1 <= x.shape[-1] <= 8192, 'block_norm: the last axis must hold 1..8192 elements, got %s', tuple(x.shape))
    D = x.shape[-1]
    _need(isinstance(groups, int) and 1 <= groups <= 256 and D % groups == 0, 'block_norm: groups must lie in 1..256 and divide %d, got %r', D, groups)
    _need(branch is not None or (gate is None and scale is None and post_weight is None and post_bias is None),
          'block_norm: gate, scale and post weights need a branch')
    _need(post_norm or (post_weight is None and post_bias is None), 'block_norm: post weights need post_norm')
    _need(pre_norm or (pre_weight is None and pre_bias is None), 'block_norm: pre weights need pre_norm')
    _need(branch is not None or pre_norm, 'block_norm: without a branch and without pre_norm there is nothing to do')
    _need(eps >= 0, 'block_norm: eps must not be negative')
    y, h = _BlockNorm.apply(x, branch, gate, scale, post_weight, post_bias, pre_weight, pre_bias, (groups, kind, gate_act, bool(post_norm), bool(pre_norm), eps))
    return (x if branch is None else y), h


# ---- action_log_probs -----------------------------------------------------------------------------------------------------------
_ACTION_TYPES = {torch.int64: 0, torch.int32: 1, torch.float32: 2}


def _action_args(features, weight, bias, actions, available):
    """(FmarlActions, the laid out tensors, which have to live until the launch)."""
    _same_device('action_log_probs', features, weight, bias, actions, available)
    K, V = weight.shape[1], weight.shape[0]
    _need(features.dtype in _DTYPES and weight.dtype == features.dtype, 'action_log_probs: features and weight must be of one type out of float32, bfloat16, float16')
    _need(bias is None or (tuple(bias.shape) == (V,) and bias.dtype == torch.float32), 'action_log_probs: bias must be (%d,)', V)
    x, w = _last(features.reshape(-1, K)), _last(weight)
    M = x.shape[0]
    _need(actions.dtype in _ACTION_TYPES and actions.numel() == M, 'action_log_probs: actions must be int64, int32 or float32 with %d entries, got %s %s', M,
          actions.dtype, tuple(actions.shape))
    actions = actions.reshape(M).contiguous()
    if available is not None:
        _need(available.dtype in (torch.float32, torch.bool, torch.uint8) and available.numel() == M * V and available.shape[-1] == V,
              'action_log_probs: available_actions must be float32, bool or uint8 (..., %d) with %d entries, got %s %s', V, M * V, available.dtype, tuple(available.shape))
        available = _last(available.reshape(M, V))
    if bias is not None:
        bias = bias.contiguous()
    a = _lib.FmarlActions(M, K, V, _DTYPES[x.dtype], _ACTION_TYPES[actions.dtype], int(available is not None and available.dtype != torch.float32), 0, x.data_ptr(),
                          x.stride(0), w.data_ptr(), w.stride(0), _ptr(bias), actions.data_ptr(), _ptr(available), 0 if available is None else available.stride(0))
    return a, (x, w, bias, actions, available)


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, weight, bias, actions, available):
        a, keep = _action_args(features, weight, bias, actions, available)
        dev, shape = features.device, features.shape[:-1]
        log_probs, entropy, lse = (torch.empty(shape, dtype=torch.float32, device=dev) for _ in range(3))
        lib = _lib.load()
        with torch.cuda.device(dev):
            ws = torch.empty(lib.fmarl_action_log_probs_workspace(a, 0), dtype=torch.uint8, device=dev)
            _lib.check(lib.fmarl_action_log_probs(a, log_probs.data_ptr(), entropy.data_ptr(), lse.data_ptr(), ws.data_ptr(), _stream(dev)), 'fmarl_action_log_probs')
        ctx.save_for_backward(features, weight, bias, actions, available, entropy, lse)
        ctx.set_materialize_grads(False)
        return log_probs, entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, d_log_probs, d_entropy):
        features, weight, bias, actions, available, entropy, lse = ctx.saved_tensors
        if d_log_probs is None and d_entropy is None:
            return (None,) * 5
        a, keep = _action_args(features, weight, bias, actions, available)
        dev = features.device
        dx, dw = torch.empty(features.shape, dtype=features.dtype, device=dev), torch.empty(weight.shape, dtype=weight.dtype, device=dev)
        db = torch.empty(bias.shape, dtype=torch.float32, device=dev) if bias is not None and ctx.needs_input_grad[2] else None
        if a.rows == 0:
            return dx, dw.zero_(), None if db is None else db.zero_(), None, None
        dl, de = (None if t is None else t.contiguous() for t in (d_log_probs, d_entropy))
        lib = _lib.load()
        with torch.cuda.device(dev):
            ws = torch.empty(lib.fmarl_action_log_probs_workspace(a, 1), dtype=torch.uint8, device=dev)
            _lib.check(lib.fmarl_action_log_probs_backward(a, entropy.data_ptr(), lse.data_ptr(), _ptr(dl), _ptr(de), dx.data_ptr(), dw.data_ptr(), _ptr(db), ws.data_ptr(),
                                                           _stream(dev)), 'fmarl_action_log_probs_backward')
        return dx, dw, db, None, None


def action_log_probs(features, weight, bias, actions, available_actions=None):
    """Log-probability and entropy of discrete actions: ``(log_probs, entropy)``, float32, of the features' leading shape.

        z = features weight^T + bias, -inf where available_actions == 0;   log_probs = z_action - lse(z),   entropy = -sum_v p_v log p_v

    features (..., K), weight (V, K) of one type (float32, bfloat16, float16), K <= 16 384, V <= 1 048 576; bias (V,) float32 or the weight's type, or None; actions:
    one per row, int64, int32 or float32 (the buffer's ``actions``; a trailing 1 is fine); available_actions: (..., V) float32, bool or uint8, or None.  A row with a
    negative action (padding) or nothing available takes no part: 0, 0 and no gradient.  An unavailable action has log-probability
    -inf, one that does not exist (>= V) NaN (and no gradient).  The logits are never stored: for many actions the softmax runs over pieces of them, and they
    are formed again for the gradient.  Differentiable in features, weight and bias, once.  Half precision operands: products are exact, sums float32; the
    gradient's dz is rounded to the operands' type before its two products."""
    _need(weight.dim() == 2 and features.dim() >= 1 and features.shape[-1] == weight.shape[1] and 1 <= weight.shape[1] <= 16384 and 1 <= weight.shape[0] <= 1 << 20,
          'action_log_probs: features (..., K) and weight (V, K) with K in 1..16384, V in 1..1048576, got %s, %s', tuple(features.shape), tuple(weight.shape))
    if bias is not None and bias.dtype != torch.float32:
        _need(bias.dtype == weight.dtype, 'action_log_probs: bias must be float32 or of the weight\'s type')
        bias = bias.float()
    return _ActionLogProbs.apply(features, weight, bias, actions, available_actions)
