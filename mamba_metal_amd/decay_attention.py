"""Linear attention with a decay for each head, over long sequences and token by token.

    S_t = exp(g_t) S_{t-1} + k_t v_t^T          y_t = scale S_t^T q_t

``decay_attention`` runs it over (batch, seqlen, heads) and is differentiable; ``decay_attention_step`` is its single
token.  It stands beside ``selective_scan`` and ``gated_scan``, whose states belong to a channel; here a head has a
(key_dim, value_dim) state, and neighbouring heads may share their q and k.  States and sums are float32 for every dtype.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from mamba_metal_amd import _lib
from mamba_metal_amd.act8 import channels_last

MAX_KEY_DIM = 128     # MM_DECAY_MAX_KEY_DIM
MAX_VALUE_DIM = 1024  # MM_DECAY_MAX_VALUE_DIM
_two, _three = _lib._i64a2, _lib._i64a3


# What a call's sizes and strides are to the library, whose conversions cost a microsecond and more each.
@functools.lru_cache(maxsize=4096)
def _strides(stride):
    """The first three of a tensor's strides; of the decays of heads (1-d), the heads' alone."""
    return _three(0, 0, *stride) if len(stride) == 1 else _three(*stride[:3])


@functools.lru_cache(maxsize=4096)
def _step_strides(stride):
    """The same of the token step's: batch and head."""
    return _two(0, *stride) if len(stride) == 1 else _two(*stride[:2])


@functools.lru_cache(maxsize=1024)
def _bytes(qk_shape, v_shape, dtype):
    """Bytes of the states that are kept, and of the forward and the backward pass's workspaces."""
    (b, n, groups, dk), (heads, dv), lib = qk_shape, v_shape[2:], _lib.load()
    return (lib.mm_decay_attention_states_size(b, n, heads, dk, dv, dtype),
            *(lib.mm_decay_attention_workspace_size(b, n, heads, groups, dk, dv, dtype, back) for back in (0, 1)))


def _empty_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _params(q, k, v, g, lengths, scale, qk_shape, v_shape):
    p = _lib.DecayAttentionParams()
    p.batch, p.seqlen, p.groups, p.key_dim = qk_shape
    p.heads, p.value_dim = v_shape[2:]
    p.q, p.q_stride = q.data_ptr(), _strides(q.stride())
    p.k, p.k_stride = k.data_ptr(), _strides(k.stride())
    p.v, p.v_stride = v.data_ptr(), _strides(v.stride())
    p.log_decay, p.log_decay_stride = g.data_ptr(), _strides(g.stride())
    if lengths is not None:
        p.lengths = lengths.data_ptr()
        p.lengths_dtype = 1 if lengths.dtype == torch.int64 else 0
    p.scale = scale
    p.dtype, p.log_decay_dtype = _lib.dtype_code(q.dtype), _lib.dtype_code(g.dtype)
    return p


def _call(name, p, nbytes, dev):
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    with _lib.on_device(dev):
        st = getattr(_lib.load(), name)(p, _lib.stream_of(dev))
    _lib.check(st, name)


def _forward(dev, q, k, v, g, h0, lengths, scale, want_state, train):
    """y, the final state (or None) and, for training, the states before each run of tokens."""
    qk_shape, v_shape = q.shape, v.shape
    p = _params(q, k, v, g, lengths, scale, qk_shape, v_shape)
    states_bytes, workspace, _ = _bytes(qk_shape, v_shape, p.dtype)
    y = _empty_like(v)
    p.y = y.data_ptr()
    state = states = None
    if h0 is not None:
        p.h0 = h0.data_ptr()
    if want_state:
        state = torch.empty((v_shape[0], v_shape[2], qk_shape[3], v_shape[3]), dtype=torch.float32, device=dev)
        p.state_out = state.data_ptr()
    if train:
        states = torch.empty(states_bytes, dtype=torch.uint8, device=dev)
        p.run_states = states.data_ptr() or None
    _call("mm_decay_attention_fwd", p, workspace, dev)
    return y, state, states


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dev, q, k, v, g, h0, lengths, scale, want_state):
        y, state, states = _forward(dev, q, k, v, g, h0, lengths, scale, want_state, True)
        ctx.meta = (dev, q.dtype, q.shape, v.shape, g.dtype, g.shape, scale,
                    (None if lengths is None else lengths.dtype,))
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, g, lengths, states)
        return (y, state) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        if dy is None and dstate is None:
            return (None,) * 9
        dev, dtype, qk_shape, v_shape, g_dtype, g_shape, scale, lengths_dtype = ctx.meta
        # (A leaf's memory, type and size may be others than in the forward pass: its data replaced, its storage freed and
        # allocated again.)
        q, k, v, g, lengths, states = _checked(ctx.saved_tensors, dev, dtype, qk_shape, v_shape, g_dtype, g_shape, *lengths_dtype)
        p = _params(q, k, v, g, lengths, scale, qk_shape, v_shape)
        p.run_states = states.data_ptr() or None
        if dy is None:  # only the final state was used
            dy = torch.zeros((1, 1, 1, v_shape[3]), dtype=dtype, device=dev).expand(v_shape)
        elif dy.dtype != dtype or (dy.stride(-1) != 1 and v_shape[3] > 1):
            dy = dy.to(dtype).contiguous()
        p.dy, p.dy_stride = dy.data_ptr(), _strides(dy.stride())
        if dstate is not None:
            dstate = dstate.contiguous()
            p.dstate = dstate.data_ptr()
        dq, dk, dv = _empty_like(q), _empty_like(k), _empty_like(v)
        p.dq, p.dk, p.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        dg = dh0 = None
        if ctx.needs_input_grad[4]:
            dg = (torch.empty if v_shape[0] and v_shape[1] else torch.zeros)(g_shape, dtype=torch.float32, device=dev)
            if len(g_shape) == 1:
                p.dlog_decay_heads = dg.data_ptr()
            else:
                p.dlog_decay = dg.data_ptr() or None
        if ctx.needs_input_grad[5]:
            dh0 = torch.empty((v_shape[0], v_shape[2], qk_shape[3], v_shape[3]), dtype=torch.float32, device=dev)
            p.dh0 = dh0.data_ptr()
        _call("mm_decay_attention_bwd", p, _bytes(qk_shape, v_shape, p.dtype)[2], dev)
        return None, dq, dk, dv, None if dg is None else dg.to(g_dtype), dh0, None, None, None


def _checked(saved, dev, dtype, qk_shape, v_shape, g_dtype, g_shape, lengths_dtype):
    """The saved tensors, which hooks or a new ``.data`` may have changed."""
    q, k, v, g, lengths, states = saved
    if lengths_dtype is not None:
        lengths = _lib.saved(lengths, lengths_dtype, (v_shape[0],), dev)
    q, k = (_lib.saved(t, dtype, qk_shape, dev, rows=True) for t in (q, k))
    v = _lib.saved(v, dtype, v_shape, dev, rows=True)
    g = _lib.saved(g, g_dtype, g_shape, dev, strided=True)
    nbytes = _bytes(qk_shape, v_shape, _lib.dtype_code(dtype))[0]
    return q, k, v, g, lengths, _lib.saved(states, torch.uint8, (nbytes,), dev)


def _check(q, k, v, g, lead, names):
    """q and k (*lead, groups, key_dim), v (*lead, heads, value_dim), g (*lead, heads) or (heads,)."""
    n, qs, vs, gs = len(lead), q.shape, v.shape, g.shape
    if len(qs) != n + 2 or len(vs) != n + 2 or vs[:n] != lead:
        raise ValueError(f"q must be {names[:-1]}, groups, key_dim) and v {names[:-1]}, heads, value_dim), got "
                         f"{tuple(qs)} and {tuple(vs)}")
    if k.shape != qs:
        raise ValueError(f"k is {tuple(k.shape)}, q {tuple(qs)}")
    groups, dk = qs[n:]
    heads, dv = vs[n:]
    if groups < 1 or heads < 1 or heads % groups:
        raise ValueError(f"{heads} heads cannot share {groups} groups of q and k")
    if not 1 <= dk <= MAX_KEY_DIM or not 1 <= dv <= MAX_VALUE_DIM:
        raise ValueError(f"key_dim {dk} must be 1 to {MAX_KEY_DIM}, value_dim {dv} 1 to {MAX_VALUE_DIM}")
    if gs != (heads,) and gs != (*lead, heads):
        raise ValueError(f"log_decay is {tuple(gs)}, expected {(heads,)} or {(*lead, heads)}")
    dtype = q.dtype
    for name, t in (("k", k), ("v", v)):
        if t.dtype != dtype:
            raise TypeError(f"{name} is {t.dtype}, q {dtype}")
    _lib.dtype_code(dtype)
    _lib.dtype_code(g.dtype)
    for name, t in (("q", q), ("k", k), ("v", v)):
        channels_last(t, name)


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *, scale: float = 1.0,
                    h0: torch.Tensor | None = None, lengths: torch.Tensor | None = None, return_state: bool = False):
    """Linear attention with a decay for each head over a batch of sequences (see the module's formulas).

    q, k: (batch, seqlen, groups, key_dim), v: (batch, seqlen, heads, value_dim), of one dtype (float32, float16,
    bfloat16) with unit channel stride, any other strides; head h uses q and k of group h // (heads // groups).
    key_dim up to 128, value_dim up to 1024.  log_decay: (batch, seqlen, heads), or (heads,) for a constant, of any of
    the three dtypes, at most 0 (-inf forgets all before; above 0 the state grows until it overflows).  h0: (batch,
    heads, key_dim, value_dim), the state before the first token, zeros if not given.  lengths: (batch,) int32 or int64
    on the same GPU; tokens from lengths[b] on (clamped to 0 .. seqlen) leave the state alone, have y = 0 and zero
    gradients, whatever their inputs hold.

    Returns y (batch, seqlen, heads, value_dim), contiguous, in v's dtype; with ``return_state`` also the state after
    each sequence's last token, (batch, heads, key_dim, value_dim) float32.

    With 16-bit inputs the scores of a run of 64 tokens and the state that meets q are rounded to 16 bits, once each,
    before their products, and so are their gradients; the state itself is not, nor are, in calls of up to 32768 tokens
    (batch * seqlen * heads), the scores and the states in gradients of q, k and log_decay.  The gradient of a float32
    log_decay beside 16-bit q, k and v is therefore as exact as theirs; a sequence's last bits may change with how many
    share its batch.  In float16 scale * dy has to stay below 65504; a token's scores go through a power of two and may be
    any numbers.  A NaN or an infinity stays in its sequence and head (in its group, for the gradients of q and k); one in
    k or v may also reach the up to 63 tokens before it in its run of 64.

    Gradients flow to q, k, v, log_decay and h0 (once, not twice, and not in forward mode).  For them a call that needs
    any keeps its inputs and, in their dtype, the state before every 64th token.

    To capture a backward pass into a graph, capture the forward pass with it, and let no eager autograd graph of the
    same leaf tensors be alive at that time."""
    if q.dim() != 4:
        raise ValueError(f"q must be (batch, seqlen, groups, key_dim), got {tuple(q.shape)}")
    _check(q, k, v, log_decay, q.shape[:2], "(batch, seqlen)")
    b, n, _, dk = q.shape
    heads, dv = v.shape[2:]
    if h0 is not None:
        if h0.shape != (b, heads, dk, dv):
            raise ValueError(f"h0 is {tuple(h0.shape)}, expected {(b, heads, dk, dv)}")
        if not h0.is_floating_point():
            raise TypeError(f"h0 is {h0.dtype}")
    if lengths is not None:
        if lengths.shape != (b,):
            raise ValueError(f"lengths is {tuple(lengths.shape)}, expected ({b},)")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"lengths is {lengths.dtype}, expected int32 or int64")
    _lib.refuse_transforms("decay_attention", q, k, v, log_decay, h0)
    dev = _lib.require_cuda(q, k, v, log_decay, h0, lengths)
    h0 = None if h0 is None else (h0 if h0.dtype == torch.float32 else h0.float()).contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, h0)):
        return _DecayAttention.apply(dev, q, k, v, log_decay, h0, lengths, float(scale), return_state)
    y, state, *_ = _forward(dev, q, k, v, log_decay, h0, lengths, float(scale), return_state, False)
    return (y, state) if return_state else y


def decay_attention_step(state: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                         *, scale: float = 1.0, state_out: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """One token of every sequence: the new state, and y (batch, heads, value_dim) in v's dtype, which is returned.

    state (batch, heads, key_dim, value_dim) contiguous float32 is updated in place, or left as it is where ``state_out``
    (the same kind of tensor) is given.  q, k: (batch, groups, key_dim), v and ``out``: (batch, heads, value_dim), of one
    dtype with unit channel stride; log_decay (batch, heads) or (heads,).  Not differentiable: a tensor that requires a
    gradient is refused while gradients are on, and one with a tangent always."""
    if q.dim() != 3:
        raise ValueError(f"q must be (batch, groups, key_dim), got {tuple(q.shape)}")
    _check(q, k, v, log_decay, q.shape[:1], "(batch)")
    b, groups, dk = q.shape
    heads, dv = v.shape[1:]
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None and (t.shape != (b, heads, dk, dv) or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 {(b, heads, dk, dv)}")
    if out is not None:
        if out.shape != v.shape:
            raise ValueError(f"out is {tuple(out.shape)}, v {tuple(v.shape)}")
        if out.dtype != v.dtype:
            raise TypeError(f"out is {out.dtype}, v {v.dtype}")
        channels_last(out, "out")
    if torch.is_grad_enabled() and (state.requires_grad or q.requires_grad or k.requires_grad or v.requires_grad
                                    or log_decay.requires_grad or any(t is not None and t.requires_grad for t in (state_out, out))):
        raise RuntimeError("decay_attention_step has no gradient: call it under no_grad or inference_mode, "
                           "or train through decay_attention")
    _lib.refuse_transforms("decay_attention_step", state, q, k, v, log_decay)
    dev = _lib.require_cuda(state, q, k, v, log_decay, state_out, out)
    lib = _lib.load()
    given = out
    if out is None:
        out = _empty_like(v)
    with _lib.on_device(dev):
        st = lib.mm_decay_attention_step(
            state.data_ptr(), state.data_ptr() if state_out is None else state_out.data_ptr(), q.data_ptr(), k.data_ptr(),
            v.data_ptr(), log_decay.data_ptr(), out.data_ptr(), b, heads, groups, dk, dv, _step_strides(q.stride()),
            _step_strides(k.stride()), _step_strides(v.stride()), _step_strides(log_decay.stride()), _step_strides(out.stride()),
            float(scale), _lib.dtype_code(q.dtype), _lib.dtype_code(log_decay.dtype), _lib.stream_of(dev))
    _lib.check(st, "mm_decay_attention_step")
    _lib.wrote(state if state_out is None else state_out)
    _lib.wrote(given)
    return out
