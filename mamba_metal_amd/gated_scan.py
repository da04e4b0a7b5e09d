"""Gated linear recurrence with one state a channel, over long sequences and token by token.

    r = sigmoid(a_gate)    i = sigmoid(x_gate)    a = exp(A[d] r)
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) i_t x_t           y = h (silu(z) where there is a z)

``gated_scan`` runs it over (batch, seqlen, dim) and is differentiable; ``gated_scan_step`` is its
single token.  It stands beside ``selective_scan``, whose channels have dstate states each and whose
input carries no gate.  Arithmetic and states are float32 for every dtype.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from mamba_metal_amd import _lib
from mamba_metal_amd.act8 import BLOCK, Act8, channels_last, empty_like
from mamba_metal_amd.selective_scan import _status_word

CHECKPOINTS = ("full", "int8")
_INPUTS = ("x", "a_gate", "x_gate", "z")


def _strides2(t):
    s = t.stride()
    return (_lib._i64a2)(s[0], s[1])


def _params(tensors, A, h0, lengths, dtype, shape, dev) -> _lib.GatedScanParams:
    p = _lib.GatedScanParams()
    for name, t in zip(_INPUTS, tensors):
        if t is not None:
            setattr(p, name, t.data_ptr())
            setattr(p, f"{name}_stride", _strides2(t))
    p.A, p.h0, p.lengths = A.data_ptr(), _lib.ptr(h0), _lib.ptr(lengths)
    p.batch, p.seqlen, p.dim = shape
    p.dtype = _lib.dtype_code(dtype)
    p.lengths_dtype = 1 if lengths is not None and lengths.dtype == torch.int64 else 0
    p.status = _status_word(dev).data_ptr()
    return p


def _set_codes(p, packed):
    for k, c in enumerate(packed):
        p.codes[k], p.exps[k] = c.codes.data_ptr(), c.exps.data_ptr()


def _call(name, p, backward, dev):
    lib = _lib.load()
    nbytes = lib.mm_gated_scan_workspace_size(p.batch, p.seqlen, p.dim, backward)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    p.workspace, p.workspace_bytes = _lib.ptr(ws), nbytes
    with _lib.on_device(dev):
        st = getattr(lib, name)(ctypes.byref(p), _lib.stream_of(dev))
    _lib.check(st, name)


def _forward(x, a_gate, x_gate, A, z, h0, lengths, want_state, train, checkpoint):
    """y, the final state (or None) and, for training, the block states and the inputs' 8-bit codes."""
    dev = _lib.require_cuda(x, a_gate, x_gate, A, z, h0, lengths)
    b, n, d = x.shape
    p = _params((x, a_gate, x_gate, z), A, h0, lengths, x.dtype, x.shape, dev)
    y = torch.empty((b, n, d), dtype=x.dtype, device=dev)
    p.y, p.y_stride = y.data_ptr(), _strides2(y)
    f32 = {"dtype": torch.float32, "device": dev}
    state = torch.empty((b, d), **f32) if want_state else None
    p.state_out = _lib.ptr(state)
    blocks, packed = None, []
    if train:
        blocks = torch.empty((b, -(-n // BLOCK), d), **f32)
        p.block_states = blocks.data_ptr()
        if checkpoint == "int8":
            packed = [empty_like(t) for t in (x, a_gate, x_gate, z) if t is not None]
            _set_codes(p, packed)
    _call("mm_gated_scan_fwd", p, 0, dev)
    return y, state, blocks, packed


def _backward(tensors, packed, A, lengths, blocks, dtype, shape, gated, dy, dstate, want_dh0):
    dev = blocks.device
    b, n, d = shape
    p = _params(tensors, A, None, lengths, dtype, shape, dev)
    p.block_states = blocks.data_ptr()
    _set_codes(p, packed)
    p.z_present = 1 if gated else 0
    if dy is None:  # only the final state was used
        dy = torch.zeros((1, 1, d), dtype=dtype, device=dev).expand(b, n, d)
    elif dy.dtype != dtype or (dy.stride(-1) != 1 and d > 1):
        dy = dy.to(dtype).contiguous()
    p.dy, p.dy_stride = dy.data_ptr(), _strides2(dy)
    if dstate is not None:
        dstate = dstate.contiguous()
        p.dstate = dstate.data_ptr()
    grads = [torch.empty((b, n, d), dtype=dtype, device=dev) if k < 3 or gated else None for k in range(4)]
    p.dx, p.da_gate, p.dx_gate, p.dz = (_lib.ptr(t) for t in grads)
    dA = (torch.empty if b else torch.zeros)((d,), dtype=torch.float32, device=dev)
    dh0 = torch.empty((b, d), dtype=torch.float32, device=dev) if want_dh0 else None
    p.dA, p.dh0 = dA.data_ptr(), _lib.ptr(dh0)
    _call("mm_gated_scan_bwd", p, 1, dev)
    return grads, dA, dh0


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a_gate, x_gate, A, z, h0, lengths, checkpoint):
        y, state, blocks, packed = _forward(x, a_gate, x_gate, A, z, h0, lengths, True, True, checkpoint)
        ctx.meta = (x.dtype, x.shape, z is not None, len(packed))
        ctx.set_materialize_grads(False)
        kept = [t for c in packed for t in (c.codes, c.exps)] if packed else [x, a_gate, x_gate, z]
        ctx.save_for_backward(A, lengths, blocks, *kept)
        return y, state

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate):
        if dy is None and dstate is None:
            return (None,) * 8
        dtype, shape, gated, npacked = ctx.meta
        A, lengths, blocks, *kept = ctx.saved_tensors
        if npacked:
            packed = [Act8(kept[2 * k], kept[2 * k + 1], shape, dtype) for k in range(npacked)]
            tensors = ()
        else:
            packed, tensors = (), kept
        (dx, da, dg, dz), dA, dh0 = _backward(tensors, packed, A, lengths, blocks, dtype, shape, gated, dy, dstate,
                                              ctx.needs_input_grad[5])
        return dx, da, dg, dA, dz, dh0, None, None


def _f32(t):
    return t if t.dtype == torch.float32 else t.float()


def gated_scan(x: torch.Tensor, a_gate: torch.Tensor, x_gate: torch.Tensor, A: torch.Tensor, *,
               z: torch.Tensor | None = None, h0: torch.Tensor | None = None,
               lengths: torch.Tensor | None = None, return_state: bool = False,
               checkpoint: str = "full"):
    """The gated recurrence over a batch of sequences (see the module's formulas).

    x, a_gate, x_gate and z: (batch, seqlen, dim) of one dtype (float32, float16, bfloat16) with unit channel
    stride, any strides of batch and time.  A: (dim,), at most 0 (-inf is a = 0; above 0 the channel gives
    NaN).  h0: (batch, dim), the state before the first token, zeros if not given.  lengths: (batch,) int32
    or int64 on the same GPU; tokens from lengths[b] on (clamped to 0 .. seqlen) leave the state alone, have
    y = 0 and zero gradients, whatever their inputs hold.

    Returns y (batch, seqlen, dim), contiguous, in x's dtype; with ``return_state`` also the state after
    each sequence's last token, (batch, dim) float32.

    Gradients flow to x, a_gate, x_gate, z, A and h0 (once, not twice).  For them a call that needs any keeps
    the state before every 16th token and, with ``checkpoint="full"``, its inputs as they are; with
    ``checkpoint="int8"`` the inputs as 8-bit codes (``act8_pack``), and the gradients are those at the values
    that the codes stand for.  At a = 1 (A = 0, or a gate so far down that A r vanishes), where the square
    root has no slope, its term counts as 0.

    To capture a backward pass into a graph, capture the forward pass with it, and let no eager autograd
    graph of the same leaf tensors be alive at that time."""
    if x.dim() != 3:
        raise ValueError(f"x must be (batch, seqlen, dim), got {tuple(x.shape)}")
    b, _, d = x.shape
    for name, t in (("x", x), ("a_gate", a_gate), ("x_gate", x_gate), ("z", z)):
        if t is None:
            continue
        if t.shape != x.shape:
            raise ValueError(f"{name} is {tuple(t.shape)}, x {tuple(x.shape)}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, x {x.dtype}")
        channels_last(t, name)
    _lib.dtype_code(x.dtype)
    _check_rest(A, h0, lengths, b, d)
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"checkpoint must be one of {CHECKPOINTS}, got {checkpoint!r}")
    _lib.require_cuda(x, a_gate, x_gate, A, z, h0, lengths)
    A = _f32(A).contiguous()
    h0 = None if h0 is None else _f32(h0).contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, a_gate, x_gate, A, z, h0)):
        y, state = _GatedScan.apply(x, a_gate, x_gate, A, z, h0, lengths, checkpoint)
    else:
        y, state, _, _ = _forward(x, a_gate, x_gate, A, z, h0, lengths, return_state, False, checkpoint)
    return (y, state) if return_state else y


def _check_rest(A, h0, lengths, b, d):
    if A.shape != (d,):
        raise ValueError(f"A is {tuple(A.shape)}, expected ({d},)")
    if not A.is_floating_point():
        raise TypeError(f"A is {A.dtype}")
    if h0 is not None:
        if h0.shape != (b, d):
            raise ValueError(f"h0 is {tuple(h0.shape)}, expected {(b, d)}")
        if not h0.is_floating_point():
            raise TypeError(f"h0 is {h0.dtype}")
    if lengths is not None:
        if lengths.shape != (b,):
            raise ValueError(f"lengths is {tuple(lengths.shape)}, expected ({b},)")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"lengths is {lengths.dtype}, expected int32 or int64")


def gated_scan_step(state: torch.Tensor, x: torch.Tensor, a_gate: torch.Tensor, x_gate: torch.Tensor,
                    A: torch.Tensor, *, z: torch.Tensor | None = None,
                    state_out: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """One token of every sequence: the new state and y (batch, dim) in x's dtype, which is returned.

    state (batch, dim) contiguous float32 is updated in place, or left as it is where ``state_out`` (the same
    kind of tensor) is given.  x, a_gate, x_gate, z: (batch, dim) of one dtype with unit channel stride; A
    (dim,).  Not differentiable: a tensor that requires a gradient is refused while gradients are on."""
    if x.dim() != 2:
        raise ValueError(f"x must be (batch, dim), got {tuple(x.shape)}")
    b, d = x.shape
    for name, t in (("x", x), ("a_gate", a_gate), ("x_gate", x_gate), ("z", z), ("out", out)):
        if t is None:
            continue
        if t.shape != x.shape:
            raise ValueError(f"{name} is {tuple(t.shape)}, x {tuple(x.shape)}")
        if t.dtype != x.dtype:
            raise TypeError(f"{name} is {t.dtype}, x {x.dtype}")
        channels_last(t, name)
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None and (t.shape != (b, d) or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 {(b, d)}")
    code = _lib.dtype_code(x.dtype)
    _check_rest(A, None, None, b, d)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (state, x, a_gate, x_gate, A, z)):
        raise RuntimeError("gated_scan_step has no gradient: call it under no_grad or inference_mode, "
                           "or train through gated_scan")
    dev = _lib.require_cuda(state, x, a_gate, x_gate, A, z, state_out, out)
    lib = _lib.load()
    A = _f32(A).contiguous()
    if out is None:
        out = torch.empty((b, d), dtype=x.dtype, device=dev)
    with _lib.on_device(dev):
        st = lib.mm_gated_scan_step(
            state.data_ptr(), state.data_ptr() if state_out is None else state_out.data_ptr(), x.data_ptr(),
            a_gate.data_ptr(), x_gate.data_ptr(), A.data_ptr(), _lib.ptr(z), out.data_ptr(), b, d, x.stride(0),
            a_gate.stride(0), x_gate.stride(0), z.stride(0) if z is not None else 0, out.stride(0), code,
            _lib.stream_of(dev))
    _lib.check(st, "mm_gated_scan_step")
    return out
