"""Gated linear recurrence with one state a channel, over long sequences and token by token.

    r = sigmoid(a_gate)    i = sigmoid(x_gate)    a = exp(A[d] r)
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) i_t x_t           y = h (silu(z) where there is a z)

``gated_scan`` runs it over (batch, seqlen, dim) and is differentiable; ``gated_scan_step`` is its
single token.  It stands beside ``selective_scan``, whose channels have dstate states each and whose
input carries no gate.  Arithmetic and states are float32 for every dtype.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from mamba_metal_amd import _lib
from mamba_metal_amd.act8 import BLOCK, channels_last
from mamba_metal_amd.selective_scan import _status_word

CHECKPOINTS = ("full", "int8")
_two = _lib._i64a2


def _params(A, lengths, dtype, shape, dev) -> _lib.GatedScanParams:
    p = _lib.GatedScanParams()
    p.A = A.data_ptr()
    if lengths is not None:
        p.lengths = lengths.data_ptr()
        p.lengths_dtype = 1 if lengths.dtype == torch.int64 else 0
    p.batch, p.seqlen, p.dim = shape
    p.dtype = _lib.dtype_code(dtype)
    p.status = _status_word(dev).data_ptr()
    return p


def _set_inputs(p, x, a_gate, x_gate, z):
    p.x, p.x_stride = x.data_ptr(), _two(*x.stride()[:2])
    p.a_gate, p.a_gate_stride = a_gate.data_ptr(), _two(*a_gate.stride()[:2])
    p.x_gate, p.x_gate_stride = x_gate.data_ptr(), _two(*x_gate.stride()[:2])
    if z is not None:
        p.z, p.z_stride = z.data_ptr(), _two(*z.stride()[:2])


def _set_codes(p, codes, exps):
    """codes (inputs, batch, blocks, dim, 16) and exps (inputs, batch, blocks, dim): act8_pack's of each input."""
    n = len(codes)
    if codes.numel():
        step = exps.numel() // n
        c, e = codes.data_ptr(), exps.data_ptr()
        for k in range(n):
            p.codes[k], p.exps[k] = c + k * step * BLOCK, e + k * step


def _call(name, p, backward, dev):
    lib = _lib.load()
    nbytes = lib.mm_gated_scan_workspace_size(p.batch, p.seqlen, p.dim, backward)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    with _lib.on_device(dev):
        st = getattr(lib, name)(p, _lib.stream_of(dev))
    _lib.check(st, name)


def _forward(dev, x, a_gate, x_gate, A, z, h0, lengths, want_state, train, checkpoint):
    """y, the final state (or None) and, for training, the block states and the inputs' 8-bit codes."""
    b, n, d = x.shape
    p = _params(A, lengths, x.dtype, (b, n, d), dev)
    _set_inputs(p, x, a_gate, x_gate, z)
    y = x.new_empty((b, n, d))
    p.y, p.y_stride = y.data_ptr(), _two(n * d, d)
    state = blocks = codes = exps = None
    if h0 is not None:
        p.h0 = h0.data_ptr()
    if want_state:
        state = torch.empty((b, d), dtype=torch.float32, device=dev)
        p.state_out = state.data_ptr()
    if train:
        nblk = -(-n // BLOCK)
        blocks = torch.empty((b, nblk, d), dtype=torch.float32, device=dev)
        p.block_states = blocks.data_ptr()
        if checkpoint == "int8":
            k = 3 if z is None else 4
            codes = torch.empty((k, b, nblk, d, BLOCK), dtype=torch.int8, device=dev)
            exps = torch.empty((k, b, nblk, d), dtype=torch.uint8, device=dev)
            _set_codes(p, codes, exps)
    _call("mm_gated_scan_fwd", p, 0, dev)
    return y, state, blocks, codes, exps


def _backward(dev, inputs, codes, exps, A, lengths, blocks, dtype, shape, gated, dy, dstate, want_dh0):
    """Gradients of x, a_gate, x_gate, z (or None), A and h0 (or None); ``inputs`` or their codes."""
    b, n, d = shape
    p = _params(A, lengths, dtype, shape, dev)
    p.block_states = blocks.data_ptr()
    if codes is not None:
        _set_codes(p, codes, exps)
        p.z_present = 1 if gated else 0
    else:
        _set_inputs(p, *inputs)
    if dy is None:  # only the final state was used
        dy = torch.zeros((1, 1, d), dtype=dtype, device=dev).expand(b, n, d)
    elif dy.dtype != dtype or (dy.stride(-1) != 1 and d > 1):
        dy = dy.to(dtype).contiguous()
    p.dy, p.dy_stride = dy.data_ptr(), _two(*dy.stride()[:2])
    if dstate is not None:
        dstate = dstate.contiguous()
        p.dstate = dstate.data_ptr()
    dx, da, dg = (dy.new_empty((b, n, d)) for _ in range(3))
    p.dx, p.da_gate, p.dx_gate = dx.data_ptr(), da.data_ptr(), dg.data_ptr()
    dz = dh0 = None
    if gated:
        dz = dy.new_empty((b, n, d))
        p.dz = dz.data_ptr()
    dA = (torch.empty if b else torch.zeros)((d,), dtype=torch.float32, device=dev)
    p.dA = dA.data_ptr()
    if want_dh0:
        dh0 = torch.empty((b, d), dtype=torch.float32, device=dev)
        p.dh0 = dh0.data_ptr()
    _call("mm_gated_scan_bwd", p, 1, dev)
    return dx, da, dg, dA, dz, dh0


def _checked(saved, dev, dtype, shape, gated, lengths_dtype):
    """The saved tensors, where hooks may have changed them."""
    (b, n, d), (A, lengths, blocks, *kept) = shape, saved
    nblk, k = -(-n // BLOCK), 4 if gated else 3
    if lengths_dtype is not None:
        lengths = _lib.saved(lengths, lengths_dtype, (b,), dev)
    if len(kept) == 2:
        kept = (_lib.saved(kept[0], torch.int8, (k, b, nblk, d, BLOCK), dev),
                _lib.saved(kept[1], torch.uint8, (k, b, nblk, d), dev))
    else:
        kept = [_lib.saved(t, dtype, shape, dev, rows=True) for t in kept[:k]] + [None] * (4 - k)
    return _lib.saved(A, torch.float32, (d,), dev), lengths, _lib.saved(blocks, torch.float32, (b, nblk, d), dev), *kept


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dev, x, a_gate, x_gate, A, z, h0, lengths, want_state, checkpoint):
        y, state, blocks, codes, exps = _forward(dev, x, a_gate, x_gate, A, z, h0, lengths, want_state, True, checkpoint)
        ctx.meta = (dev, x.dtype, x.shape, z is not None,
                    _lib.hooked() and (None if lengths is None else lengths.dtype,))
        ctx.set_materialize_grads(False)
        if codes is not None:
            ctx.save_for_backward(A, lengths, blocks, codes, exps)
        else:
            ctx.save_for_backward(A, lengths, blocks, x, a_gate, x_gate, z)
        return (y, state) if want_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        if dy is None and dstate is None:
            return (None,) * 10
        dev, dtype, shape, gated, hooked = ctx.meta
        saved = ctx.saved_tensors
        if hooked:
            saved = _checked(saved, dev, dtype, shape, gated, *hooked)
        A, lengths, blocks, *kept = saved
        inputs, codes, exps = (None, *kept) if len(kept) == 2 else (kept, None, None)
        grads = _backward(dev, inputs, codes, exps, A, lengths, blocks, dtype, shape, gated, dy, dstate,
                          ctx.needs_input_grad[6])
        return None, *grads, None, None, None


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

    Not-a-numbers and infinities stay in their sequence and channel and reach all later tokens there (an infinite
    state may become NaN).

    Gradients flow to x, a_gate, x_gate, z, A and h0 (once, not twice, and not in forward mode).  For them a call that needs any keeps
    the state before every 16th token and, with ``checkpoint="full"``, its inputs as they are; with
    ``checkpoint="int8"`` the inputs as 8-bit codes (``act8_pack``), and the gradients are those at the values
    that the codes stand for.  At a = 1 (A = 0, or a gate so far down that A r vanishes), where the square
    root has no slope, its term counts as 0.

    To capture a backward pass into a graph, capture the forward pass with it, and let no eager autograd
    graph of the same leaf tensors be alive at that time."""
    if x.dim() != 3:
        raise ValueError(f"x must be (batch, seqlen, dim), got {tuple(x.shape)}")
    b, _, d = x.shape
    _check_alike(x, (("a_gate", a_gate), ("x_gate", x_gate), ("z", z)))
    _lib.dtype_code(x.dtype)
    _check_rest(A, h0, lengths, b, d)
    if checkpoint not in CHECKPOINTS:
        raise ValueError(f"checkpoint must be one of {CHECKPOINTS}, got {checkpoint!r}")
    _lib.refuse_transforms("gated_scan", x, a_gate, x_gate, A, z, h0)
    dev = _lib.require_cuda(x, a_gate, x_gate, A, z, h0, lengths)
    A = _f32(A).contiguous()
    h0 = None if h0 is None else _f32(h0).contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, a_gate, x_gate, A, z, h0)):
        return _GatedScan.apply(dev, x, a_gate, x_gate, A, z, h0, lengths, return_state, checkpoint)
    y, state, *_ = _forward(dev, x, a_gate, x_gate, A, z, h0, lengths, return_state, False, checkpoint)
    return (y, state) if return_state else y


def _check_alike(x, others):
    """x has unit channel stride, and the others its shape, its dtype and that."""
    shape, dtype = x.shape, x.dtype
    channels_last(x, "x")
    for name, t in others:
        if t is None:
            continue
        if t.shape != shape:
            raise ValueError(f"{name} is {tuple(t.shape)}, x {tuple(shape)}")
        if t.dtype != dtype:
            raise TypeError(f"{name} is {t.dtype}, x {dtype}")
        channels_last(t, name)


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
    (dim,).  Not differentiable: a tensor that requires a gradient is refused while gradients are on, and one
    with a tangent always."""
    if x.dim() != 2:
        raise ValueError(f"x must be (batch, dim), got {tuple(x.shape)}")
    b, d = x.shape
    _check_alike(x, (("a_gate", a_gate), ("x_gate", x_gate), ("z", z), ("out", out)))
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None and (t.shape != (b, d) or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous float32 {(b, d)}")
    code = _lib.dtype_code(x.dtype)
    _check_rest(A, None, None, b, d)
    if torch.is_grad_enabled() and (state.requires_grad or x.requires_grad or a_gate.requires_grad
                                    or x_gate.requires_grad or A.requires_grad or (z is not None and z.requires_grad)):
        raise RuntimeError("gated_scan_step has no gradient: call it under no_grad or inference_mode, "
                           "or train through gated_scan")
    _lib.refuse_transforms("gated_scan_step", state, x, a_gate, x_gate, A, z)
    dev = _lib.require_cuda(state, x, a_gate, x_gate, A, z, state_out, out)
    lib = _lib.load()
    if A.dtype != torch.float32 or not A.is_contiguous():
        A = A.float().contiguous()
    if out is None:
        out = x.new_empty((b, d))
    with _lib.on_device(dev):
        st = lib.mm_gated_scan_step(
            state.data_ptr(), state.data_ptr() if state_out is None else state_out.data_ptr(), x.data_ptr(),
            a_gate.data_ptr(), x_gate.data_ptr(), A.data_ptr(), _lib.ptr(z), out.data_ptr(), b, d, x.stride(0),
            a_gate.stride(0), x_gate.stride(0), z.stride(0) if z is not None else 0, out.stride(0), code,
            _lib.stream_of(dev))
    _lib.check(st, "mm_gated_scan_step")
    return out
